// The entry points of the attention over a cache in 4 bits
// (include/mia_hip.h): arguments, workspace and how a call is cut; its kernels
// are in attn_q4.inc.
#include "attn_q4.h"

namespace {

using mhip_q4::Cut;
using mhip_q4::Job;
using mhip_q4::Stat;
using mhip_q4::SUM_EACH;
using mhip_q4::TILE;
using mhip_q4::WAVES;

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

int up(long long n, int to) { return (int)((n + to - 1) / to * to); }

// How a call is cut. Up to 512 positions a workgroup takes an item whole, which saves the join
// (5 us with its launch). Longer ones are cut into parts for all workgroups to be on their CUs at
// once, with some to spare, as an item's last part is shorter (two on a CU, one with heads of more than
// 192 elements, whose stages are large): 32 slots of up to 8000 positions 41.4 us with 448 parts in
// all, 44 with 640 and 47 with 896, where some have to wait for others to end; 16 slots of up to 2900
// 19.4, 20.5 with 640 and 20.9 with 896.
constexpr int WHOLE = 512, PARTS = 448, PARTS_LARGE = 224, LEAST = 2;

// Weights are added up from kept scores where a slot and head have one tile of up to 16 rows, some
// 2048 workgroups of 256 positions at least (memory is what they wait for). Else they are from
// new scores, by wavefronts that share positions where there are enough rows for them, with more
// positions for each once 256 workgroups have some (a chunk of 500 tokens over 6000: 299 us with its
// attention, 315 with 512 workgroups; 8 drafted tokens of 8 slots of up to 1000, fp32: 32 both).
constexpr int SUM_WGS = 256;
bool kept(const Cut &k) { return k.nq == 1 && k.tiles == 1; }

Cut cut_of(const mhip_page_dims *s, int n_heads, int n, int mc, int max_len) {
    Cut k;
    const int rows = mc * (n_heads / s->n_kv_heads);
    k.nq = rows <= 16 ? 1 : mhip_q4::wide_tiles(s->head_dim / 32);
    k.tiles = (rows + 16 * k.nq - 1) / (16 * k.nq);
    const long long items = (long long)n * k.tiles;
    const int parts = s->head_dim > 192 ? PARTS_LARGE : PARTS;
    // (a chunk at a slot's end: all items are about as long and none would be cut; 500 tokens over 6000
    // 152 us so, 160 with a join that finds nothing to do)
    const bool alike = n == 1 && mc <= max_len / 2 && items * s->n_kv_heads >= parts;
    const bool cut = items <= mhip_q4::ITEMS_MAX && max_len > WHOLE && items * s->n_kv_heads < 4 * parts && !alike;
    k.wgs = cut ? (parts + s->n_kv_heads - 1) / s->n_kv_heads : 0;
    const long long heads = (long long)n * s->n_kv_heads;
    if (kept(k)) {
        const long long each = max_len * heads / 2048;
        k.wsides = 1;
        k.wlen = each < 256 ? 256 : each > 1024 ? 1024 : up(each, 256);
    } else {
        k.wsides = k.tiles >= 3 ? 4 : k.tiles;
        const int side = WAVES / k.wsides;
        const long long each = (max_len + TILE - 1) / TILE * heads / (SUM_WGS * side);
        k.wlen = (each < 1 ? 1 : each > SUM_EACH ? SUM_EACH : (int)each) * side * TILE;
    }
    k.wparts = max_len > 0 ? (max_len + k.wlen - 1) / k.wlen : 1;
    return k;
}

bool shape_ok(const mhip_page_dims *s, int type, int n_heads, int n, int mc, int max_len) {
    return s->type == MHIP_Q4 && type >= MHIP_F32 && type <= MHIP_BF16 && n_heads >= 1 && n_heads <= 65536 &&
           n_heads % s->n_kv_heads == 0 && n >= 1 && n <= s->max_seqs && mc >= 1 &&
           (long long)n * mc * n_heads <= (1 << 26) - 4 && max_len >= 0 &&
           max_len <= (long long)s->max_blocks * s->page;
}

// A launch holds less than 2^32 threads: 2^24 workgroups of 256 (those that add weights up have up to 2^19
// more beside them, which join parts).
bool fits(const mhip_page_dims *s, int n, const Cut &k) {
    const long long items = (long long)n * s->n_kv_heads;
    return items * k.tiles < 1 << 24 && items * k.wparts < (1 << 24) - (1 << 19);
}

// The workspace: where items are cut, the results of the parts, what is kept of them and
// where each item's begin; what is kept of each row, where weights are added up.
struct Work {
    size_t o, part, row, start, kept, step;
};
Work work_of(const mhip_page_dims *s, int n_heads, int n, int mc, int max_len, const Cut &k, bool weights) {
    const size_t parts = k.wgs ? ((size_t)k.wgs + (size_t)n * k.tiles) * s->n_kv_heads * 16 * k.nq : 0;
    Work w;
    w.o = align256(parts * s->head_dim * 4);
    w.part = align256(parts * sizeof(Stat));
    w.row = weights ? align256((size_t)n * mc * n_heads * sizeof(Stat)) : 0;
    w.start = k.wgs ? align256(((size_t)n * k.tiles + 1) * 4) : 0;
    // (whole tiles of 32 positions)
    w.step = weights && kept(k) ? (size_t)up(max_len, 32) * mc * (n_heads / s->n_kv_heads) : 0;
    w.kept = align256(w.step * n * s->n_kv_heads * 4);
    return w;
}

}  // namespace

extern "C" {

size_t mhip_attention_q4_ws_bytes(const mhip_page_dims *s, int type, int n_heads, int n, int max_count, int max_len,
                                  int weights) {
    if (!mhip_pages_plan_bytes(s) || !shape_ok(s, type, n_heads, n, max_count, max_len)) return 0;
    const Cut k = cut_of(s, n_heads, n, max_count, max_len);
    if (!fits(s, n, k)) return 0;
    const Work w = work_of(s, n_heads, n, max_count, max_len, k, weights != 0);
    return w.o + w.part + w.row + w.start + w.kept + 256;
}

int mhip_attention_q4(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, int type, int n_heads,
                      const void *d_q, int ldq, void *d_out, int ldo, const int *d_seqs, const int *d_count, int n,
                      int max_count, int max_len, float scale, float *d_weights, void *d_ws) {
    const char *what = "attention q4";
    if (mhip::check_pages(c, s, p, what)) return -1;
    if (s->type != MHIP_Q4) return mhip::fail(c, "%s: a cache of type %d is not in 4 bits", what, s->type);
    if (type < MHIP_F32 || type > MHIP_BF16) return mhip::fail(c, "%s: rows of type %d", what, type);
    if (layer < 0 || layer >= s->n_layers) return mhip::fail(c, "%s: layer %d of %d", what, layer, s->n_layers);
    if (n == 0 || max_count == 0) return 0;
    if (!shape_ok(s, type, n_heads, n, max_count, max_len))
        return mhip::fail(c, "%s: %d heads over %d, %d x %d tokens, %d positions", what, n_heads, s->n_kv_heads, n,
                          max_count, max_len);
    const int esz = mhip::type_bytes(type);
    if (ldq < n_heads * s->head_dim || ldo < n_heads * s->head_dim)
        return mhip::fail(c, "%s: rows %d and %d apart (width %d)", what, ldq, ldo, n_heads * s->head_dim);
    if (!(scale >= 0x1p-64f && scale <= 0x1p64f))
        return mhip::fail(c, "%s: scale %g outside [2^-64, 2^64]", what, scale);
    if (!d_q || !d_out || !d_seqs || !d_ws) return mhip::fail(c, "%s: a null argument", what);
    if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_weights) % 16 || (size_t)ldq * esz % 16 ||
        (size_t)ldo * esz % 16 || (uintptr_t)d_ws % 256)
        return mhip::fail(c, "%s: rows and weights must start on 16 bytes, the workspace on 256", what);
    const Cut k = cut_of(s, n_heads, n, max_count, max_len);
    if (!fits(s, n, k)) return mhip::fail(c, "%s: too many rows or parts in one call", what);
    if (mhip::use_device(c)) return -1;
    const Work w = work_of(s, n_heads, n, max_count, max_len, k, d_weights != nullptr);
    Job a;
    a.s = *s;
    a.p = *p;
    a.layer = layer;
    a.nh = n_heads;
    a.group = n_heads / s->n_kv_heads;
    a.q = d_q;
    a.ldq = ldq;
    a.out = d_out;
    a.ldo = ldo;
    a.seqs = d_seqs;
    a.count = d_count;
    a.n = n;
    a.mc = max_count;
    a.max_len = max_len;
    a.c = scale * 1.44269504088896341f;
    a.lp = __builtin_ctz(s->page);
    a.tiles = k.tiles;
    a.wgs = k.wgs;
    a.least = LEAST;
    uint8_t *ws = (uint8_t *)d_ws;
    a.o = (float *)ws;
    a.part = (Stat *)(ws + w.o);
    a.row = (Stat *)(ws + w.o + w.part);
    a.start = (int *)(ws + w.o + w.part + w.row);
    a.kept = w.kept ? (float *)(ws + w.o + w.part + w.row + w.start) : nullptr;
    a.keep_step = w.step;
    a.weights = d_weights;
    a.wparts = k.wparts;
    a.wlen = k.wlen;
    a.wsides = k.wsides;
    if (type == MHIP_F32) return mhip_q4::launch_f32(c, a, k);
    if (type == MHIP_F16) return mhip_q4::launch_f16(c, a, k);
    return mhip_q4::launch_bf16(c, a, k);
}

}  // extern "C"
