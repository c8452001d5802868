// The entry points of the attention over a paged cache (include/mia_hip.h):
// arguments, workspace and how a call is cut; its kernels are in
// attn_shared.inc.
#include "attn_shared.h"

namespace {

using mhip_shared::Cut;
using mhip_shared::Job;
using mhip_shared::PART_MAX;
using mhip_shared::TILE;

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a call is cut. A part of the prefix serves up to 128 rows (16-bit heads up
// to 128); tiles of 64 rows do better up to 256 rows in all (bf16, 8 rows a slot behind 8000
// tokens: 24 slots 21.4 us, with tiles of 128 rows 24.5; 32 slots 24.0 and 25.6; 40 slots 30.9 and
// 31.0; 56 slots 52.7 and 45.7). Every part's results pass through memory once more, so there are
// only as many as keep the CUs busy: 256 workgroups for the prefix (64 slots
// behind 8000: 8 parts 45 us, 16 parts 32.6, 32 parts 41) and 256 for the slots (32
// unshared slots of up to 8000 tokens: 2 parts 75 us, 8 parts 81; 64 of 300
// tokens: 1 part 10.4 us, 2 parts 15.4). Without a prefix one part needs no join, so the
// number is rounded down (200 workgroups or 400: 500 positions 12.7 and 16.6 us, 2000
// positions 36.4 and 40.6), else up (fp16, 168 or 336: 20.1 and 17.1). Where a CU holds one
// workgroup only the two together should not be more than the CUs. fp32 tiles keep the matrix cores busy, so that two workgroups on a CU
// take twice as long: slots of up to 512 positions behind a prefix stay in one part each
// where that keeps the launch at one a CU (64 slots' workgroups or 128 beside 160 of the
// prefix: 300 positions 22.8 us and 26.9, 400 26.5 and 29.0, 500 29.0 and 29.3, 600 31.4 and
// 29.1; 128 or 256 beside 56: 300 positions 15.2 and 17.3, 600 20.1 and 19.9); else they
// are cut as others are (beside 248: 400 positions 36.5 and 30.6).
Cut cut_of(const mhip_page_dims *s, int n_heads, int n, int mc, int prefix, int max_len) {
    Cut k;
    const int group = n_heads / s->n_kv_heads, rest = max_len - prefix;
    const long long rows = (long long)n * mc * group;
    k.stiles = (mc * group + 15) / 16;
    k.wr = prefix == 0 ? 1 : rows > 32 ? 4 : rows > 16 ? 2 : 1;
    k.rt = prefix > 0 && rows > 256 && s->head_dim <= 128 && s->type != MHIP_F32 ? 2 : 1;
    const int tile = k.wr * k.rt * 16;
    k.ptiles = prefix > 0 ? (int)((rows + tile - 1) / tile) : 0;
    const long long items = (long long)n * s->n_kv_heads * k.stiles;

    auto cut = [&](long long parts) {  // `parts` for each slot
        k.slen = rest > 0 ? (int)((rest + parts - 1) / parts + TILE - 1) / TILE * TILE : TILE;
        k.ss = rest > 0 ? (rest + k.slen - 1) / k.slen : 1;
        k.sp = 0;
        k.plen = 0;
        if (prefix == 0) return;
        const int padded = s->head_dim <= 64 ? 64 : s->head_dim <= 128 ? 128 : 256;
        const bool single = padded * mhip::type_bytes(s->type) > (tile > 16 ? 512 : 256);
        long long wgs = (single ? 256 : 512) - items * k.ss;
        if (wgs > 256) wgs = 256;
        if (wgs < 128) wgs = 128;
        long long pp = wgs / ((long long)k.ptiles * s->n_kv_heads);
        const int pmost = (prefix + 127) / 128, pleast = (prefix + PART_MAX - 1) / PART_MAX;
        if (pp > pmost) pp = pmost;
        if (pp < pleast) pp = pleast;
        k.plen = (int)((prefix + pp - 1) / pp + TILE - 1) / TILE * TILE;
        k.sp = (prefix + k.plen - 1) / k.plen;
    };
    auto wgs = [&]() { return items * k.ss + (long long)s->n_kv_heads * k.ptiles * k.sp; };
    const int most = (rest + 255) / 256, least = (rest + PART_MAX - 1) / PART_MAX;
    long long parts = prefix == 0 ? 256 / items : (256 + items - 1) / items;
    if (parts > most) parts = most;
    if (parts < least) parts = least;
    if (parts < 1) parts = 1;
    cut(1);
    const bool one = s->type == MHIP_F32 && prefix > 0 && rest <= 512 && wgs() <= 256;
    if (parts > 1) cut(parts);
    if (one && wgs() > 256) cut(1);
    return k;
}

bool shape_ok(const mhip_page_dims *s, int n_heads, int n, int mc, int prefix, int max_len) {
    return s->type != MHIP_Q4 && n_heads >= 1 && n_heads <= 65536 && n_heads % s->n_kv_heads == 0 && n >= 1 &&
           n <= s->max_seqs && mc >= 1 && (long long)n * mc * n_heads < 1 << 26 && prefix >= 0 &&
           max_len >= prefix && max_len <= (long long)s->max_blocks * s->page;
}

// A launch holds less than 2^32 threads: 2^24 workgroups of 256 (k_join: one for four rows).
bool fits(const mhip_page_dims *s, int n_heads, int n, int mc, const Cut &k) {
    return s->n_kv_heads * ((long long)k.ptiles * k.sp + (long long)n * k.stiles * k.ss) < 1 << 24 &&
           (k.sp + k.ss == 1 || (long long)n * mc * n_heads <= (1 << 26) - 4);
}

}  // namespace

extern "C" {

size_t mhip_attention_shared_ws_bytes(const mhip_page_dims *s, int n_heads, int n, int max_count,
                                      int prefix, int max_len) {
    if (!mhip_pages_plan_bytes(s) || !shape_ok(s, n_heads, n, max_count, prefix, max_len)) return 0;
    const Cut k = cut_of(s, n_heads, n, max_count, prefix, max_len);
    if (!fits(s, n_heads, n, max_count, k)) return 0;
    const size_t rows = (size_t)n * max_count * n_heads, parts = (size_t)k.sp + k.ss;
    return align256(parts * rows * s->head_dim * 4) + align256(parts * rows * 8);
}

int mhip_attention_shared(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer,
                          int n_heads, const void *d_q, int ldq, void *d_out, int ldo,
                          const int *d_seqs, const int *d_count, int n, int max_count,
                          int prefix_seq, int prefix, int max_len, float scale, void *d_ws) {
    const char *what = "attention shared";
    if (mhip::check_pages(c, s, p, what)) return -1;
    if (s->type == MHIP_Q4) return mhip::fail(c, "%s: a cache in 4 bits is read by mhip_attention_q4", what);
    if (layer < 0 || layer >= s->n_layers) return mhip::fail(c, "%s: layer %d of %d", what, layer, s->n_layers);
    if (n == 0 || max_count == 0) return 0;
    if (!shape_ok(s, n_heads, n, max_count, prefix, max_len))
        return mhip::fail(c, "%s: %d heads over %d, %d x %d tokens, prefix %d of %d positions", what,
                          n_heads, s->n_kv_heads, n, max_count, prefix, max_len);
    if (prefix > 0 && (prefix_seq < 0 || prefix_seq >= s->max_seqs))
        return mhip::fail(c, "%s: prefix of slot %d of %d", what, prefix_seq, s->max_seqs);
    const int esz = mhip::type_bytes(s->type);
    if (ldq < n_heads * s->head_dim || ldo < n_heads * s->head_dim)
        return mhip::fail(c, "%s: rows %d and %d apart (width %d)", what, ldq, ldo, n_heads * s->head_dim);
    if (!(scale >= 0x1p-64f && scale <= 0x1p64f))
        return mhip::fail(c, "%s: scale %g outside [2^-64, 2^64]", what, scale);
    if (!d_q || !d_out || !d_seqs || !d_ws) return mhip::fail(c, "%s: a null argument", what);
    if (((uintptr_t)d_q | (uintptr_t)d_out) % 16 || (size_t)ldq * esz % 16 || (size_t)ldo * esz % 16 ||
        (uintptr_t)d_ws % 256)
        return mhip::fail(c, "%s: rows must start on 16 bytes, the workspace on 256", what);
    const Cut k = cut_of(s, n_heads, n, max_count, prefix, max_len);
    if (!fits(s, n_heads, n, max_count, k)) return mhip::fail(c, "%s: too many rows or parts in one call", what);
    if (mhip::use_device(c)) return -1;
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
    a.prefix_seq = prefix_seq;
    a.prefix = prefix;
    a.max_len = max_len;
    a.c = scale * 1.44269504088896341f;
    a.lp = __builtin_ctz(s->page);
    a.sp = k.sp;
    a.plen = k.plen;
    a.ptiles = k.ptiles;
    a.ss = k.ss;
    a.slen = k.slen;
    a.stiles = k.stiles;
    const size_t rows = (size_t)n * max_count * n_heads, parts = (size_t)k.sp + k.ss;
    a.o = (float *)d_ws;
    a.ml = (float *)((uint8_t *)d_ws + align256(parts * rows * s->head_dim * 4));
    if (s->type == MHIP_F32) return mhip_shared::launch_f32(c, a, k);
    if (s->type == MHIP_F16) return mhip_shared::launch_f16(c, a, k);
    return mhip_shared::launch_bf16(c, a, k);
}

}  // extern "C"
