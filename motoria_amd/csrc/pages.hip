// The pages of a key/value cache (include/mia_hip.h): which slot holds which
// page, and the copies that forks and compaction need.
//
// Which page goes where is decided by one workgroup (a scan over the counts
// of references gives the free pages of lowest index in order; the list's
// prefix sums say who gets which), so that the result does not depend on any
// order of atomics and a call is done whole or not at all. What a call then
// has to move is written into the plan, and a second launch moves it with
// every CU. All of it runs on the device: no wait, nothing allocated, the
// same calls in a captured graph.
//
// Measured (48 layers, 4 heads of 128 in bf16, pages of 16): compaction of 75 pages,
// 238 MB read and written, 57 us (4.2 TB/s; a large copy reaches 4.92) after a plan
// of 5.5; 48 forks, 73 MB, 23 us after 6; extend 5.6, a layer's rows of 64 tokens 3.0
// (each alone; small launches one after another take 3.6).
#include "pages_plan.h"

namespace {

constexpr int WIDE = 1024;               // a deciding workgroup that goes over every page

__global__ __launch_bounds__(NT) void k_extend(mhip_page_dims s, mhip_pages p, const int *seqs,
                                               const int *count, int n) {
    __shared__ Desk d;
    int *first, *list;
    const int want = decide(s, p, d, n, first, list, [&](int i, int &bad) {
        const int q = seqs[i], k = count ? count[i] : 1;
        if ((unsigned)q >= (unsigned)s.max_seqs || k < 0 || mark(d, q)) {
            bad = MHIP_PAGES_BAD;
            return 0LL;
        }
        const int l = p.len[q];
        if (n <= NT) {
            d.slot[i] = q;
            d.len[i] = l;
        }
        if (l < 0) bad = MHIP_PAGES_BAD;
        else if ((long long)l + k > (long long)s.max_blocks * s.page) bad = MHIP_PAGES_NO_SPACE;
        return bad ? 0LL : (long long)(blocks_of(l + k, s.page) - blocks_of(l, s.page));
    }, [](int) { return false; });
    if (want < 0) return;
    for (int x = threadIdx.x; x < want; x += NT) {
        const int i = entry_of(first, n, x), q = n <= NT ? d.slot[i] : seqs[i], g = list[x];
        const int b = blocks_of(n <= NT ? d.len[i] : p.len[q], s.page) + (x - first[i]);
        p.table[(size_t)q * s.max_blocks + b] = g;
        p.refs[g] = 1;
        if (x == want - 1) p.state[ST_HINT] = g + 1;
    }
    if (n > NT) __syncthreads();  // every length has been read
    for (int i = threadIdx.x; i < n; i += NT) {
        const int q = n <= NT ? d.slot[i] : seqs[i];
        p.len[q] = (n <= NT ? d.len[i] : p.len[q]) + (count ? count[i] : 1);
    }
}

__global__ __launch_bounds__(NT) void k_fork_plan(mhip_page_dims s, mhip_pages p, const int *src,
                                                  const int *dst, int n, int deep) {
    __shared__ Desk d;
    const Plan pl = plan_of(p.plan, s.n_pages);
    int *first, *list;
    const int want = decide(s, p, d, n, first, list, [&](int i, int &bad) {
        const int a = src[i], b = dst[i];
        if ((unsigned)a >= (unsigned)s.max_seqs || (unsigned)b >= (unsigned)s.max_seqs ||
            mark(d, b)) {
            bad = MHIP_PAGES_BAD;
            return 0LL;
        }
        const int l = p.len[a], lb = p.len[b];
        if (n <= NT) {
            d.slot[i] = a;
            d.len[i] = l;
        }
        if (lb != 0 || l < 0 || l > (long long)s.max_blocks * s.page) bad = MHIP_PAGES_BAD;
        return bad ? 0LL : (long long)(deep ? blocks_of(l, s.page) : l % s.page != 0);
    }, [&](int i) {  // a source that is also a destination
        const int a = src[i];
        return (unsigned)a < (unsigned)s.max_seqs && (d.seen[a >> 5] >> (a & 31) & 1);
    });
    if (threadIdx.x == 0) {
        pl.head[PL_PAIRS] = max(want, 0);
        pl.head[PL_OK] = want >= 0;
    }
    for (int x = threadIdx.x; x < want; x += NT) {
        const int i = entry_of(first, n, x), g = list[x];
        const int a = n <= NT ? d.slot[i] : src[i], l = n <= NT ? d.len[i] : p.len[a];
        const int b = deep ? x - first[i] : l / s.page;
        pl.src[x] = p.table[(size_t)a * s.max_blocks + b];
        pl.dst[x] = g;
        pl.rows[x] = min(s.page, l - b * s.page);
        p.table[(size_t)dst[i] * s.max_blocks + b] = g;
        p.refs[g] = 1;
        if (x == want - 1) p.state[ST_HINT] = g + 1;
    }
}

__global__ __launch_bounds__(WIDE) void k_compact_plan(mhip_page_dims s, mhip_pages p) {
    __shared__ long long lds[WIDE / 64];
    const Plan pl = plan_of(p.plan, s.n_pages);
    long long mine = 0, live;
    for (int i = threadIdx.x; i < s.n_pages; i += WIDE) mine += p.refs[i] > 0;
    (void)scan<WIDE>(mine, &live, lds);
    // holes below `live` and pages in use from there on: as many of each
    int holes = 0, movers = 0;
    for (int base = 0; base < s.n_pages; base += WIDE * PER) {
        const int at = base + threadIdx.x * PER;
        unsigned h = 0, m = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = at + j;
            if (i >= s.n_pages) break;
            const bool used = p.refs[i] > 0;
            if (i < live && !used) h |= 1u << j;
            if (i >= live && used) m |= 1u << j;
            if (i >= live) pl.map[i] = i;
        }
        long long all;  // two sums in one scan: movers in the high half
        const long long x = scan<WIDE>((long long)__popc(m) << 32 | __popc(h), &all, lds);
        int rh = holes + (int)(x & 0xffffffff), rm = movers + (int)(x >> 32);
        for (int j = 0; j < PER; j++) {
            if (h >> j & 1) pl.dst[rh++] = at + j;
            if (m >> j & 1) pl.src[rm++] = at + j;
        }
        holes += (int)(all & 0xffffffff);
        movers += (int)(all >> 32);
    }
    __syncthreads();
    const int pairs = min(holes, movers);
    for (int i = threadIdx.x; i < pairs; i += WIDE) {
        const int a = pl.src[i], b = pl.dst[i];
        pl.map[a] = b;
        pl.rows[i] = s.page;
        p.refs[b] = p.refs[a];
        p.refs[a] = 0;
    }
    if (threadIdx.x == 0) {
        pl.head[PL_PAIRS] = pairs;
        pl.head[PL_OK] = (int)live;
        p.state[ST_HINT] = (int)live;
    }
}

// The plan's copies: an item is one page in one layer of one array, its
// rows one run per head (in 4 bits the whole page: tokens share its words); 256 threads
// with four 16-byte pieces each in flight.
__device__ void copy_pages(const mhip_page_dims &s, const mhip_pages &p, const Plan &pl, int block,
                           int blocks) {
    const bool whole = s.type == MHIP_Q4;
    const int esz = s.type == MHIP_F32 ? 4 : 2, unit = s.head_dim * esz / 16;  // pieces of a row
    const size_t head = whole ? mhip::q4_block(s) / 16 : (size_t)s.page * unit, page = head * s.n_kv_heads;
    const long long items = (long long)pl.head[PL_PAIRS] * s.n_layers * 2;
    for (long long it = block; it < items; it += blocks) {
        const int x = (int)(it / (2 * s.n_layers)), y = (int)(it % (2 * s.n_layers));
        const int a = pl.src[x], b = pl.dst[x];
        if ((unsigned)a >= (unsigned)s.n_pages || (unsigned)b >= (unsigned)s.n_pages) {
            if (threadIdx.x == 0) atomicOr(&p.state[ST_BITS], MHIP_PAGES_BAD);
            continue;
        }
        uint4 *base = (uint4 *)(y & 1 ? p.v : p.k) + (size_t)(y >> 1) * s.n_pages * page;
        const uint4 *from = base + a * page;
        uint4 *to = base + b * page;
        const unsigned run = whole ? (unsigned)head : (unsigned)pl.rows[x] * unit, all = run * s.n_kv_heads;
        for (unsigned i = threadIdx.x; i < all; i += 4 * blockDim.x) {
            uint4 r[4];
            size_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned k = i + j * blockDim.x;
                o[j] = (k / run) * head + k % run;
                if (k < all) r[j] = from[o[j]];
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * blockDim.x < all) to[o[j]] = r[j];
        }
    }
}

// The children's rows of the table (the first n workgroups), and the copies.
__global__ __launch_bounds__(256) void k_fork(mhip_page_dims s, mhip_pages p, const int *src,
                                              const int *dst, int n, int deep) {
    const Plan pl = plan_of(p.plan, s.n_pages);
    if (!pl.head[PL_OK]) return;
    if ((int)blockIdx.x >= n) {
        copy_pages(s, p, pl, blockIdx.x - n, gridDim.x - n);
        return;
    }
    const int a = src[blockIdx.x], b = dst[blockIdx.x], l = p.len[a];
    const int full = l / s.page, have = blocks_of(l, s.page);
    const int *from = p.table + (size_t)a * s.max_blocks;
    int *to = p.table + (size_t)b * s.max_blocks;
    for (int i = threadIdx.x; i < s.max_blocks; i += blockDim.x) {
        if (i >= have) {
            to[i] = -1;
        } else if (i < full && !deep) {
            const int g = from[i];
            to[i] = g;
            if ((unsigned)g < (unsigned)s.n_pages) atomicAdd(&p.refs[g], 1);
            else atomicOr(&p.state[ST_BITS], MHIP_PAGES_BAD);
        }
    }
    if (threadIdx.x == 0) p.len[b] = l;
}

constexpr int TABLE_WGS = 64;  // workgroups of k_compact that rewrite the table

__global__ __launch_bounds__(256) void k_compact(mhip_page_dims s, mhip_pages p) {
    const Plan pl = plan_of(p.plan, s.n_pages);
    if (pl.head[PL_PAIRS] == 0) return;
    if (blockIdx.x >= TABLE_WGS) {
        copy_pages(s, p, pl, blockIdx.x - TABLE_WGS, gridDim.x - TABLE_WGS);
        return;
    }
    const int live = pl.head[PL_OK];
    const size_t all = (size_t)s.max_seqs * s.max_blocks;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)TABLE_WGS * 256) {
        const int g = p.table[i];
        if (g >= live && g < s.n_pages) p.table[i] = pl.map[g];
    }
}

// One workgroup per entry; the one that finds the slot's length set empties it.
__global__ __launch_bounds__(256) void k_free(mhip_page_dims s, mhip_pages p, const int *seqs) {
    __shared__ int had;
    const int q = seqs[blockIdx.x];
    if ((unsigned)q >= (unsigned)s.max_seqs) {
        if (threadIdx.x == 0) atomicOr(&p.state[ST_BITS], MHIP_PAGES_BAD);
        return;
    }
    if (threadIdx.x == 0) had = atomicExch(&p.len[q], 0);
    __syncthreads();
    const int have = had <= 0 ? 0 : min(blocks_of(had, s.page), s.max_blocks);
    int *row = p.table + (size_t)q * s.max_blocks;
    for (int i = threadIdx.x; i < have; i += blockDim.x) {
        const int g = row[i];
        row[i] = -1;
        if ((unsigned)g >= (unsigned)s.n_pages) {
            atomicOr(&p.state[ST_BITS], MHIP_PAGES_BAD);
        } else if (atomicSub(&p.refs[g], 1) == 1) {
            atomicMin(&p.state[ST_HINT], g);
        }
    }
}

// A thread per 16-byte piece of the rows (keys' pieces, then values'):
// gridDim.y workgroups share a row, or one takes several (`each`).
__global__ __launch_bounds__(256) void k_write(mhip_page_dims s, mhip_pages p, int layer,
                                               const int *seqs, const int *count, int rows,
                                               int max_count, const uint4 *k, const uint4 *v,
                                               size_t step, int unit, int each) {
    const unsigned pieces = (unsigned)s.n_kv_heads * unit;  // of one array's row
    unsigned x, row;
    if (each > 1) {
        const unsigned in = threadIdx.x / (2 * pieces);
        if (in >= (unsigned)each) return;
        row = blockIdx.x * each + in;
        x = threadIdx.x - in * 2 * pieces;
    } else {
        row = blockIdx.x;
        x = blockIdx.y * 256 + threadIdx.x;
    }
    if (row >= (unsigned)rows || x >= 2 * pieces) return;
    const int i = max_count == 1 ? row : row / max_count, j = max_count == 1 ? 0 : row % max_count;
    const unsigned y = x < pieces ? x : x - pieces;
    // (the row's bytes are in the caller's arrays whether its slot is right or not)
    const uint4 piece = (x < pieces ? k : v)[(size_t)row * step + y];
    const int q = seqs[i], m = count ? count[i] : max_count;
    if (j >= m) return;
    int g = -1;
    const int pos = (unsigned)q < (unsigned)s.max_seqs ? p.len[q] - m + j : -1;
    const int lp = __builtin_ctz(s.page);
    if (pos >= 0 && pos >> lp < s.max_blocks && m <= max_count)
        g = p.table[(size_t)q * s.max_blocks + (pos >> lp)];
    if ((unsigned)g >= (unsigned)s.n_pages) {
        if (x == 0) atomicOr(&p.state[ST_BITS], MHIP_PAGES_BAD);
        return;
    }
    const unsigned h = y / unit, c = y % unit;
    const size_t to = (((((size_t)layer * s.n_pages + g) * s.n_kv_heads + h) << lp) +
                       (pos & (s.page - 1))) * unit + c;
    ((uint4 *)(x < pieces ? p.k : p.v))[to] = piece;
}

__global__ __launch_bounds__(256) void k_clear(mhip_page_dims s, mhip_pages p) {
    const size_t all = (size_t)s.max_seqs * s.max_blocks;
    const size_t i0 = (size_t)blockIdx.x * 256 + threadIdx.x, d = (size_t)gridDim.x * 256;
    for (size_t i = i0; i < all; i += d) p.table[i] = -1;
    for (size_t i = i0; i < (size_t)s.max_seqs; i += d) p.len[i] = 0;
    for (size_t i = i0; i < (size_t)s.n_pages; i += d) p.refs[i] = 0;
    if (i0 < 16) p.state[i0] = 0;
}

// The free pages into state[ST_FREE], the error bits into state[ST_FREE + 1]
// (and cleared).
__global__ __launch_bounds__(WIDE) void k_status(mhip_page_dims s, mhip_pages p) {
    __shared__ long long lds[WIDE / 64];
    long long mine = 0, all;
    for (int i = threadIdx.x; i < s.n_pages; i += WIDE) mine += p.refs[i] <= 0;
    (void)scan<WIDE>(mine, &all, lds);
    if (threadIdx.x == 0) {
        p.state[ST_FREE] = (int)all;
        p.state[ST_FREE + 1] = p.state[ST_BITS];
        p.state[ST_BITS] = 0;
    }
}

bool dims_ok(const mhip_page_dims *s) {
    return s && ((s->type >= MHIP_F32 && s->type <= MHIP_BF16) ||
                 (s->type == MHIP_Q4 && s->head_dim % 32 == 0)) &&
           s->n_layers >= 1 && s->n_layers <= 65536 && s->n_kv_heads >= 1 && s->n_kv_heads <= 256 && s->head_dim >= 16 &&
           s->head_dim <= 256 && s->head_dim % 16 == 0 && s->page >= 16 && s->page <= 256 &&
           (s->page & (s->page - 1)) == 0 && s->n_pages >= 1 && s->n_pages <= 1 << 20 &&
           s->max_seqs >= 1 && s->max_seqs <= 65536 && s->max_blocks >= 1 &&
           (long long)s->max_blocks * s->page <= 1 << 30;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t pool_bytes(const mhip_page_dims *s) {
    const size_t blocks = (size_t)s->n_layers * s->n_pages * s->n_kv_heads;
    if (s->type == MHIP_Q4) return blocks * mhip::q4_block(*s);
    return blocks * s->page * s->head_dim * mhip::type_bytes(s->type);
}

// Workgroups for copies of at most `pairs` pages: an item each, at most
// eight per CU.
unsigned copy_grid(const mhip_page_dims *s, long long pairs) {
    const long long items = pairs * s->n_layers * 2;
    return (unsigned)(items < 2048 ? items : 2048);
}

using mhip::check_list;

}  // namespace

namespace mhip {

int check_list(mhip_ctx *c, const mhip_page_dims *s, const void *list, int n, const char *what) {
    if (n < 0 || n > s->max_seqs)
        return fail(c, "%s: %d entries, the cache has %d slots", what, n, s->max_seqs);
    if (n && !list) return fail(c, "%s: a null argument", what);
    return 0;
}

int check_pages(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, const char *what) {
    if (!s || !p) return fail(c, "%s: a null argument", what);
    if (!dims_ok(s))
        return fail(c, "%s: type %d, %d layers, %d heads of %d, %d pages of %d, %d slots of %d "
                    "pages: not a cache this library runs", what, s->type, s->n_layers,
                    s->n_kv_heads, s->head_dim, s->n_pages, s->page, s->max_seqs, s->max_blocks);
    if (!p->k || !p->v || !p->table || !p->len || !p->refs || !p->state || !p->plan)
        return fail(c, "%s: a null array of the cache", what);
    if (((uintptr_t)p->k | (uintptr_t)p->v) % 16)
        return fail(c, "%s: the cache's arrays must be 16-byte aligned", what);
    return 0;
}

}  // namespace mhip

extern "C" {

size_t mhip_pages_plan_bytes(const mhip_page_dims *s) {
    return dims_ok(s) ? ((size_t)PL_HEAD + 4 * (size_t)s->n_pages + s->max_seqs) * 4 : 0;
}

size_t mhip_pages_bytes(const mhip_page_dims *s) {
    if (!dims_ok(s)) return 0;
    return 2 * align256(pool_bytes(s)) + align256((size_t)s->max_seqs * s->max_blocks * 4) +
           align256((size_t)s->max_seqs * 4) + align256((size_t)s->n_pages * 4) + align256(64) +
           align256(mhip_pages_plan_bytes(s));
}

int mhip_pages_carve(const mhip_page_dims *s, void *d_base, mhip_pages *out) {
    if (!dims_ok(s) || !d_base || !out || (uintptr_t)d_base % 256) return -1;
    uint8_t *b = (uint8_t *)d_base;
    auto take = [&](size_t bytes) {
        uint8_t *r = b;
        b += align256(bytes);
        return r;
    };
    out->k = take(pool_bytes(s));
    out->v = take(pool_bytes(s));
    out->table = (int *)take((size_t)s->max_seqs * s->max_blocks * 4);
    out->len = (int *)take((size_t)s->max_seqs * 4);
    out->refs = (int *)take((size_t)s->n_pages * 4);
    out->state = (int *)take(64);
    out->plan = (int *)take(mhip_pages_plan_bytes(s));
    return 0;
}

int mhip_pages_clear(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p) {
    if (mhip::check_pages(c, s, p, "pages clear") || mhip::use_device(c)) return -1;
    k_clear<<<512, 256, 0, c->stream>>>(*s, *p);
    return mhip::check_launch(c, "pages clear");
}

int mhip_pages_extend(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p,
                      const int *d_seqs, const int *d_count, int n) {
    if (mhip::check_pages(c, s, p, "pages extend") || check_list(c, s, d_seqs, n, "pages extend"))
        return -1;
    if (!n) return 0;
    if (mhip::use_device(c)) return -1;
    k_extend<<<1, NT, 0, c->stream>>>(*s, *p, d_seqs, d_count, n);
    return mhip::check_launch(c, "pages extend");
}

int mhip_pages_write(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer,
                     const int *d_seqs, const int *d_count, int n, int max_count,
                     const void *d_k, const void *d_v, int ld) {
    if (mhip::check_pages(c, s, p, "pages write") || check_list(c, s, d_seqs, n, "pages write"))
        return -1;
    if (s->type == MHIP_Q4) return mhip::fail(c, "pages write: a cache in 4 bits takes its rows by mhip_pages_write_q4");
    const int esz = mhip::type_bytes(s->type), width = s->n_kv_heads * s->head_dim;
    if (layer < 0 || layer >= s->n_layers)
        return mhip::fail(c, "pages write: layer %d of %d", layer, s->n_layers);
    if (max_count < 0 || ld < width)
        return mhip::fail(c, "pages write: %d tokens a slot, rows %d apart (width %d)", max_count,
                          ld, width);
    if (!n || !max_count) return 0;
    if (!d_k || !d_v) return mhip::fail(c, "pages write: a null argument");
    if (((uintptr_t)d_k | (uintptr_t)d_v) % 16 || (size_t)ld * esz % 16)
        return mhip::fail(c, "pages write: rows must start on 16 bytes");
    if ((long long)n * max_count >= 1 << 24)  // (a launch holds less than 2^32 threads)
        return mhip::fail(c, "pages write: %d x %d rows in one call", n, max_count);
    if (mhip::use_device(c)) return -1;
    const int unit = s->head_dim * esz / 16, pieces = 2 * s->n_kv_heads * unit, rows = n * max_count;
    const int each = pieces <= 128 ? 256 / pieces : 1;
    const dim3 grid(mhip::blocks_for(rows, each), (pieces + 255) / 256);
    k_write<<<grid, 256, 0, c->stream>>>(*s, *p, layer, d_seqs, d_count, rows, max_count,
                                         (const uint4 *)d_k, (const uint4 *)d_v,
                                         (size_t)ld * esz / 16, unit, each);
    return mhip::check_launch(c, "pages write");
}

int mhip_pages_fork(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, const int *d_src,
                    const int *d_dst, int n, int flags) {
    if (mhip::check_pages(c, s, p, "pages fork") || check_list(c, s, d_src, n, "pages fork") ||
        check_list(c, s, d_dst, n, "pages fork"))
        return -1;
    if (flags & ~MHIP_PAGES_DEEP) return mhip::fail(c, "pages fork: unknown flags %d", flags);
    if (!n) return 0;
    if (mhip::use_device(c)) return -1;
    const int deep = flags & MHIP_PAGES_DEEP;
    long long pairs = (long long)n * (deep ? s->max_blocks : 1);
    if (pairs > s->n_pages) pairs = s->n_pages;
    k_fork_plan<<<1, NT, 0, c->stream>>>(*s, *p, d_src, d_dst, n, deep);
    k_fork<<<n + copy_grid(s, pairs), 256, 0, c->stream>>>(*s, *p, d_src, d_dst, n, deep);
    return mhip::check_launch(c, "pages fork");
}

int mhip_pages_free(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, const int *d_seqs,
                    int n) {
    // (a list may name a slot twice, so it may be longer than there are slots)
    if (mhip::check_pages(c, s, p, "pages free")) return -1;
    if (n < 0 || n >= 1 << 24 || (n && !d_seqs)) return mhip::fail(c, "pages free: %d entries", n);
    if (!n) return 0;
    if (mhip::use_device(c)) return -1;
    k_free<<<n, 256, 0, c->stream>>>(*s, *p, d_seqs);
    return mhip::check_launch(c, "pages free");
}

int mhip_pages_compact(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p) {
    if (mhip::check_pages(c, s, p, "pages compact") || mhip::use_device(c)) return -1;
    k_compact_plan<<<1, WIDE, 0, c->stream>>>(*s, *p);
    k_compact<<<TABLE_WGS + copy_grid(s, (s->n_pages + 1) / 2), 256, 0, c->stream>>>(*s, *p);
    return mhip::check_launch(c, "pages compact");
}

int mhip_pages_status(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int status[2]) {
    if (mhip::check_pages(c, s, p, "pages status")) return -1;
    if (!status) return mhip::fail(c, "pages status: a null argument");
    if (mhip::use_device(c)) return -1;
    k_status<<<1, WIDE, 0, c->stream>>>(*s, *p);
    int w[2];
    if (mhip::check_launch(c, "pages status") || mhip_d2h(c, w, p->state + ST_FREE, sizeof w))
        return -1;
    status[0] = w[1];
    status[1] = w[0];
    return 0;
}

}  // extern "C"
