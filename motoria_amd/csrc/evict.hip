// Eviction from a cache in 4 bits by accumulated attention weight
// (include/mia_hip.h). For a slot longer than `keep`, and in each layer and head by
// itself, the last `recent` tokens and the keep - recent others of the greatest weight stay,
// in their order, as tokens 0 .. keep - 1.
//
//   k_evict_begin  a workgroup per slot, layer and head: the least weight that
//                  stays by three rounds of counting (11, 11 and 10 bits of the weight as a
//                  whole number), then the positions that stay, in order; one more keeps the
//                  books meanwhile (4 short slots 14.9 us in all, with a launch for the plan
//                  and one for the books 24.9)
//   k_evict_move   workgroups per slot, layer, head and array move what stays
//
// Tokens only move towards the front, so within a page they move in place: a
// workgroup takes its tokens in order, 512 at a time, and writes where it has read.
//
// 8000 tokens to 4000 in 48 layers of 4 heads of 128: selecting 17 us (a row of weights is read five
// times, from the cache after the first), moving 126, where a copy of the bytes would take 51: a
// value's code is a byte of a word of four tokens, and the chunks of a head have to follow each
// other. (Chunks of 128 whose places are looked up in turn: 258 us. A chunk asked for while the one
// before is written: the same 126, in twice the registers.)
#include "cache_q4.h"
#include "pages_plan.h"

namespace {

using mhip_q4::Shape;

constexpr int SEL = 512;        // threads that select
constexpr int BINS = 2048;
constexpr int CHUNK = 512;      // tokens that move at a time
constexpr int MOVE = 512;       // threads that move them

// The workspace of a call.
struct Work {
    int *stay;       // [n][layers][heads][keep] positions
    int *from, *to;  // [n][blocks of max_len], [n][blocks of keep] pages
    int *need;       // [n] pages shared with others; -1: none moves, -2: a page out of range
    uint8_t *shared; // [n][blocks of keep]
    int fb, tb;
    size_t bytes;
};
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
Work work_of(const mhip_page_dims *s, int n, int keep, int max_len, void *d_ws) {
    Work w;
    const int most = keep < max_len ? keep : max_len;
    w.fb = (max_len + s->page - 1) / s->page;
    w.tb = (most + s->page - 1) / s->page;
    uint8_t *b = (uint8_t *)d_ws;
    w.bytes = 0;
    auto take = [&](size_t bytes) {
        uint8_t *r = b + w.bytes;
        w.bytes += align256(bytes);
        return r;
    };
    w.need = (int *)take((size_t)n * 4);
    w.from = (int *)take((size_t)n * w.fb * 4);
    w.to = (int *)take((size_t)n * w.tb * 4);
    w.shared = take((size_t)n * w.tb);
    w.stay = (int *)take((size_t)n * s->n_layers * s->n_kv_heads * most * 4);
    return w;
}

// A weight as a whole number of the same order (-0 as 0, NaN below all).
__device__ __forceinline__ unsigned key_of(float w) {
    const unsigned u = __float_as_uint(w + 0.0f);
    return w != w ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ inline int slot_length(const mhip_page_dims &s, const mhip_pages &p, int q, int max_len) {
    if ((unsigned)q >= (unsigned)s.max_seqs) return -1;
    const int l = p.len[q];
    return l > max_len ? -1 : l;
}

// The books of a call, by one workgroup beside those that select: pages for those that other
// slots hold too, tables and counts of references, the old and the new pages into the workspace. A
// wavefront takes an entry at a time. (Lengths change with the moves: selecting reads them.)
__device__ void keep_books(const mhip_page_dims &s, const mhip_pages &p, Desk &d, const int *seqs, int n, int keep,
                           int max_len, const Work &w) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = wave; i < n; i += SEL / 64) {
        const int q = seqs[i], len = slot_length(s, p, q, max_len);
        int need = -1;
        if (len > keep) {
            const int have = blocks_of(len, s.page);
            need = 0;
            for (int b0 = 0; b0 < have; b0 += 64) {
                const int b = b0 + lane;
                const int g = b < have ? p.table[(size_t)q * s.max_blocks + b] : 0;
                const bool bad = (unsigned)g >= (unsigned)s.n_pages, held = !bad && b < have && b < w.tb && p.refs[g] > 1;
                if (b < have && b < w.tb) w.shared[(size_t)i * w.tb + b] = (uint8_t)held;
                if (__any(bad)) {
                    need = -2;
                    break;
                }
                need += __popcll(__ballot(held));
            }
        }
        if (lane == 0) w.need[i] = need;
    }
    __syncthreads();
    const Plan pl = plan_of(p.plan, s.n_pages);
    int *first, *list;
    const int want = decide<SEL>(s, p, d, n, first, list, [&](int i, int &bad) {
        const int q = seqs[i];
        if ((unsigned)q >= (unsigned)s.max_seqs || mark(d, q) || p.len[q] < 0 || p.len[q] > max_len ||
            w.need[i] == -2) {
            bad = MHIP_PAGES_BAD;
            return 0LL;
        }
        return (long long)max(w.need[i], 0);
    }, [](int) { return false; });
    if (threadIdx.x == 0) {
        pl.head[PL_PAIRS] = 0;
        pl.head[PL_OK] = want >= 0;
    }
    if (want < 0) return;
    for (int x = threadIdx.x; x < want; x += SEL) {
        const int g = list[x];
        p.refs[g] = 1;
        if (x == want - 1) p.state[ST_HINT] = g + 1;
    }
    __syncthreads();
    for (int i = wave; i < n; i += SEL / 64) {
        if (w.need[i] < 0) continue;
        const int q = seqs[i], have = blocks_of(p.len[q], s.page);
        int *row = p.table + (size_t)q * s.max_blocks;
        int next = first[i];
        for (int b0 = 0; b0 < have; b0 += 64) {
            const int b = b0 + lane;
            const bool front = b < w.tb, swap = b < have && front && w.shared[(size_t)i * w.tb + b];
            const unsigned long long swaps = __ballot(swap);
            const int at = next + __popcll(swaps & ((1ull << lane) - 1));
            next += __popcll(swaps);
            if (b >= have) continue;
            const int g = row[b], to = swap ? list[at] : g;
            w.from[(size_t)i * w.fb + b] = g;
            if (front) w.to[(size_t)i * w.tb + b] = to;
            if (swap || !front) {
                row[b] = front ? to : -1;
                if (atomicSub(&p.refs[g], 1) == 1) atomicMin(&p.state[ST_HINT], g);
            }
        }
    }
}

__global__ __launch_bounds__(SEL) void k_evict_begin(mhip_page_dims s, mhip_pages p, const float *weights,
                                                      const int *seqs, int n, int keep, int recent, int max_len,
                                                      Work w) {
    __shared__ union {
        Desk desk;
        struct {
            int bins[BINS];
            long long sums[SEL / 64];
            int found[2];
        } of;
    } lds;
    if (blockIdx.x == 0) {
        keep_books(s, p, lds.desk, seqs, n, keep, max_len, w);
        return;
    }
    int *bins = lds.of.bins, *found = lds.of.found;
    long long *sums = lds.of.sums;
    const int tid = threadIdx.x;
    const long long items = (long long)n * s.n_layers * s.n_kv_heads;
    for (long long it = blockIdx.x - 1; it < items; it += gridDim.x - 1) {
        const int h = (int)(it % s.n_kv_heads), layer = (int)(it / s.n_kv_heads % s.n_layers);
        const int i = (int)(it / s.n_kv_heads / s.n_layers), q = seqs[i];
        const int len = slot_length(s, p, q, max_len);
        if (len <= keep) continue;
        const float *row = weights + mhip_q4::weights_row(s, layer, q, h);
        int *stay = w.stay + (size_t)it * keep;
        const int nc = len - recent, kc = keep - recent;  // candidates, and how many of them stay
        unsigned least = 0;                               // the least key that stays
        int equal = kc;                                   // how many of that very key do
        int taken = 0;                                    // bits of `least` that are known
        while (kc > 0 && taken < 32) {
            const int width = taken < 22 ? 11 : 10, shift = 32 - taken - width;
            for (int b = tid; b < BINS; b += SEL) bins[b] = 0;
            __syncthreads();
            for (int x = tid * 4; x < nc; x += SEL * 4) {  // (a row is whole fours of floats)
                const float4 v = *(const float4 *)(row + x);
                const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned k = key_of(f[e]);
                    if (x + e < nc && (taken == 0 || k >> (32 - taken) == least >> (32 - taken)))
                        atomicAdd(&bins[k >> shift & ((1u << width) - 1)], 1);
                }
            }
            __syncthreads();
            // from the highest bin down: the one in which the count reaches `equal`
            constexpr int EACH = BINS / SEL;
            const int top = BINS - 1 - tid * EACH;
            int mine = 0;
#pragma unroll
            for (int e = 0; e < EACH; e++) mine += bins[top - e];
            long long all;
            int above = (int)scan<SEL>(mine, &all, sums);
            if (above < equal && above + mine >= equal) {
                int b = top;
                while (above + bins[b] < equal) above += bins[b--];
                found[0] = b;
                found[1] = equal - above;
            }
            __syncthreads();
            least |= (unsigned)found[0] << shift;
            equal = found[1];
            taken += width;
            __syncthreads();
        }
        // the candidates that stay, each thread a run of positions
        if (kc > 0) {
            const int run = ((nc + SEL - 1) / SEL + 3) & ~3, x0 = min(nc, tid * run), x1 = min(nc, x0 + run);
            int more = 0, same = 0;
            for (int x = x0; x < x1; x += 4) {
                const float4 v = *(const float4 *)(row + x);
                const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned k = key_of(f[e]);
                    more += x + e < x1 && k > least;
                    same += x + e < x1 && k == least;
                }
            }
            long long all;
            const long long before = scan<SEL>((long long)more << 32 | same, &all, sums);
            more = (int)(before >> 32);
            same = (int)(before & 0xffffffff);
            for (int x = x0; x < x1; x += 4) {
                const float4 v = *(const float4 *)(row + x);
                const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (x + e >= x1) break;
                    const unsigned k = key_of(f[e]);
                    if (k > least || (k == least && same < equal)) stay[more + min(same, equal)] = x + e;
                    more += k > least;
                    same += k == least;
                }
            }
        }
        for (int x = tid; x < recent; x += SEL) stay[kc + x] = nc + x;
    }
}

// What this thread has read is here, and so is what the others have.
__device__ __forceinline__ void all_read() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Workgroups that share a head's keys (or values): each moves its part of every token. (8000 tokens
// to 4000 in 48 layers, a first call: 162 us, with two 185, with one 225.)
__host__ __device__ constexpr int sides(int groups) { return groups >= 4 ? 4 : groups >= 2 ? 2 : 1; }

// Tokens of a chunk: the page in which each is and will be (of this layer and head), and its number there.
struct Chunk {
    unsigned from[CHUNK], to[CHUNK];
    uint8_t at[CHUNK];
    int moves[MOVE / 64];
};
static_assert(CHUNK <= MOVE, "a thread looks at one token of a chunk");

template <int G>
__global__ __launch_bounds__(MOVE) void k_evict_move(mhip_page_dims s, mhip_pages p, float *weights,
                                                     const int *seqs, int n, int keep, Work w) {
    __shared__ Chunk d[3];
    const Shape f = mhip_q4::shape_of(s);
    if (!plan_of(p.plan, s.n_pages).head[PL_OK]) return;
    constexpr int SIDES = sides(G), PJ = (G + SIDES - 1) / SIDES, COLS = 16 / SIDES;
    const int tid = threadIdx.x, lp = __builtin_ctz(s.page), mask = s.page - 1;
    const long long items = 2LL * n * s.n_layers * s.n_kv_heads, all = (items + 7) / 8 * 8 * SIDES;
    for (long long b = blockIdx.x; b < all; b += gridDim.x) {
        // (workgroups that share lines are eight apart, on one XCD)
        const int side = (int)(b / 8 % SIDES);
        const long long it = b / (8 * SIDES) * 8 + b % 8, list = it / 2;
        const bool keys = it % 2 == 0;
        if (it >= items) continue;
        const int h = (int)(list % s.n_kv_heads), layer = (int)(list / s.n_kv_heads % s.n_layers);
        const int i = (int)(list / s.n_kv_heads / s.n_layers);
        if (w.need[i] < 0) continue;
        const int *stay = w.stay + (size_t)list * keep;
        const int *from = w.from + (size_t)i * w.fb, *to = w.to + (size_t)i * w.tb;
        uint8_t *base = (uint8_t *)(keys ? p.k : p.v) + ((size_t)layer * s.n_pages * s.n_kv_heads + h) * f.block;
        const size_t page = s.n_kv_heads * f.block;
        const int q = seqs[i];
        float *wrow = weights + mhip_q4::weights_row(s, layer, q, h);
        if (keys && h == 0 && layer == 0 && side == 0 && tid == 0) p.len[q] = keep;
        const int whole = (keep + 3) & ~3;  // (past the end, in a four that is not whole: the token that is there)
        auto look = [&](Chunk &c, int r0) {
            bool moves = false;
            if (tid < CHUNK && r0 + tid < whole) {
                const int r = r0 + tid, a = r < keep ? stay[r] : r, will = to[r >> lp];
                const int is = r < keep ? from[a >> lp] : will;
                c.from[tid] = is;
                c.to[tid] = will;
                c.at[tid] = a & mask;
                moves = a != r || is != will;
            }
            moves = __any(moves);
            if ((tid & 63) == 0) c.moves[tid >> 6] = moves;
        };
        int now = 0;
        look(d[0], 0);
        __syncthreads();
        // A turn reads a chunk and finds out what the next one is while that is on its way. Behind the
        // barrier everyone has read this chunk, so it can be written; the next one's
        // tokens are all behind it. (Three descriptions, as this one's is still in use then.)
        for (int r0 = 0; r0 < keep; r0 += CHUNK) {
            const Chunk &c = d[now];
            now = now == 2 ? 0 : now + 1;
            const int m = min(CHUNK, keep - r0);
            bool moves = false;
#pragma unroll
            for (int e = 0; e < MOVE / 64; e++) moves |= c.moves[e] != 0;
            constexpr int P = (CHUNK * PJ + MOVE - 1) / MOVE, W = (CHUNK / 4 * COLS * G + MOVE - 1) / MOVE;
            _Float16 sc[P], lo[P];
            float wt = 0.0f;
            if (keys) {
                uint4 code[P];
                if (moves) {
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        const int x = tid + e * MOVE, t = x / PJ, j = x % PJ * SIDES + side;
                        if (t < m && j < G) {
                            const uint8_t *b = base + c.from[t] * page;
                            const int at = c.at[t];
                            code[e] = *(const uint4 *)(b + mhip_q4::key_word(f, at, 0, 0) + j * 16);
                            sc[e] = *(const _Float16 *)(b + mhip_q4::scale_at(f, at, j));
                            lo[e] = *(const _Float16 *)(b + mhip_q4::low_at(f, true, at, j));
                        }
                    }
                    if (side == 0 && tid < m) wt = wrow[stay[r0 + tid]];
                }
                look(d[now], r0 + CHUNK);
                all_read();
                if (moves) {
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        const int x = tid + e * MOVE, t = x / PJ, j = x % PJ * SIDES + side;
                        if (t < m && j < G) {
                            uint8_t *b = base + c.to[t] * page;
                            const int at = (r0 + t) & mask;
                            *(uint4 *)(b + mhip_q4::key_word(f, at, 0, 0) + j * 16) = code[e];
                            *(_Float16 *)(b + mhip_q4::scale_at(f, at, j)) = sc[e];
                            *(_Float16 *)(b + mhip_q4::low_at(f, true, at, j)) = lo[e];
                        }
                    }
                    if (side == 0 && tid < m) wrow[r0 + tid] = wt;
                }
            } else {
                uint8_t code[W][4];  // (of a word of the destination: a byte of each of its four tokens)
                if (moves) {
#pragma unroll
                    for (int e = 0; e < W; e++) {
                        const int x = tid + e * MOVE, four = x / (COLS * G), cj = x % (COLS * G) + side * COLS * G;
                        if (four * 4 < m) {
#pragma unroll
                            for (int y = 0; y < 4; y++) {
                                const int t = four * 4 + y;
                                code[e][y] = base[c.from[t] * page + mhip_q4::value_byte(f, c.at[t], cj / G, cj % G)];
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        const int x = tid + e * MOVE, t = x / PJ, j = x % PJ * SIDES + side;
                        if (t < m && j < G) {
                            const uint8_t *b = base + c.from[t] * page;
                            sc[e] = *(const _Float16 *)(b + mhip_q4::scale_at(f, c.at[t], j));
                            lo[e] = *(const _Float16 *)(b + mhip_q4::low_at(f, false, c.at[t], j));
                        }
                    }
                }
                look(d[now], r0 + CHUNK);
                all_read();
                if (moves) {
#pragma unroll
                    for (int e = 0; e < W; e++) {
                        const int x = tid + e * MOVE, four = x / (COLS * G), cj = x % (COLS * G) + side * COLS * G;
                        if (four * 4 < m) {
                            const int at = (r0 + four * 4) & mask;
                            // (tokens 0, 2, 1, 3: cache_q4.h)
                            const unsigned word = code[e][0] | code[e][2] << 8 | code[e][1] << 16 | (unsigned)code[e][3] << 24;
                            *(unsigned *)(base + c.to[four * 4] * page + mhip_q4::value_byte(f, at, cj / G, cj % G)) = word;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        const int x = tid + e * MOVE, t = x / PJ, j = x % PJ * SIDES + side;
                        if (t < m && j < G) {
                            uint8_t *b = base + c.to[t] * page;
                            const int at = (r0 + t) & mask;
                            *(_Float16 *)(b + mhip_q4::scale_at(f, at, j)) = sc[e];
                            *(_Float16 *)(b + mhip_q4::low_at(f, false, at, j)) = lo[e];
                        }
                    }
                }
            }
        }
        __syncthreads();  // (the descriptions, for the next item)
    }
}

bool shape_ok(const mhip_page_dims *s, int n, int keep, int recent, int max_len) {
    return s->type == MHIP_Q4 && n >= 1 && n <= s->max_seqs && keep >= 1 && recent >= 0 && recent <= keep &&
           max_len >= 0 && max_len <= (long long)s->max_blocks * s->page &&
           (double)n * s->n_layers * s->n_kv_heads * keep < 0x1p58;  // (a workspace of less than 2^60 bytes)
}

template <int G>
void move(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, float *weights, const int *seqs, int n, int keep,
          const Work &w) {
    const long long all = (2LL * n * s->n_layers * s->n_kv_heads + 7) / 8 * 8 * sides(G);
    k_evict_move<G><<<(unsigned)(all < 1 << 20 ? all : 1 << 20), MOVE, 0, c->stream>>>(*s, *p, weights, seqs, n,
                                                                                         keep, w);
}

}  // namespace

extern "C" {

size_t mhip_pages_evict_ws_bytes(const mhip_page_dims *s, int n, int keep, int max_len) {
    if (!mhip_pages_plan_bytes(s) || !shape_ok(s, n, keep, 0, max_len)) return 0;
    return work_of(s, n, keep, max_len, nullptr).bytes;
}

int mhip_pages_evict(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, float *d_weights, const int *d_seqs,
                     int n, int keep, int recent, int max_len, void *d_ws) {
    const char *what = "pages evict";
    if (mhip::check_pages(c, s, p, what) || mhip::check_list(c, s, d_seqs, n, what)) return -1;
    if (s->type != MHIP_Q4) return mhip::fail(c, "%s: a cache of type %d is not in 4 bits", what, s->type);
    if (!shape_ok(s, n ? n : 1, keep, recent, max_len))
        return mhip::fail(c, "%s: %d tokens stay, %d of them the last, slots of up to %d", what, keep, recent, max_len);
    if (!n) return 0;
    if (!d_weights || !d_ws) return mhip::fail(c, "%s: a null argument", what);
    if ((uintptr_t)d_weights % 16 || (uintptr_t)d_ws % 256)
        return mhip::fail(c, "%s: the weights must start on 16 bytes, the workspace on 256", what);
    if (mhip::use_device(c)) return -1;
    const Work w = work_of(s, n, keep, max_len, d_ws);
    const long long items = (long long)n * s->n_layers * s->n_kv_heads;
    k_evict_begin<<<(unsigned)(items < 1 << 20 ? items : 1 << 20) + 1, SEL, 0, c->stream>>>(
        *s, *p, d_weights, d_seqs, n, keep, recent, max_len, w);
    switch (s->head_dim / 32) {
        case 1: move<1>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 2: move<2>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 3: move<3>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 4: move<4>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 5: move<5>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 6: move<6>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        case 7: move<7>(c, s, p, d_weights, d_seqs, n, keep, w); break;
        default: move<8>(c, s, p, d_weights, d_seqs, n, keep, w); break;
    }
    return mhip::check_launch(c, what);
}

}  // extern "C"
