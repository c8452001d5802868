// How a call on the pages of a cache decides which page goes where: one
// workgroup, a scan over the counts of references, all of a call or nothing
// (pages.hip, evict.hip).
#pragma once

#include "mhip_internal.h"

namespace {

constexpr int NT = 256;                  // a deciding workgroup: barriers of four wavefronts cost
                                         // 1.5 us less than those of sixteen (extend 7.2 -> 5.6)
constexpr int MOST_THREADS = 512;        // of a workgroup that decides beside others' work (evict.hip)
constexpr int PER = 8;                   // pages a thread looks at per round of a scan
constexpr int SEQ_WORDS = 65536 / 32;    // one bit per slot
enum { ST_BITS = 0, ST_HINT = 1, ST_FREE = 2 };  // words of mhip_pages.state
enum { PL_PAIRS = 0, PL_OK = mhip::PLAN_OK, PL_HEAD = 16 };  // words of mhip_pages.plan

// The plan: [PL_HEAD] words, then per page the source, destination and rows of
// a copy and the page's new index, then per list entry the pages before its own.
struct Plan {
    int *head, *src, *dst, *rows, *map, *first;
};
__host__ __device__ inline Plan plan_of(int *p, int n_pages) {
    Plan r;
    r.head = p;
    r.src = p + PL_HEAD;
    r.dst = r.src + n_pages;
    r.rows = r.dst + n_pages;
    r.map = r.rows + n_pages;
    r.first = r.map + n_pages;
    return r;
}

// Exclusive prefix sum of v over the workgroup; total in every thread.
// (Sums of at most n_pages or max_seqs * max_blocks: 64 bits for the latter.)
template <int N>
__device__ long long scan(long long v, long long *total, long long *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long s = v;
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < N / 64; w++) {
        const long long x = lds[w];
        before += w < wave ? x : 0;
        all += x;
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

__device__ inline int blocks_of(int tokens, int page) { return (tokens + page - 1) / page; }

// LDS of a workgroup that decides. Its loads depend on each other (entry,
// length, pages), at about 0.7 us a level, so what can be asked for early is, and
// lists of up to NT entries and pages stay here.
struct Desk {
    unsigned seen[SEQ_WORDS];
    long long sums[MOST_THREADS / 64];
    int first[NT], list[NT], slot[NT], len[NT];
    int bad;
};

// Which of this thread's PER pages from `base` on are free.
__device__ unsigned free_mask(const mhip_page_dims &s, const mhip_pages &p, int base) {
    const int at = base + threadIdx.x * PER;
    unsigned is = 0;
#pragma unroll
    for (int j = 0; j < PER; j++)
        if (at + j < s.n_pages && p.refs[at + j] <= 0) is |= 1u << j;
    return is;
}

// The first `want` free pages in ascending order into out[]; whether there
// are as many. Every page below `from` (the hint) is in use; is: free_mask there.
template <int N>
__device__ bool take_free(const mhip_page_dims &s, const mhip_pages &p, int want, int *out, int from,
                          unsigned is, long long *sums) {
    int got = 0;
    for (int base = from; base < s.n_pages && got < want; base += N * PER) {
        const int at = base + threadIdx.x * PER;
        if (base != from) is = free_mask(s, p, base);
        long long all;
        int r = got + (int)scan<N>(__popc(is), &all, sums);
        for (int j = 0; j < PER; j++)
            if (is >> j & 1) {
                if (r < want) out[r] = at + j;
                r++;
            }
        got = min(want, got + (int)all);
    }
    __syncthreads();  // out[] is written
    return got == want;
}

// The entry whose pages page number x of the call belongs to.
__device__ inline int entry_of(const int *first, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (first[m] <= x) lo = m;
        else hi = m - 1;
    }
    return lo;
}

// What a call over n entries needs: need(i, bad) pages for entry i (and error
// bits). Takes the pages (list[]) if nothing is wrong, with the prefix sums of the
// needs in first[]. Returns their number, or -1 with the error bits set.
// late(i): whether entry i is wrong now that all have been looked at.
template <int N = NT, class F, class L>
__device__ int decide(const mhip_page_dims &s, const mhip_pages &p, Desk &d, int n, int *&first,
                      int *&list, F need, L late) {
    const Plan pl = plan_of(p.plan, s.n_pages);
    const int from = max(0, min(p.state[ST_HINT], s.n_pages));
    const unsigned is = free_mask(s, p, from);
    for (int i = threadIdx.x; i < (s.max_seqs + 31) / 32; i += N) d.seen[i] = 0;
    if (threadIdx.x == 0) d.bad = 0;
    __syncthreads();
    first = n <= NT ? d.first : pl.first;
    long long run = 0;
    for (int base = 0; base < n; base += N) {
        const int i = base + threadIdx.x;
        long long all;
        int bad = 0;
        const long long mine = i < n ? need(i, bad) : 0;
        if (bad) atomicOr(&d.bad, bad);
        const long long x = scan<N>(bad ? 0 : mine, &all, d.sums);
        if (i < n) first[i] = (int)min(run + x, (long long)1 << 30);
        run += all;
    }
    for (int i = threadIdx.x; i < n; i += N)
        if (late(i)) atomicOr(&d.bad, MHIP_PAGES_BAD);
    __syncthreads();
    int err = d.bad;
    list = run <= NT ? d.list : pl.dst;
    if (!err && (run > s.n_pages || !take_free<N>(s, p, (int)run, list, from, is, d.sums)))
        err = MHIP_PAGES_NO_SPACE;
    if (err && threadIdx.x == 0) atomicOr(&p.state[ST_BITS], err);
    return err ? -1 : (int)run;
}

// Marks slot q as named by the list; whether it was already.
__device__ inline bool mark(Desk &d, int q) {
    return atomicOr(&d.seen[q >> 5], 1u << (q & 31)) >> (q & 31) & 1;
}

}  // namespace
