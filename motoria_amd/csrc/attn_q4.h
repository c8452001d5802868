// What the translation units of the attention over a cache in 4 bits exchange: the
// arguments of a call and how it is cut (attn_q4.hip), one unit per type of the
// rows (attn_q4_*.hip, from attn_q4.inc).
#pragma once

#include "cache_q4.h"

namespace mhip_q4 {

constexpr int NT = 256, WAVES = 4;
constexpr int TILE = 32;                 // positions that a wavefront works on at a time
constexpr int PART_MAX = 4096;           // positions of a part
constexpr int PART_PAGES = PART_MAX / 16 + 2;
constexpr int SUM_MAX = 1024;            // positions of a workgroup that adds weights up

// What is kept of a row and part: the reference of its weights, their sum, and the factor
// of its scores (scale * log2(e), less the power of two that its queries were taken by).
struct Stat {
    float m, l, c, none;
};

// The arguments of one call.
struct Job {
    mhip_page_dims s;
    mhip_pages p;
    int layer, nh, group;                // query heads, and per key/value head
    const void *q;
    size_t ldq;
    void *out;
    size_t ldo;
    const int *seqs, *count;
    int n, mc, max_len;                  // entries, tokens of each at most, positions
    float c;                             // scale * log2(e)
    int lp;                              // log2(page)
    int parts, plen, tiles;              // parts of a slot, positions of each, row tiles of a slot
    float *o;                            // partial results [part][row][hd]
    Stat *part;                          // [part][row]
    Stat *row;                           // [row]: of all parts
    float *weights;
    int wparts, wlen;                    // the same for the weights
};

// How a call is cut; nq: tiles of 16 rows of a workgroup.
struct Cut {
    int nq, tiles, parts, plen, wparts, wlen;
};

// Tiles of 16 rows of a workgroup that has more than one.
constexpr int wide_tiles(bool f32, int groups) { return f32 ? (groups > 4 ? 1 : 2) : groups > 4 ? 2 : 4; }

int launch_f32(mhip_ctx *c, const Job &a, const Cut &k);
int launch_f16(mhip_ctx *c, const Job &a, const Cut &k);
int launch_bf16(mhip_ctx *c, const Job &a, const Cut &k);

}  // namespace mhip_q4
