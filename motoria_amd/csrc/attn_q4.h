// What the translation units of the attention over a cache in 4 bits exchange: the
// arguments of a call and how it is cut (attn_q4.hip), one unit per type of the
// rows (attn_q4_*.hip, from attn_q4.inc).
#pragma once

#include "cache_q4.h"

namespace mhip_q4 {

constexpr int NT = 256, WAVES = 4;
constexpr int TILE = 32;                 // positions that a wavefront works on at a time
constexpr int PART_MAX = 4096;           // positions whose pages are in LDS at a time
constexpr int PART_PAGES = PART_MAX / 16 + 2;
constexpr int ITEMS_MAX = 512;           // items of a call that is cut into parts
constexpr int SUM_EACH = 4;              // tiles of a wavefront that adds weights up from new scores
constexpr int SUM_TILES = SUM_EACH * WAVES;

// What is kept of a row and part: the reference of its weights, their sum (of a whole
// row: one over it), the factor of its scores (scale * log2(e), less the
// powers of two that its queries were taken by), and the positions that it sees.
struct alignas(16) Stat {
    float m, l, c;
    int sees;
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
    int tiles;                           // row tiles of an entry (each an item)
    int wgs, least;                      // parts wanted (0: a workgroup an item), steps of one at least
    float *o;                            // partial results [part][head][row of the tile][hd]
    Stat *part;                          // [part][head][row of the tile]
    Stat *row;                           // [row]: of all parts
    int *start;                          // the parts before each item, and all of them
    float *weights;
    int wparts, wlen;                    // workgroups of a slot and head that add them up, positions of each
    int wsides;                          // wavefronts of one that share its positions and take rows in turn
    float *kept;                         // scores of a call with up to 16 rows a slot and head, or null
    size_t keep_step;                    // of one slot and head
};

// How a call is cut; nq: tiles of 16 rows of a workgroup.
struct Cut {
    int nq, tiles, wgs, wparts, wlen, wsides;
};


// Tiles of 16 rows of a workgroup that has more than one: two share a tile's codes and s (a chunk of 500
// tokens over 6000, 32 heads over 4 of 128: bf16 152 us with two, 182 with one, fp32 159 and 192). With heads
// of more than 128 elements two take more registers than half of a SIMD's, and half as many workgroups: 8 heads over 2
// of 256 98 us with one, 102 with two; with more of them two would be faster (16 heads 153, with one 191).
constexpr int wide_tiles(int groups) { return groups > 4 ? 1 : 2; }

int launch_f32(mhip_ctx *c, const Job &a, const Cut &k);
int launch_f16(mhip_ctx *c, const Job &a, const Cut &k);
int launch_bf16(mhip_ctx *c, const Job &a, const Cut &k);

}  // namespace mhip_q4
