// What the translation units of the shared-prefix attention exchange: the
// arguments of a call and how it is cut (attn_shared.hip), one unit per
// element type (attn_shared_*.hip, from attn_shared.inc).
#pragma once

#include "mhip_internal.h"

namespace mhip_shared {

constexpr int NT = 256, TILE = 64;
constexpr int PART_MAX = 4096;               // positions of a part
constexpr int PART_PAGES = PART_MAX / 16 + 2;

// The arguments of one call.
struct Job {
    mhip_page_dims s;
    mhip_pages p;
    int layer, nh, group;          // query heads, and per key/value head
    const void *q;
    size_t ldq;
    void *out;
    size_t ldo;
    const int *seqs, *count;
    int n, mc;                     // entries, tokens of each at most
    int prefix_seq, prefix, max_len;
    float c;                       // scale * log2(e)
    int lp;                        // log2(page)
    int sp, plen, ptiles;          // prefix parts, positions of each, row tiles
    int ss, slen, stiles;          // parts behind the prefix, positions of each, row tiles of a slot
    float *o, *ml;                 // partial results [part][row][hd], [part][row][2]
};

// How a call is cut: rows of a prefix tile (wr * rt tiles of 16), parts of the
// prefix and of the slots.
struct Cut {
    int wr, rt, ptiles, sp, plen, ss, slen, stiles;
};

int launch_f32(mhip_ctx *c, const Job &a, const Cut &k);
int launch_f16(mhip_ctx *c, const Job &a, const Cut &k);
int launch_bf16(mhip_ctx *c, const Job &a, const Cut &k);

}  // namespace mhip_shared
