// Where the bytes of a cache in 4 bits are (include/mia_hip.h, mhip_pages): the
// block of one layer, page and head.
//
// A value is s c + m with a code c of 0 .. 15; s and m in fp16 for 32 values of a
// token. The orders are those in which the matrix cores take their operands
// (attn_q4.inc), so that a lane's codes of a tile are one run of bytes and need no
// exchange with other lanes:
//   keys   (a token is a row of the operand, a lane group has 8 of 32 elements):
//     codes  words [page][4 g][G j], elements 32 j + 8 g .. + 7; element 2 i in nibble i,
//            2 i + 1 in nibble i + 4, which are neighbours as fp16 pairs
//     s      [page / 4][G j][4], as a lane has the scores of four tokens
//     m      [page][G j], an operand by itself
//   values (an element is a row, a lane has four tokens of it):
//     codes  bytes [page / 4][16 c][G j][4]: element 32 j + 2 c in the low, the next one in the
//            high half; tokens 0, 2, 1, 3, which makes tokens 0 and 1 an fp16 pair
//     s, m   [page / 4][G j][4] each
#pragma once

#include "mhip_internal.h"

namespace mhip_q4 {

constexpr int GROUP = 32;            // values that share s and m
constexpr float MOST = 32768.0f;     // values are kept within +-2^15, so that s c + m is an fp16 value

struct Shape {
    int page, hd, G;                 // tokens of a page, head_dim, groups of 32 of a row
    size_t block;                    // bytes
    unsigned scale, low;             // offsets of s and m in a block
};
__host__ __device__ inline Shape shape_of(const mhip_page_dims &s) {
    Shape r;
    r.page = s.page;
    r.hd = s.head_dim;
    r.G = s.head_dim / GROUP;
    r.block = mhip::q4_block(s);
    r.scale = (unsigned)(s.page * s.head_dim / 2);
    r.low = r.scale + (unsigned)(s.page * s.head_dim / 16);
    return r;
}

// Offsets in a block, of token t of the page: the word of keys' elements 32 j + 8 g .. + 7,
// the byte of values' 32 j + 2 c and + 1, and s and m of group j.
__host__ __device__ inline unsigned key_word(const Shape &f, int t, int g, int j) {
    return (unsigned)((t * 4 + g) * f.G + j) * 4;
}
__host__ __device__ inline unsigned value_byte(const Shape &f, int t, int c, int j) {
    return (unsigned)(((t >> 2) * 16 + c) * f.G + j) * 4 + (((t & 1) << 1) | ((t >> 1) & 1));
}
__host__ __device__ inline unsigned by_four(const Shape &f, int t, int j) {
    return (unsigned)(((t >> 2) * f.G + j) * 4 + (t & 3)) * 2;
}
__host__ __device__ inline unsigned scale_at(const Shape &f, int t, int j) { return f.scale + by_four(f, t, j); }
__host__ __device__ inline unsigned low_at(const Shape &f, bool keys, int t, int j) {
    return f.low + (keys ? (unsigned)(t * f.G + j) * 2 : by_four(f, t, j));
}

// The weights that attention adds up: [layer][slot][head][max_blocks * page].
__host__ __device__ inline size_t weights_row(const mhip_page_dims &s, int layer, int slot, int head) {
    return (((size_t)layer * s.max_seqs + slot) * s.n_kv_heads + head) * ((size_t)s.max_blocks * s.page);
}

}  // namespace mhip_q4
