// Rows into and out of a cache in 4 bits (include/mia_hip.h; the layout:
// cache_q4.h), and the accumulated weights of a forked slot.
//
// For 32 values x of a token: lo and hi their least and greatest, m = fp16(lo),
// s = fp16((hi - m) / 15) with an fp32 difference and quotient, and
//   c = how many k of 0 .. 14 have x - m >= (k + 1/2) s   (0 where s is 0).
// The nearest code is estimated in fp32; where the estimate is within 2^-16 of a border
// (its own error is below 2^-17) the comparison is made in 64 bits, in which (k + 1/2) s is exact
// and x - m is rounded once (exact unless x and m are more than 2^29 apart in size). That difference is the
// definition's, so a code does not depend on how it was found.
//
// A thread has eight values of a token, or of four tokens that lie in a word of values' codes
// (whose bytes are four tokens', and s and m the same): with a byte and two a store, prompts of
// 7 slots of up to 1900 tokens (8 heads of 64, fp16: 13.7 MB in and out again) took 16.6 us to write and
// 11.3 to read, with fours 12.5 and 8.6, of which a copy of the bytes would be 3.7 each. What is left
// is instructions (5 us of the write) and the chain of slot, length, page and values at its
// start. Calls of few tokens are bound by that chain and the launch: 64 slots of one token 3.6 and 3.2 us.
#include "cache_q4.h"

namespace {

using mhip_q4::Shape;

__device__ inline float value(float x) { return x; }
__device__ inline float value(_Float16 x) { return (float)x; }
__device__ inline float value(__bf16 x) { return (float)x; }

// The codes of eight values.
__device__ __forceinline__ void codes_of(const float (&x)[8], float m, float s, unsigned (&c)[8]) {
    const float inv = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;  // (within 2^-23 of 1 / s)
    float near = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float at = __builtin_fmaf(x[e] - m, inv, 0.5f);
        c[e] = (unsigned)__builtin_amdgcn_fmed3f(at, 0.0f, 15.0f);
        near = fmaxf(near, fabsf(__builtin_amdgcn_fractf(at) - 0.5f));
    }
    if (near <= 0.5f - 0x1p-16f) return;
    const double step = (double)s;
    if (s > 0.0f)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double d = (double)x[e] - (double)m;
            const int up = d >= (c[e] + 0.5) * step, down = d < (c[e] - 0.5) * step;
            c[e] = (unsigned)min(max((int)c[e] + up - down, 0), 15);
        }
}

// The value of another of four neighbouring lanes.
template <int P> __device__ __forceinline__ float beside(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), P, 0xf, 0xf, true));
}

// Tokens t0 .. t0 + TOK - 1 of a page that a thread takes together (four on a multiple of four, or
// one), which of them are in the call, and the first one's row; false where none can be done. `bad`:
// some are in the call but have no place.
template <int TOK> struct Tokens {
    int page, t0, slot, pos, row;
    bool in[TOK];
};
template <int TOK>
__device__ inline bool tokens_of(const mhip_page_dims &s, const mhip_pages &p, const int *seqs, const int *count,
                                 unsigned unit, int max_count, Tokens<TOK> &k, bool &bad) {
    const int each = TOK == 1 ? max_count : (max_count + 6) / 4;
    const int i = each == 1 ? unit : unit / each, j = each == 1 ? 0 : unit % each;
    const int q = seqs[i], m = count ? max(count[i], 0) : max_count;
    const int lp = __builtin_ctz(s.page);
    const bool is = (unsigned)q < (unsigned)s.max_seqs && m <= max_count;
    const int first = is ? p.len[q] - m : 0;  // of the call's positions; below 0 there is none
    const int pos = (TOK == 1 ? first : first & ~3) + j * TOK;
    bool any = false;
    bad = false;
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        const bool of = pos + t >= first && pos + t - first < m;
        k.in[t] = is && of && pos + t >= 0;
        any |= k.in[t];
        bad |= of && !k.in[t];
    }
    k.page = any && pos >> lp < s.max_blocks ? p.table[(size_t)q * s.max_blocks + (pos >> lp)] : -1;
    if ((unsigned)k.page >= (unsigned)s.n_pages) {
        bad |= any;
        any = false;
    }
    k.t0 = pos & (s.page - 1);
    k.slot = q;
    k.pos = pos;
    k.row = i * max_count + pos - first;
    return any;
}

// A thread has eight values of a row, four neighbours a group of 32 (keys'
// threads, then values'): gridDim.y workgroups share a row (or four rows), or one takes several.
struct Place {
    unsigned unit, x;
    bool is;
};
__device__ inline Place place_of(unsigned pieces, int units, int each) {
    Place r;
    if (each > 1) {
        const unsigned in = threadIdx.x / pieces;
        r.unit = blockIdx.x * each + in;
        r.x = threadIdx.x - in * pieces;
        r.is = in < (unsigned)each && r.unit < (unsigned)units;
    } else {
        r.unit = blockIdx.x;
        r.x = blockIdx.y * 256 + threadIdx.x;
        r.is = r.x < pieces;
    }
    return r;
}

typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));

template <class T, int TOK>
__global__ __launch_bounds__(256) void k_write_q4(mhip_page_dims s, mhip_pages p, int layer, const int *seqs,
                                                  const int *count, int units, int max_count, const T *k,
                                                  const T *v, size_t ld, float *weights, int each) {
    const Shape f = mhip_q4::shape_of(s);
    const unsigned half = (unsigned)s.n_kv_heads * f.G * 4;
    const Place at = place_of(2 * half, units, each);
    if (!at.is) return;
    const bool keys = at.x < half;
    const unsigned y = keys ? at.x : at.x - half;
    const int h = y / (f.G * 4), j = y / 4 % f.G, g = y & 3;
    const T *from = (keys ? k : v) + (size_t)y * 8;
    uint4 raw[TOK][sizeof(T) / 2];
    // (one token's row is known without its place: its values are on their way meanwhile)
    if (TOK == 1)
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; e++) raw[0][e] = ((const uint4 *)(from + (size_t)at.unit * ld))[e];
    Tokens<TOK> tok;
    bool bad;
    const bool some = tokens_of<TOK>(s, p, seqs, count, at.unit, max_count, tok, bad);
    if (bad && at.x == 0) atomicOr(&p.state[0], MHIP_PAGES_BAD);
    if (!some) return;
    if (TOK > 1)
#pragma unroll
        for (int t = 0; t < TOK; t++)
#pragma unroll
            for (int e = 0; e < (int)sizeof(T) / 2; e++)
                raw[t][e] = tok.in[t] ? ((const uint4 *)(from + (size_t)(tok.row + t) * ld))[e] : uint4{0, 0, 0, 0};
    uint8_t *to = (uint8_t *)(keys ? p.k : p.v) +
                  (((size_t)layer * s.n_pages + tok.page) * s.n_kv_heads + h) * f.block;
    bool odd = false, all = true;
    unsigned byte[4] = {};  // of each pair of values, its tokens'
    u16x4 scale, low;
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        float x[8];
        unsigned most = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = value(((const T *)raw[t])[e]);
            most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
        }
        if (most > __float_as_uint(mhip_q4::MOST)) {  // (an infinity's or NaN's bits are more, too)
            odd = true;
#pragma unroll
            for (int e = 0; e < 8; e++)
                x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -mhip_q4::MOST), mhip_q4::MOST);
        }
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) {
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
        lo = fminf(lo, beside<0xb1>(lo));  // one lane on or back, then two
        hi = fmaxf(hi, beside<0xb1>(hi));
        lo = fminf(lo, beside<0x4e>(lo));
        hi = fmaxf(hi, beside<0x4e>(hi));
        const float m = (float)(_Float16)lo + 0.0f;  // (-0 as 0: which zero of several is least is not defined)
        const float width = fmaxf(hi - m, 0.0f) + 0.0f;  // (m may round to more than hi)
        // width / 15, rounded once: a quotient within an ulp, and its exact remainder times a correctly
        // rounded reciprocal (Markstein's theorem; where the remainder is too small to be exact, s is 0)
        const float guess = width * (1.0f / 15.0f);
        float step = __builtin_fmaf(__builtin_fmaf(-15.0f, guess, width), 1.0f / 15.0f, guess);
        asm("" : "+v"(step));  // (rounded to fp32 before it is to fp16: one instruction would do both at once)
        const _Float16 sh = (_Float16)step;
        unsigned c[8], w = 0;
        codes_of(x, m, (float)sh, c);
#pragma unroll
        for (int e = 0; e < 8; e++) w |= c[e] << (4 * (e / 2 + 4 * (e & 1)));
#pragma unroll
        for (int e = 0; e < 4; e++) byte[e] |= (c[2 * e] | c[2 * e + 1] << 4) << 8 * ((t & 1) << 1 | t >> 1);
        scale[t] = __builtin_bit_cast(unsigned short, sh);
        low[t] = __builtin_bit_cast(unsigned short, (_Float16)m);
        all &= tok.in[t];
        if (keys && tok.in[t]) {
            *(unsigned *)(to + mhip_q4::key_word(f, tok.t0 + t, g, j)) = w;
            if (g == 0) *(unsigned short *)(to + mhip_q4::low_at(f, true, tok.t0 + t, j)) = low[t];
            if (weights && g == 0 && j == 0)
                weights[mhip_q4::weights_row(s, layer, tok.slot, h) + tok.pos + t] = 0.0f;
        }
    }
    if (odd) atomicOr(&p.state[0], MHIP_PAGES_NOT_FINITE);
    if (TOK == 4 && all) {
        if (!keys)
#pragma unroll
            for (int e = 0; e < 4; e++) *(unsigned *)(to + mhip_q4::value_byte(f, tok.t0, 4 * g + e, j)) = byte[e];
        if (g == 0) *(u16x4 *)(to + mhip_q4::scale_at(f, tok.t0, j)) = scale;
        if (g == 0 && !keys) *(u16x4 *)(to + mhip_q4::low_at(f, false, tok.t0, j)) = low;
        return;
    }
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        if (!tok.in[t]) continue;
        if (!keys)
#pragma unroll
            for (int e = 0; e < 4; e++)
                to[mhip_q4::value_byte(f, tok.t0 + t, 4 * g + e, j)] = (uint8_t)(byte[e] >> 8 * ((t & 1) << 1 | t >> 1));
        if (g == 0) *(unsigned short *)(to + mhip_q4::scale_at(f, tok.t0 + t, j)) = scale[t];
        if (g == 0 && !keys) *(unsigned short *)(to + mhip_q4::low_at(f, false, tok.t0 + t, j)) = low[t];
    }
}

template <class T, int TOK>
__global__ __launch_bounds__(256) void k_read_q4(mhip_page_dims s, mhip_pages p, int layer, const int *seqs,
                                                 const int *count, int units, int max_count, T *k, T *v,
                                                 size_t ld, int each) {
    const Shape f = mhip_q4::shape_of(s);
    const unsigned half = (unsigned)s.n_kv_heads * f.G * 4;
    const Place at = place_of(2 * half, units, each);
    if (!at.is) return;
    const bool keys = at.x < half;
    const unsigned y = keys ? at.x : at.x - half;
    const int h = y / (f.G * 4), j = y / 4 % f.G, g = y & 3;
    Tokens<TOK> tok;
    bool bad;
    const bool some = tokens_of<TOK>(s, p, seqs, count, at.unit, max_count, tok, bad);
    if (bad && at.x == 0) atomicOr(&p.state[0], MHIP_PAGES_BAD);
    if (!some) return;
    const uint8_t *from = (const uint8_t *)(keys ? p.k : p.v) +
                          (((size_t)layer * s.n_pages + tok.page) * s.n_kv_heads + h) * f.block;
    // (a page's words are there whether all of their tokens are or not)
    unsigned w[4];
    unsigned short scale[TOK], low[TOK];
#pragma unroll
    for (int t = 0; t < TOK; t++) low[t] = *(const unsigned short *)(from + mhip_q4::low_at(f, keys, tok.t0 + t, j));
    if constexpr (TOK == 4) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = *(const unsigned *)(from + (keys ? mhip_q4::key_word(f, tok.t0 + e, g, j)
                                                    : mhip_q4::value_byte(f, tok.t0, 4 * g + e, j)));
        *(u16x4 *)scale = *(const u16x4 *)(from + mhip_q4::scale_at(f, tok.t0, j));
    } else {
        scale[0] = *(const unsigned short *)(from + mhip_q4::scale_at(f, tok.t0, j));
        if (keys) w[0] = *(const unsigned *)(from + mhip_q4::key_word(f, tok.t0, g, j));
        else
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = from[mhip_q4::value_byte(f, tok.t0, 4 * g + e, j)];
    }
    T *to = (keys ? k : v) + (size_t)y * 8;
#pragma unroll
    for (int t = 0; t < TOK; t++) {
        const float st = (float)__builtin_bit_cast(_Float16, scale[t]), m = (float)__builtin_bit_cast(_Float16, low[t]);
        // a token's codes a byte each, in the order that keys' word has: 0, 4, 1, 5 and 2, 6, 3, 7
        unsigned some4 = w[t], more = w[t] >> 4;
        if (!keys) {
            const unsigned pick = 0x0c0c0400u + (unsigned)((t & 1) << 1 | t >> 1) * 0x101u;  // (0c: a 0)
            const unsigned all8 = TOK == 1 ? w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24
                                           : __builtin_amdgcn_perm(w[1], w[0], pick) | __builtin_amdgcn_perm(w[3], w[2], pick) << 16;
            const unsigned even = all8, uneven = all8 >> 4;
            some4 = __builtin_amdgcn_perm(uneven, even, 0x06040200u);
            more = __builtin_amdgcn_perm(uneven, even, 0x07050301u);
        }
        some4 &= 0x0f0f0f0fu;
        more &= 0x0f0f0f0fu;
        T r[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const unsigned c = (e & 2 ? more : some4) >> 8 * ((e & 1) << 1 | e >> 2) & 0xff;
            r[e] = (T)(st * (float)c + m);  // (the product is exact)
        }
        if (!tok.in[t]) continue;
#pragma unroll
        for (int e = 0; e < (int)sizeof(T) / 2; e++) ((uint4 *)(to + (size_t)(tok.row + t) * ld))[e] = ((uint4 *)r)[e];
    }
}

// The children's weights, once their fork is known to have been done: a
// workgroup takes rows of one entry, layer and head.
__global__ __launch_bounds__(256) void k_fork_weights(mhip_page_dims s, mhip_pages p, float *weights,
                                                      const int *src, const int *dst, int n, const int *ok) {
    if (!*ok) return;
    const long long items = (long long)n * s.n_layers * s.n_kv_heads;
    for (long long it = blockIdx.x; it < items; it += gridDim.x) {
        const int h = (int)(it % s.n_kv_heads), layer = (int)(it / s.n_kv_heads % s.n_layers);
        const int i = (int)(it / s.n_kv_heads / s.n_layers), a = src[i], b = dst[i], len = p.len[b];
        const float *from = weights + mhip_q4::weights_row(s, layer, a, h);
        float *to = weights + mhip_q4::weights_row(s, layer, b, h);
        for (int x = threadIdx.x; x < len; x += 256) to[x] = from[x];
    }
}

// What write and read have in common; each: rows of a workgroup.
int check_rows(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, int type, const int *d_seqs,
               int n, int max_count, const void *d_k, const void *d_v, int ld, const char *what) {
    if (mhip::check_pages(c, s, p, what) || mhip::check_list(c, s, d_seqs, n, what)) return -1;
    if (s->type != MHIP_Q4) return mhip::fail(c, "%s: a cache of type %d is not in 4 bits", what, s->type);
    if (type < MHIP_F32 || type > MHIP_BF16) return mhip::fail(c, "%s: rows of type %d", what, type);
    if (layer < 0 || layer >= s->n_layers) return mhip::fail(c, "%s: layer %d of %d", what, layer, s->n_layers);
    const int width = s->n_kv_heads * s->head_dim;
    if (max_count < 0 || ld < width)
        return mhip::fail(c, "%s: %d tokens a slot, rows %d apart (width %d)", what, max_count, ld, width);
    if (!n || !max_count) return 0;
    if (!d_k || !d_v) return mhip::fail(c, "%s: a null argument", what);
    if (((uintptr_t)d_k | (uintptr_t)d_v) % 16 || (size_t)ld * mhip::type_bytes(type) % 16)
        return mhip::fail(c, "%s: rows must start on 16 bytes", what);
    if ((long long)n * max_count >= 1 << 24)  // (a launch holds less than 2^32 threads)
        return mhip::fail(c, "%s: %d x %d rows in one call", what, n, max_count);
    return 0;
}

// Calls of more than four tokens a slot take them in fours (8 slots of 1000: 16.7 us written and read,
// with rows one by one 18.2; no difference where there are fewer); each: units of a workgroup.
struct Cut {
    bool fours;
    int units, each;
    dim3 grid;
};
Cut cut_of(const mhip_page_dims *s, int n, int max_count) {
    Cut r;
    r.fours = max_count > 4;
    r.units = n * (r.fours ? (max_count + 6) / 4 : max_count);
    const int pieces = 2 * s->n_kv_heads * s->head_dim / 8;
    r.each = pieces <= 128 ? 256 / pieces : 1;
    r.grid = dim3(mhip::blocks_for(r.units, r.each), (pieces + 255) / 256);
    return r;
}

template <class T>
void write(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, const int *seqs, const int *count,
           int n, int max_count, const void *k, const void *v, int ld, float *weights) {
    const Cut u = cut_of(s, n, max_count);
    auto *kernel = u.fours ? k_write_q4<T, 4> : k_write_q4<T, 1>;
    kernel<<<u.grid, 256, 0, c->stream>>>(*s, *p, layer, seqs, count, u.units, max_count, (const T *)k, (const T *)v,
                                          (size_t)ld, weights, u.each);
}
template <class T>
void read(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, const int *seqs, const int *count,
          int n, int max_count, void *k, void *v, int ld) {
    const Cut u = cut_of(s, n, max_count);
    auto *kernel = u.fours ? k_read_q4<T, 4> : k_read_q4<T, 1>;
    kernel<<<u.grid, 256, 0, c->stream>>>(*s, *p, layer, seqs, count, u.units, max_count, (T *)k, (T *)v, (size_t)ld,
                                          u.each);
}

}  // namespace

extern "C" {

size_t mhip_weights_bytes(const mhip_page_dims *s) {
    if (!mhip_pages_plan_bytes(s) || s->type != MHIP_Q4) return 0;
    if ((double)s->n_layers * s->max_seqs * s->n_kv_heads * s->max_blocks * s->page >= 0x1p58) return 0;
    return (size_t)s->n_layers * s->max_seqs * s->n_kv_heads * s->max_blocks * s->page * 4;
}

int mhip_pages_write_q4(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, int type,
                        const int *d_seqs, const int *d_count, int n, int max_count, const void *d_k,
                        const void *d_v, int ld, float *d_weights) {
    const char *what = "pages write_q4";
    if (check_rows(c, s, p, layer, type, d_seqs, n, max_count, d_k, d_v, ld, what)) return -1;
    if ((uintptr_t)d_weights % 16) return mhip::fail(c, "%s: the weights must be 16-byte aligned", what);
    if (!n || !max_count) return 0;
    if (mhip::use_device(c)) return -1;
    if (type == MHIP_F32) write<float>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld, d_weights);
    else if (type == MHIP_F16) write<_Float16>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld, d_weights);
    else write<__bf16>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld, d_weights);
    return mhip::check_launch(c, what);
}

int mhip_pages_read_q4(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, int type,
                       const int *d_seqs, const int *d_count, int n, int max_count, void *d_k, void *d_v, int ld) {
    const char *what = "pages read_q4";
    if (check_rows(c, s, p, layer, type, d_seqs, n, max_count, d_k, d_v, ld, what)) return -1;
    if (!n || !max_count) return 0;
    if (mhip::use_device(c)) return -1;
    if (type == MHIP_F32) read<float>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld);
    else if (type == MHIP_F16) read<_Float16>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld);
    else read<__bf16>(c, s, p, layer, d_seqs, d_count, n, max_count, d_k, d_v, ld);
    return mhip::check_launch(c, what);
}

int mhip_pages_fork_weights(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, float *d_weights,
                            const int *d_src, const int *d_dst, int n, int flags) {
    const char *what = "pages fork_weights";
    if (mhip::check_pages(c, s, p, what)) return -1;
    if (s->type != MHIP_Q4) return mhip::fail(c, "%s: a cache of type %d is not in 4 bits", what, s->type);
    if (!d_weights || (uintptr_t)d_weights % 16) return mhip::fail(c, "%s: the weights are null or not on 16 bytes", what);
    if (mhip_pages_fork(c, s, p, d_src, d_dst, n, flags)) return -1;
    if (!n) return 0;
    const long long items = (long long)n * s->n_layers * s->n_kv_heads;
    k_fork_weights<<<(unsigned)(items < 4096 ? items : 4096), 256, 0, c->stream>>>(*s, *p, d_weights, d_src, d_dst, n,
                                                                                 p->plan + mhip::PLAN_OK);
    return mhip::check_launch(c, what);
}

}  // extern "C"
