// Rows into and out of a cache in 4 bits (include/mia_hip.h; the layout:
// cache_q4.h), and the accumulated weights of a forked slot.
//
// For 32 values x of a token: lo and hi their least and greatest, m = fp16(lo),
// s = fp16((hi - m) / 15) with an fp32 difference and quotient, and
//   c = how many k of 0 .. 14 have x - m >= (k + 1/2) s   (0 where s is 0).
// The nearest code is estimated in fp32; where the estimate is within 2^-16 of a border
// (its own error is below 2^-17) the comparison is made in 64 bits, in which x - m and
// (k + 1/2) s are exact, so a code does not depend on how it was found.
#include "cache_q4.h"

namespace {

using mhip_q4::Shape;

__device__ inline float value(float x) { return x; }
__device__ inline float value(_Float16 x) { return (float)x; }
__device__ inline float value(__bf16 x) { return (float)x; }

__device__ __forceinline__ unsigned code_of(float x, float m, float s, float inv) {
    const float e = (x - m) * inv + 0.5f, whole = floorf(e);
    int c = (int)fminf(fmaxf(whole, 0.0f), 15.0f);
    const float over = e - whole;
    if (over < 0x1p-16f || over > 1.0f - 0x1p-16f) {
        const double d = (double)x - (double)m, step = (double)s;
        if (c < 15 && d >= (c + 0.5) * step) c++;
        else if (c > 0 && d < (c - 0.5) * step) c--;
    }
    return (unsigned)c;
}

// A row of a call and the place of its token; false where there is none.
struct Token {
    int page, t, slot, pos;
};
__device__ inline bool token_of(const mhip_page_dims &s, const mhip_pages &p, const int *seqs, const int *count,
                                unsigned row, int max_count, Token &k, bool &bad) {
    const int i = max_count == 1 ? row : row / max_count, j = max_count == 1 ? 0 : row % max_count;
    const int q = seqs[i], m = count ? count[i] : max_count;
    bad = false;
    if (j >= m) return false;
    const int lp = __builtin_ctz(s.page);
    const int pos = (unsigned)q < (unsigned)s.max_seqs ? p.len[q] - m + j : -1;
    int g = -1;
    if (pos >= 0 && pos >> lp < s.max_blocks && m <= max_count) g = p.table[(size_t)q * s.max_blocks + (pos >> lp)];
    bad = (unsigned)g >= (unsigned)s.n_pages;
    k = Token{g, pos & (s.page - 1), q, pos};
    return !bad;
}

// A thread has eight values of a row, four neighbours a group of 32 (keys'
// threads, then values'): gridDim.y workgroups share a row, or one takes several.
struct Place {
    unsigned row, x;
    bool is;
};
__device__ inline Place place_of(unsigned pieces, int rows, int each) {
    Place r;
    if (each > 1) {
        const unsigned in = threadIdx.x / pieces;
        r.row = blockIdx.x * each + in;
        r.x = threadIdx.x - in * pieces;
        r.is = in < (unsigned)each && r.row < (unsigned)rows;
    } else {
        r.row = blockIdx.x;
        r.x = blockIdx.y * 256 + threadIdx.x;
        r.is = r.x < pieces;
    }
    return r;
}

template <class T>
__global__ __launch_bounds__(256) void k_write_q4(mhip_page_dims s, mhip_pages p, int layer, const int *seqs,
                                                  const int *count, int rows, int max_count, const T *k,
                                                  const T *v, size_t ld, float *weights, int each) {
    const Shape f = mhip_q4::shape_of(s);
    const unsigned half = (unsigned)s.n_kv_heads * f.G * 4;
    const Place at = place_of(2 * half, rows, each);
    if (!at.is) return;
    const bool keys = at.x < half;
    const unsigned y = keys ? at.x : at.x - half;
    const int h = y / (f.G * 4), j = y / 4 % f.G, g = y & 3;
    T r[8];
    const T *from = (keys ? k : v) + (size_t)at.row * ld + (size_t)y * 8;
#pragma unroll
    for (int e = 0; e < (int)sizeof(T) / 2; e++) ((uint4 *)r)[e] = ((const uint4 *)from)[e];
    Token tok;
    bool bad;
    if (!token_of(s, p, seqs, count, at.row, max_count, tok, bad)) {
        if (bad && at.x == 0) atomicOr(&p.state[0], MHIP_PAGES_BAD);
        return;
    }
    float x[8];
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = value(r[e]);
        odd |= !(fabsf(x[e]) <= mhip_q4::MOST);
        x[e] = x[e] != x[e] ? 0.0f : fminf(fmaxf(x[e], -mhip_q4::MOST), mhip_q4::MOST);
    }
    if (odd) atomicOr(&p.state[0], MHIP_PAGES_NOT_FINITE);
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; e++) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, d));
        hi = fmaxf(hi, __shfl_xor(hi, d));
    }
    const float m = (float)(_Float16)lo + 0.0f;  // (-0 as 0: which zero of several is least is not defined)
    const _Float16 mh = (_Float16)m;
    const _Float16 sh = (_Float16)((fmaxf(hi - m, 0.0f) + 0.0f) / 15.0f);  // (m may round to more than hi)
    const float st = (float)sh, inv = st > 0.0f ? 1.0f / st : 0.0f;
    unsigned c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = st > 0.0f ? code_of(x[e], m, st, inv) : 0;
    uint8_t *to = (uint8_t *)(keys ? p.k : p.v) +
                  (((size_t)layer * s.n_pages + tok.page) * s.n_kv_heads + h) * f.block;
    if (keys) {
        unsigned w = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) w |= c[e] << (4 * (e / 2 + 4 * (e & 1)));
        *(unsigned *)(to + mhip_q4::key_word(f, tok.t, g, j)) = w;
        if (weights && g == 0 && j == 0)
            weights[mhip_q4::weights_row(s, layer, tok.slot, h) + tok.pos] = 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            to[mhip_q4::value_byte(f, tok.t, 4 * g + e, j)] = (uint8_t)(c[2 * e] | c[2 * e + 1] << 4);
    }
    if (g == 0) {
        *(_Float16 *)(to + mhip_q4::scale_at(f, tok.t, j)) = sh;
        *(_Float16 *)(to + mhip_q4::low_at(f, keys, tok.t, j)) = mh;
    }
}

template <class T>
__global__ __launch_bounds__(256) void k_read_q4(mhip_page_dims s, mhip_pages p, int layer, const int *seqs,
                                                 const int *count, int rows, int max_count, T *k, T *v,
                                                 size_t ld, int each) {
    const Shape f = mhip_q4::shape_of(s);
    const unsigned half = (unsigned)s.n_kv_heads * f.G * 4;
    const Place at = place_of(2 * half, rows, each);
    if (!at.is) return;
    const bool keys = at.x < half;
    const unsigned y = keys ? at.x : at.x - half;
    const int h = y / (f.G * 4), j = y / 4 % f.G, g = y & 3;
    Token tok;
    bool bad;
    if (!token_of(s, p, seqs, count, at.row, max_count, tok, bad)) {
        if (bad && at.x == 0) atomicOr(&p.state[0], MHIP_PAGES_BAD);
        return;
    }
    const uint8_t *from = (const uint8_t *)(keys ? p.k : p.v) +
                          (((size_t)layer * s.n_pages + tok.page) * s.n_kv_heads + h) * f.block;
    const float st = (float)*(const _Float16 *)(from + mhip_q4::scale_at(f, tok.t, j));
    const float m = (float)*(const _Float16 *)(from + mhip_q4::low_at(f, keys, tok.t, j));
    unsigned c[8];
    if (keys) {
        const unsigned w = *(const unsigned *)(from + mhip_q4::key_word(f, tok.t, g, j));
#pragma unroll
        for (int e = 0; e < 8; e++) c[e] = w >> (4 * (e / 2 + 4 * (e & 1))) & 15;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const unsigned b = from[mhip_q4::value_byte(f, tok.t, 4 * g + e, j)];
            c[2 * e] = b & 15;
            c[2 * e + 1] = b >> 4;
        }
    }
    T r[8];
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = (T)(st * (float)c[e] + m);  // (the product is exact)
    T *to = (keys ? k : v) + (size_t)at.row * ld + (size_t)y * 8;
#pragma unroll
    for (int e = 0; e < (int)sizeof(T) / 2; e++) ((uint4 *)to)[e] = ((uint4 *)r)[e];
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

struct Cut {
    int each;
    dim3 grid;
};
Cut cut_of(const mhip_page_dims *s, int rows) {
    Cut r;
    const int pieces = 2 * s->n_kv_heads * s->head_dim / 8;
    r.each = pieces <= 128 ? 256 / pieces : 1;
    r.grid = dim3(mhip::blocks_for(rows, r.each), (pieces + 255) / 256);
    return r;
}

template <class T>
void write(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, const int *seqs, const int *count,
           int n, int max_count, const void *k, const void *v, int ld, float *weights) {
    const Cut u = cut_of(s, n * max_count);
    k_write_q4<T><<<u.grid, 256, 0, c->stream>>>(*s, *p, layer, seqs, count, n * max_count, max_count, (const T *)k,
                                                 (const T *)v, (size_t)ld, weights, u.each);
}
template <class T>
void read(mhip_ctx *c, const mhip_page_dims *s, const mhip_pages *p, int layer, const int *seqs, const int *count,
          int n, int max_count, void *k, void *v, int ld) {
    const Cut u = cut_of(s, n * max_count);
    k_read_q4<T><<<u.grid, 256, 0, c->stream>>>(*s, *p, layer, seqs, count, n * max_count, max_count, (T *)k, (T *)v,
                                                (size_t)ld, u.each);
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
