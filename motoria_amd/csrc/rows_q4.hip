// Products with 4-bit weights in groups (include/mia_hip.h):
//   out[t][r] = sum over groups g of scale[r][g] * (sum over c in g of code[r][c] x[t][c]).
//
// What bounds it: up to about 16 tokens the weights' bytes (4.5 bits each with
// groups of 32), so the codes have to become matrix operands in few
// instructions. A code is exact in fp16: nibble k and k + 4 of a word, masked
// together and merged with the exponent of 1024, are the fp16 values 1024 + (code
// + 8) (or 1024 + 16 (code + 8)), and one packed subtraction (or fused
// multiply-add) leaves the two codes: 9 instructions for 8 weights. The inner
// sums then run on the matrix cores, 16 rows x 16 tokens x 32 columns an
// instruction with fp32 accumulators; with one token 15 of 16 of its columns are idle,
// which still is faster than the vector units (2.25 instructions a weight).
//
// x as fp16 operands (up to FEW tokens; fp32 x; 17 to 32 tokens of 16-bit x with many
// rows): each token's segment of 1024 columns is scaled by a power of two that
// brings its largest value to [2^14, 2^15). A bf16 value then is an fp16 value (8 bits;
// exact down to 2^-31 of the largest). An fp32 value is split: hi = fp16(x'), lo =
// fp16((x' - hi) 2^11), together within 2^-23 of x (a step of fp32's own rounding)
// down to 2^-27 of the segment's largest value (then fp16's least step counts, 2^-36
// of x'), as lo carries its own exponent; their products are accumulated apart and
// joined in fp32. fp16 x is taken as it is; elsewhere 16-bit x of either type is
// (k_q4_wide).
//
// Measured (us, a call in a row of calls; bytes of the weights at what a large copy
// reaches, 4.92 TB/s, in brackets): a head of 151936 x 2048, fp32, groups of 32, one token
// 40 [36], fp16 with groups of 128 33 [33]; 512 to 4096 x 2048, one token 5, a launch among
// others being 3.6; 4096 x 2048 in bf16 with 16 tokens 5.2, with 64 tokens 7.0, where a
// workgroup waits for 256 KB of operands from L2; the head with 16 tokens, fp32 81 [36],
// bf16, groups of 128, 57.5 [33], with 64 tokens 162.
#include "mhip_internal.h"
#include <type_traits>

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

constexpr int SEG = 1024;  // columns that share a token's power of two
constexpr int TG = 64;     // tokens of one workgroup, at most
constexpr int MOST_TOKENS = 65535 * TG;

// The workspace: per group of TG tokens (nt of them) the operands
// [cols/32][pieces][nt][32] fp16, in each 32 the order of codes(), then
// [cols/SEG][TG] the factors back.
struct Tokens {
    size_t operands, factors, group;  // bytes of each, and of a group
};
__host__ __device__ inline Tokens tokens_of(int type, int cols, int n) {
    Tokens t;
    const size_t nt = n < TG ? n : TG, pieces = type == MHIP_F32 ? 2 : 1;
    t.operands = ((size_t)cols * pieces * nt * 2 + 255) & ~(size_t)255;
    t.factors = ((size_t)((cols + SEG - 1) / SEG) * TG * 4 + 255) & ~(size_t)255;
    t.group = t.operands + t.factors;
    return t;
}

__device__ inline float value(float x) { return x; }
__device__ inline float value(_Float16 x) { return (float)x; }
__device__ inline float value(__bf16 x) { return (float)x; }

// 2^(14 - exponent of the largest magnitude m of a segment); values below
// 2^-112 keep the factor 2^126.
__device__ __forceinline__ float segment_scale(float m) {
    return ldexpf(1.0f, min(126, 14 - (m > 0.0f ? ilogbf(m) : 14)));
}
__device__ __forceinline__ float finite_max(float m, float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() && a > m ? a : m;
}
// hi and lo of a scaled value (an infinity or NaN is in hi alone)
__device__ __forceinline__ _Float16 lo_of(float s, _Float16 hi) {
    const float rest = (s - (float)hi) * 2048.0f;
    return fabsf(rest) < __builtin_inff() ? (_Float16)rest : (_Float16)0.0f;
}

// One workgroup a token and segment, four columns a thread.
template <class T>
__global__ __launch_bounds__(256) void k_q4_tokens(const T *x, int ldx, int cols, int n, int type,
                                                   uint8_t *ws) {
    constexpr bool split = sizeof(T) == 4;
    __shared__ float top[4];
    const int t = blockIdx.x, seg = blockIdx.y, tg = t / TG, nt = min(TG, n - tg * TG);
    const Tokens l = tokens_of(type, cols, n);
    uint8_t *base = ws + (size_t)tg * l.group;
    const int c = seg * SEG + threadIdx.x * 4;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < cols) {
        T r[4];
        if constexpr (split) *(uint4 *)r = *(const uint4 *)(x + (size_t)t * ldx + c);
        else *(uint2 *)r = *(const uint2 *)(x + (size_t)t * ldx + c);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = value(r[j]);
    }
    float scale = 1.0f;
    if (type != MHIP_F16) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) m = finite_max(m, v[j]);
        for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
        __syncthreads();
        scale = segment_scale(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    }
    if (threadIdx.x == 0)
        ((float *)(base + l.operands))[(size_t)seg * TG + t % TG] = 1.0f / scale;  // exact: a power of two
    if (c >= cols) return;
    // columns 4i .. 4i + 3 of an eight: nibbles k and k + 4 are neighbours, so
    // column k of the eight goes to place 2k (k < 4) or 2 (k - 4) + 1
    const size_t block = c / 32, pieces = split ? 2 : 1;
    _Float16 *o = (_Float16 *)base + ((block * pieces) * nt + t % TG) * 32 + (c % 32 / 8) * 8 +
                  (c % 8 == 4 ? 1 : 0);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float s = v[j] * scale;
        const _Float16 hi = (_Float16)s;
        o[2 * j] = hi;
        if constexpr (split) o[(size_t)nt * 32 + 2 * j] = lo_of(s, hi);
    }
}

// Eight codes (nibbles of w) as fp16, nibble k next to nibble k + 4.
__device__ __forceinline__ h8 codes(unsigned w) {
    const h2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f}, off16 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const h2 by = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned z = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & 0x000f000fu) ^ 0x64086408u) + off;
    const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00f000f0u) ^ 0x64806480u), by, off16);
    const h2 c = __builtin_bit_cast(h2, (z & 0x000f000fu) ^ 0x64086408u) + off;
    const h2 d = __builtin_elementwise_fma(__builtin_bit_cast(h2, (z & 0x00f000f0u) ^ 0x64806480u), by, off16);
    return (h8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight codes in their order as bf16, through fp32, 2^-11 of their size (exact), so that the
// sum of 128 of them times any values of x stays in fp32's range before the group's scale
// meets it. A difference of exponents, kept at 0 for codes of 0.
constexpr float BF_UP = 2048.0f;
__device__ __forceinline__ b8 codes_bf(unsigned w) {
    typedef unsigned short s2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    auto code = [&](int k) { return (__bf16)((float)((int)(w << (28 - 4 * k)) >> 28)); };
    u4 r;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        unsigned two = __builtin_bit_cast(unsigned, (b2){code(2 * k), code(2 * k + 1)});
        asm("" : "+v"(two));  // (else the pair is taken apart)
        r[k] = __builtin_bit_cast(unsigned, __builtin_elementwise_sub_sat(__builtin_bit_cast(s2, two), (s2)(11 << 7)));
    }
    return __builtin_bit_cast(b8, r);
}

// A lane of group g (16 lanes) has loaded words 0..3 of its column block; the matrix
// instructions want word g of group j's block: the transpose of words and lane
// groups, by exchanging halves (32 lanes) and quarters (16).
__device__ __forceinline__ void blocks_from_lanes(unsigned w[4]) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const auto r = __builtin_amdgcn_permlane32_swap(w[j], w[j + 2], false, false);
        w[j] = r[0];
        w[j + 2] = r[1];
    }
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        const auto r = __builtin_amdgcn_permlane16_swap(w[j], w[j + 1], false, false);
        w[j] = r[0];
        w[j + 1] = r[1];
    }
}

__device__ inline void put(float *o, float v) { *o = v; }
__device__ inline void put(_Float16 *o, float v) { *o = (_Float16)v; }
__device__ inline void put(__bf16 *o, float v) { *o = (__bf16)v; }

template <int N> struct Words { typedef unsigned type __attribute__((ext_vector_type(N))); };
template <> struct Words<1> { typedef unsigned type; };

constexpr int CHUNK = 256;     // columns of a wavefront's step
constexpr int FEW = 8;         // tokens whose operands a workgroup forms itself
constexpr int FEW_LDS = 65536; // bytes of LDS for them

// WR x WK wavefronts: a tile of 16 rows for each of WR, the columns' chunks of
// 256 dealt out to WK; TT tiles of 16 tokens; DEPTH chunks requested ahead. The
// tokens' operands come through LDS, kc columns at a time, from the workspace;
// with N > 0 (1: one token, FEW: up to FEW) the workgroup forms them from x itself,
// which saves a launch, and for fp32 x hi and lo of a token are two of the
// instruction's sixteen token rows. With N > 0 and WK = 1 a wavefront takes one
// tile after another, `stride` apart, with the next one's chunks on their
// way. WHOLE: rows of whole chunks, a chunk's scales on their boundary (one
// load). A chunk of 256 codes is 128 bytes of a row: with half of that the lines of
// sixteen rows had left the CU's cache before their second half was asked for.
template <class T, int G, bool WHOLE, int N, int TT, int WR, int WK, int DEPTH>
__global__ __launch_bounds__(64 * WR * WK) void k_q4(T *out, size_t ldo, const uint8_t *w,
                                                     const uint16_t *scales, int rows, int cols,
                                                     int n, int kc, const uint8_t *ws, const T *x,
                                                     size_t ldx, int type) {
    constexpr bool split = sizeof(T) == 4;  // hi and lo of a token: two token rows
    static_assert(N > 0 || !split, "from the workspace, 16-bit x");
    constexpr int P = split ? 2 : 1, NT = 64 * WR * WK, GC = CHUNK / G;  // groups of a chunk
    constexpr int TL = N == 1 ? 1 : split ? 2 : 4;                       // tokens of a lane and tile
    constexpr bool MANY = N > 0 && WK == 1;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR, g = lane >> 4, lr = lane & 15;
    const int tg = blockIdx.y, nt = min(TG, n - tg * TG);
    const int nchunk = (cols + CHUNK - 1) / CHUNK, nblock = cols / 32, ngroup = cols / G;
    const int ntile = (rows + 15) / 16, stride = gridDim.x * WR;
    int tile = blockIdx.x * WR + wr;
    const int my_tiles = MANY ? (tile < ntile ? (ntile - tile + stride - 1) / stride : 0) : 1;
    float total[TT][TL];
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
        for (int r = 0; r < TL; r++) total[t][r] = 0.0f;

    // A slot per chunk on its way: codes (blocks 2g and 2g + 1 of 32 columns for
    // lane group g), and the scales of its groups, two a word (one where they are
    // loaded one by one).
    constexpr int SW = WHOLE ? (GC + 1) / 2 : GC;
    using scale_words = typename Words<SW>::type;
    u4 wq[DEPTH][2];
    scale_words sq[DEPTH];
    // chunks wk, wk + WK, ... of each tile
    const int mine = nchunk > wk ? (nchunk - wk + WK - 1) / WK : 0;
    int next_tile = tile, next_c = 0;
    // Loads without a branch, so that the waits count them: past the end they
    // read what is there and nobody uses.
    auto request = [&](int d) {
        const int chunk = min(wk + next_c * WK, nchunk - 1);
        const size_t row = min(next_tile * 16 + lr, rows - 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            int block = chunk * (CHUNK / 32) + 2 * g + h;
            if constexpr (!WHOLE) block = min(block, nblock - 1);
            wq[d][h] = *(const u4 *)(w + row * (cols / 2) + (size_t)block * 16);
        }
        const uint16_t *at = scales + row * ngroup;
        if constexpr (WHOLE) {
            sq[d] = *(const scale_words *)(at + chunk * GC);
        } else {
#pragma unroll
            for (int j = 0; j < GC; j++) sq[d][j] = at[min(chunk * GC + j, ngroup - 1)];
        }
        if (++next_c >= mine) {
            next_c = 0;
            next_tile = min(next_tile + stride, ntile - 1);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; d++) request(d);

    const size_t step = (size_t)P * nt * 64;  // bytes of a block of 32 columns
    float *fl = (float *)(lds + (size_t)(kc / 32) * step);
    int k0 = -kc;  // the columns in LDS: k0 .. k0 + kc - 1
    // The next columns' operands into LDS: every wavefront gets here equally
    // often, whichever chunk it is at.
    auto stage = [&]() {
        k0 += kc;
        if constexpr (N > 0) {
            // a wavefront per token and segment, 16 columns a lane
            const int segs = (cols + SEG - 1) / SEG;
            for (int i = wave; i < n * segs; i += WR * WK) {
                const int t = i % n, seg = i / n;
                float v[2][8];
                float m = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int c = seg * SEG + h * 512 + lane * 8;
                    T r[8] = {};
                    if (c < cols) {
                        const T *at = x + (size_t)t * ldx + c;
                        *(uint4 *)r = *(const uint4 *)at;
                        if constexpr (split) *(uint4 *)(r + 4) = *(const uint4 *)(at + 4);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        v[h][j] = value(r[j]);
                        m = finite_max(m, v[h][j]);
                    }
                }
                float scale = 1.0f;
                if (type != MHIP_F16) {
                    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
                    scale = segment_scale(m);
                }
                if (lane == 0) fl[seg * TG + t] = 1.0f / scale;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int c = seg * SEG + h * 512 + lane * 8;
                    if (c >= cols) continue;
                    _Float16 *o = (_Float16 *)(lds + (size_t)(c / 32) * step) + t * 32 + c % 32;
                    h8 hi, lo;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int to = j < 4 ? 2 * j : 2 * j - 7;  // column j next to j + 4
                        hi[to] = (_Float16)(v[h][j] * scale);
                        if constexpr (split) lo[to] = lo_of(v[h][j] * scale, hi[to]);
                    }
                    *(h8 *)o = hi;
                    if constexpr (split) *(h8 *)(o + n * 32) = lo;
                }
            }
            __syncthreads();
        } else {
            const Tokens l = tokens_of(type, cols, n);
            const uint8_t *xg = ws + (size_t)tg * l.group;
            const float *fg = (const float *)(xg + l.operands);
            const int kn = min(kc, cols - k0), segs = (kn + SEG - 1) / SEG;
            __syncthreads();
            const uint4 *from = (const uint4 *)(xg + (size_t)(k0 / 32) * step);
            const int units = (int)((size_t)(kn / 32) * step / 16);
            for (int i = tid; i < units; i += NT) ((uint4 *)lds)[i] = from[i];
            for (int i = tid; i < segs * TG; i += NT)
                fl[i] = i % TG < nt ? fg[(size_t)(k0 / SEG) * TG + i] : 0.0f;
            __syncthreads();
        }
    };
    // a lane's token rows of the operands (past the last token: the last one's,
    // whose results are not stored), and its own tokens
    int from[TT], own[TT][TL];
#pragma unroll
    for (int t = 0; t < TT; t++) {
        from[t] = split ? (min(lr >> 1, nt - 1) + (lr & 1) * nt) * 64 + g * 16
                       : min(t * 16 + lr, nt - 1) * 64 + g * 16;
#pragma unroll
        for (int r = 0; r < TL; r++) own[t][r] = split ? 2 * g + r : t * 16 + 4 * g + r;
    }
    if constexpr (N > 0) stage();
    int c = 0;
    auto store = [&]() {
        const int row = tile * 16 + lr;
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < TL; r++)
                if (row < rows && own[t][r] < nt)
                    put(out + (size_t)(tg * TG + own[t][r]) * ldo + row, total[t][r]);
    };
    auto work = [&](int d) {  // the next chunk, from slot d
        const int chunk = wk + c * WK;
        if constexpr (N == 0)
            while (chunk * CHUNK >= k0 + kc) stage();
        unsigned q[2][4];
        float sc[GC];
        {
            // (the slot is taken apart here and not, with a wait, where it was loaded)
            u4 c0 = wq[d][0], c1 = wq[d][1];
            scale_words sw = sq[d];
            asm volatile("" : "+v"(c0), "+v"(c1), "+v"(sw));
#pragma unroll
            for (int j = 0; j < 4; j++) {
                q[0][j] = c0[j];
                q[1][j] = c1[j];
            }
#pragma unroll
            for (int j = 0; j < GC; j++) {
                unsigned h;
                if constexpr (SW == 1) h = sw >> (16 * j);
                else h = WHOLE ? sw[j / 2] >> (16 * (j & 1)) : sw[j];
                sc[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)h);
            }
        }
        request(d);
        __builtin_amdgcn_sched_barrier(0x78f);  // (all but memory reads may pass)
        blocks_from_lanes(q[0]);
        blocks_from_lanes(q[1]);
        const int b0 = chunk * (CHUNK / 32) - k0 / 32, blocks = nblock - chunk * (CHUNK / 32);
        float part[TT][TL];
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < TL; r++) part[t][r] = 0.0f;
        f4 sum[TT];
#pragma unroll
        for (int j = 0; j < CHUNK / 32; j++) {
            if (WHOLE || j < blocks) {
                const h8 b = codes(q[j & 1][j >> 1]);
                const bool begin = j % (G / 32) == 0, end = (j + 1) % (G / 32) == 0;
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    const uint8_t *at = lds + (size_t)(b0 + j) * step + from[t];
                    const f4 z = {0, 0, 0, 0};
                    sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const h8 *)at, b, begin ? z : sum[t], 0, 0, 0);
                    if (end) {
#pragma unroll
                        for (int r = 0; r < TL; r++) {
                            const float v = split ? __builtin_fmaf(sum[t][(2 * r + 1) & 3], 0x1p-11f, sum[t][2 * r & 3])
                                                  : sum[t][r];
                            part[t][r] = __builtin_fmaf(sc[j / (G / 32)], v, part[t][r]);
                        }
                    }
                }
            }
        }
        // back to x's own scale
        const float *f = fl + (chunk * CHUNK - k0) / SEG * TG;
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < TL; r++)
                total[t][r] = __builtin_fmaf(part[t][r], f[N > 0 ? min(own[t][r], nt - 1) : own[t][r]], total[t][r]);
        if (++c == mine && MANY) {
            store();
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int r = 0; r < TL; r++) total[t][r] = 0.0f;
            c = 0;
            tile += stride;
        }
    };
    const int steps = my_tiles * mine;
    int i = 0;
    for (; i + DEPTH <= steps; i += DEPTH)
#pragma unroll
        for (int d = 0; d < DEPTH; d++) work(d);
#pragma unroll
    for (int d = 0; d < DEPTH; d++)
        if (i + d < steps) work(d);
    if constexpr (MANY) return;
    while (k0 + kc < cols) stage();  // a wavefront whose chunks ended earlier
    if constexpr (WK > 1) {
        // the column shares' sums, added in their order by the first of them
        __syncthreads();
        float *sum = (float *)lds;
        if (wk > 0) {
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int r = 0; r < TL; r++)
                    sum[(((wk - 1) * WR + wr) * TT * TL + t * TL + r) * 64 + lane] = total[t][r];
        }
        __syncthreads();
        if (wk > 0) return;
        for (int k = 0; k < WK - 1; k++)
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int r = 0; r < TL; r++)
                    total[t][r] += sum[((k * WR + wr) * TT * TL + t * TL + r) * 64 + lane];
    }
    store();
}

// More than FEW tokens: RT tiles of 16 rows, the chunks of 256 columns dealt out
// to eight wavefronts. Each operand of the tokens is used
// once in the workgroup, so it comes straight from memory (L2) into registers: 16-bit
// x from x itself, unscaled and whole -- bf16 codes for a bf16 product, which
// cost two to three times the instructions that fp16 ones do, shared by the TT tiles of
// 16 tokens -- and fp32 x from the workspace. The registers of four wavefronts a SIMD keep the
// loads where they are written (fewer, and they move behind their uses: 151936 x 2048
// bf16, 16 tokens, 70 us; 57).
template <class T, int G, bool WHOLE, int TT, int RT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 4))) void k_q4_wide(T *out, size_t ldo, const uint8_t *w,
                                                 const uint16_t *scales, int rows, int cols, int n,
                                                 const uint8_t *ws, const T *x, size_t ldx) {
    constexpr bool split = sizeof(T) == 4, bf = std::is_same<T, __bf16>::value;
    constexpr int GC = CHUNK / G, WK = 8;
    __shared__ float sum[WK * RT * TT * 4 * 64];
    const int lane = threadIdx.x & 63, wk = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, lr = lane & 15;
    const int t0 = blockIdx.y * TT * 16, nt = min(TT * 16, n - t0);  // this workgroup's tokens
    const int tg = t0 / TG, of_group = min(TG, n - tg * TG);         // ... in a group of the workspace
    const int nchunk = (cols + CHUNK - 1) / CHUNK, nblock = cols / 32, ngroup = cols / G;
    const uint8_t *wr[RT];
    const uint16_t *sr[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        const size_t row = min(((int)blockIdx.x * RT + i) * 16 + lr, rows - 1);
        wr[i] = w + row * (cols / 2);
        sr[i] = scales + row * ngroup;
    }
    const Tokens l = tokens_of(split ? MHIP_F32 : MHIP_F16, cols, n);
    const uint8_t *xg = ws + (size_t)tg * l.group;
    const float *fg = (const float *)(xg + l.operands) + t0 % TG;
    // A lane's token row (past the last: the last one's). A load of the same half
    // line (64 bytes) of sixteen rows runs at half the rate, so of two blocks
    // of 32 columns every other row asks for the second one first, and swaps them
    // before the products (4096 x 2048, 64 tokens, bf16: 7.0 us, else 10.0).
    // (Sixteen rows on, addresses are the same in their last 8 bits.)
    const uint8_t *from[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
        const int tok = min(t * 16 + lr, nt - 1);
        from[t] = split ? xg + (t0 % TG + tok) * 64 + g * 16 : (const uint8_t *)(x + (size_t)(t0 + tok) * ldx + g * 8);
    }
    const bool swap = ((uintptr_t)from[0] >> 6 ^ lr) & 1;
    const size_t step = split ? (size_t)2 * of_group * 64 : 64;  // bytes from a block of 32 columns to the next
    f4 total[RT][TT];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int t = 0; t < TT; t++) total[i][t] = (f4){0, 0, 0, 0};
    for (int chunk = wk; chunk < nchunk; chunk += WK) {
        unsigned q[RT][2][4];
        uint16_t raw[RT][GC];
#pragma unroll
        for (int i = 0; i < RT; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                int block = chunk * (CHUNK / 32) + 2 * g + h;
                if constexpr (!WHOLE) block = min(block, nblock - 1);
                *(u4 *)q[i][h] = *(const u4 *)(wr[i] + (size_t)block * 16);
            }
            if constexpr (WHOLE) {
                using words = typename Words<GC / 2>::type;
                *(words *)raw[i] = *(const words *)(sr[i] + chunk * GC);
            } else {
#pragma unroll
                for (int j = 0; j < GC; j++) raw[i][j] = sr[i][min(chunk * GC + j, ngroup - 1)];
            }
        }
        const int b0 = chunk * (CHUNK / 32), blocks = nblock - b0;
        // the tokens' operands of the next blocks on their way
        constexpr int AHEAD = split ? 2 : TT == 1 ? 8 : 4;
        u4 xa[AHEAD][TT], xb[AHEAD][TT];
        auto fetch = [&](int j) {
#pragma unroll
            for (int t = 0; t < TT; t++) {
                // (from b0 on: the addresses of a whole chunk differ by constants)
                const int other = split || !swap ? 0 : j & 1 ? -1 : 1;
                const uint8_t *at = from[t] + (size_t)b0 * step;
                at += WHOLE ? other * 64 + j * (ptrdiff_t)step : min(j + other, blocks - 1) * (ptrdiff_t)step;
                xa[j % AHEAD][t] = *(const u4 *)at;
                if constexpr (split) xb[j % AHEAD][t] = *(const u4 *)(at + (size_t)of_group * 64);
            }
        };
#pragma unroll
        for (int j = 0; j < AHEAD; j++) fetch(j);
        __builtin_amdgcn_sched_barrier(0x78f);  // (all but memory reads may pass)
        float sc[RT][GC];
#pragma unroll
        for (int i = 0; i < RT; i++) {
#pragma unroll
            for (int j = 0; j < GC; j++) sc[i][j] = (float)__builtin_bit_cast(_Float16, raw[i][j]) * (bf ? BF_UP : 1.0f);
            blocks_from_lanes(q[i][0]);
            blocks_from_lanes(q[i][1]);
        }
        f4 part[RT][TT], hi[RT][TT], lo[RT][TT];
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int t = 0; t < TT; t++) part[i][t] = (f4){0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < CHUNK / 32; j++) {
            if (!split && j % 2 == 0) {
#pragma unroll
                for (int t = 0; t < TT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const unsigned u = xa[j % AHEAD][t][e], v = xa[(j + 1) % AHEAD][t][e];
                        xa[j % AHEAD][t][e] = swap ? v : u;
                        xa[(j + 1) % AHEAD][t][e] = swap ? u : v;
                    }
            }
            if (WHOLE || j < blocks) {
                using weights = std::conditional_t<bf, b8, h8>;
                weights b[RT];
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    if constexpr (bf) b[i] = codes_bf(q[i][j & 1][j >> 1]);
                    else b[i] = codes(q[i][j & 1][j >> 1]);
                }
                const bool begin = j % (G / 32) == 0, end = (j + 1) % (G / 32) == 0;
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    u4 a = xa[j % AHEAD][t];
                    const u4 a2 = xb[j % AHEAD][t];
                    if constexpr (!split && !bf)  // column k of an eight next to column k + 4, as codes() has them
                        a = (u4){__builtin_amdgcn_perm(a[2], a[0], 0x05040100), __builtin_amdgcn_perm(a[2], a[0], 0x07060302),
                                 __builtin_amdgcn_perm(a[3], a[1], 0x05040100), __builtin_amdgcn_perm(a[3], a[1], 0x07060302)};
#pragma unroll
                    for (int i = 0; i < RT; i++) {
                        const f4 z = {0, 0, 0, 0}, c = begin ? z : hi[i][t];
                        if constexpr (bf)
                            hi[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), b[i], c, 0, 0, 0);
                        else
                            hi[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), b[i], c, 0, 0, 0);
                        if constexpr (split)
                            lo[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a2), b[i],
                                                                              begin ? z : lo[i][t], 0, 0, 0);
                        if (end) {
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                float v = hi[i][t][r];
                                if constexpr (split) v = __builtin_fmaf(lo[i][t][r], 0x1p-11f, v);
                                part[i][t][r] = __builtin_fmaf(sc[i][j / (G / 32)], v, part[i][t][r]);
                            }
                        }
                    }
                }
            }
            if (j + AHEAD < CHUNK / 32) fetch(j + AHEAD);
            __builtin_amdgcn_sched_barrier(0x78f);  // (all but memory reads may pass)
        }
#pragma unroll
        for (int t = 0; t < TT; t++) {
            f4 back = {1.0f, 1.0f, 1.0f, 1.0f};  // to x's own scale
            if constexpr (split) back = *(const f4 *)(fg + (size_t)(chunk * CHUNK / SEG) * TG + t * 16 + g * 4);
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) total[i][t][r] = __builtin_fmaf(part[i][t][r], back[r], total[i][t][r]);
        }
    }
    // the column shares' sums, added in their order, some by each wavefront
    constexpr int ALL = RT * TT * 4;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) sum[(wk * ALL + (i * TT + t) * 4 + r) * 64 + lane] = total[i][t][r];
    __syncthreads();
    for (int y = wk; y < ALL; y += WK) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < WK; k++) v += sum[(k * ALL + y) * 64 + lane];
        const int at = (blockIdx.x * RT + y / (TT * 4)) * 16 + lr, tok = y / 4 % TT * 16 + 4 * g + y % 4;
        if (at < rows && tok < nt) put(out + (size_t)(t0 + tok) * ldo + at, v);
    }
}

// One thread a group (weights are quantized once, when a model is loaded).
__global__ __launch_bounds__(256) void k_quantize_q4(const float *w, size_t groups, int group,
                                                     uint8_t *codes, uint16_t *scales) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= groups) return;
    const float *v = w + i * group;
    float top = 0.0f;
    for (int j = 0; j < group; j++) top = fmaxf(top, fabsf(v[j]));
    const _Float16 h = (_Float16)fminf(top / 7.0f, 65504.0f);
    const float s = (float)h;
    scales[i] = __builtin_bit_cast(uint16_t, h);
    unsigned *o = (unsigned *)(codes + i * group / 2);
    for (int j = 0; j < group; j += 8) {
        unsigned word = 0;
        for (int k = 0; k < 8; k++) {
            const float q = s > 0.0f ? rintf(v[j + k] / s) : 0.0f;
            word |= ((unsigned)(int)fminf(fmaxf(q, -8.0f), 7.0f) & 15u) << (4 * k);
        }
        o[j / 8] = word;
    }
}

__global__ __launch_bounds__(256) void k_dequantize_q4(const uint8_t *codes, const uint16_t *scales,
                                                       size_t n, int group, float *w) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) return;
    const float s = (float)__builtin_bit_cast(_Float16, scales[i / group]);
    const unsigned word = *(const unsigned *)(codes + i / 2);
    for (int k = 0; k < 8; k++) w[i + k] = s * (float)((int)(word << (28 - 4 * k)) >> 28);
}

int check_q4(mhip_ctx *c, const char *what, const void *d_codes, const void *d_scales, int rows,
             int cols, int group) {
    // (a launch holds less than 2^32 threads: one for 8 weights)
    if (rows < 0 || rows > 1 << 28 || cols < 0 || cols > 1 << 24 || (long long)rows * cols > 1LL << 34 ||
        (group != 32 && group != 64 && group != 128) || cols % group)
        return mhip::fail(c, "%s: %d rows of %d in groups of %d (32, 64 or 128, dividing the row)",
                          what, rows, cols, group);
    if (rows && cols && (!d_codes || !d_scales)) return mhip::fail(c, "%s: a null argument", what);
    if ((uintptr_t)d_codes % 16 || (uintptr_t)d_scales % 2)
        return mhip::fail(c, "%s: the codes must be 16-byte aligned", what);
    return 0;
}

// One shape of the kernel.
template <class T, int G, bool WHOLE, int N, int TT, int WR, int WK, int DEPTH>
int launch(mhip_ctx *c, int type, T *out, int ldo, const void *w, const void *s, int rows, int cols,
           int n, const void *ws, const T *x, int ldx) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;
    const int nt = n < TG ? n : TG;
    // columns per LDS stage: all of them for operands formed in place, else a segment
    int kc = SEG;
    if (kc > cols || N > 0) kc = (cols + CHUNK - 1) / CHUNK * CHUNK;
    size_t lds = (size_t)kc * P * nt * 2 + (size_t)((kc + SEG - 1) / SEG) * TG * 4;
    const size_t join = (size_t)(WK - 1) * WR * TT * 1024;
    if (lds < join) lds = join;
    auto k = k_q4<T, G, WHOLE, N, TT, WR, WK, DEPTH>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 160 * 1024);
        if (mhip::check(c, e, "matvec_q4 LDS attribute")) return -1;
    }
    int wgs = (rows + WR * 16 - 1) / (WR * 16);
    if (N > 0 && WK == 1 && wgs > 768) wgs = 768;  // three a CU: each takes tile after tile
    const dim3 grid(wgs, (n + TG - 1) / TG);
    k<<<grid, 64 * WR * WK, lds, c->stream>>>(out, ldo, (const uint8_t *)w, (const uint16_t *)s, rows,
                                              cols, n, kc, (const uint8_t *)ws, x, ldx, type);
    return mhip::check_launch(c, "matvec_q4");
}

// Up to FEW tokens: from 12288 rows on there is a tile for each of three workgroups' wavefronts on every
// CU, which then take whole rows one after another; below, the columns are split
// over a workgroup's wavefronts (2048 columns, one token: 8192 rows 6.4 us, whole
// rows 7.9; 16384 rows 11.3 us, whole rows 8.1; head of 151936 rows 73 and 40 us).
constexpr int MANY_ROWS = 12288;

template <class T, int G, bool WHOLE, int TT>
int many_tokens(mhip_ctx *c, int type, T *out, int ldo, const void *w, const void *s, int rows,
                int cols, int n, void *ws, const T *x, int ldx) {
    // 17 to 32 tokens of 16-bit x: from LDS where rows are many (bf16, 32 tokens of
    // 2048 columns: 16384 rows 15.1 us, k_q4_wide 12.1; 32768 rows 18.3 and 21.9; 151936 rows
    // 72 and 104)
    constexpr bool may = TT == 2 && sizeof(T) == 2;
    const bool many = may && rows >= 2 * MANY_ROWS;
    if (many || type == MHIP_F32) {
        k_q4_tokens<T><<<dim3(n, (cols + SEG - 1) / SEG), 256, 0, c->stream>>>(x, ldx, cols, n, type,
                                                                               (uint8_t *)ws);
        if (mhip::check_launch(c, "matvec_q4 tokens")) return -1;
    }
    if constexpr (may)
        if (many) return launch<T, G, WHOLE, 0, TT, 4, 2, 2>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
    // (fp32 x takes twice the registers: 32 tokens a workgroup at most; 64 tokens of
    // 11008 x 4096 40 us, all in one 74)
    constexpr int WT = TT == 4 && sizeof(T) == 4 ? 2 : TT;
    // (at most 65535 workgroups in a launch's second dimension: fp32 calls may take several
    // launches of whole groups of the workspace, the last one of more than a group)
    auto wide = [&](auto k, int rt) {
        const size_t group = tokens_of(type, cols, n).group;
        for (int t = 0, part; t < n; t += part) {
            part = n - t <= 65535 * 16 * WT ? n - t : 1 << 20;
            k<<<dim3((rows + 16 * rt - 1) / (16 * rt), (part + 16 * WT - 1) / (16 * WT)), 512, 0, c->stream>>>(
                out + (size_t)t * ldo, ldo, (const uint8_t *)w, (const uint16_t *)s, rows, cols, part,
                (const uint8_t *)ws + t / TG * group, x + (size_t)t * ldx, ldx);
        }
    };
    // two tiles of rows a workgroup where one each would be more than one per CU (64
    // tokens, bf16, 6144 x 2048: 12.5 us, two tiles 9.7; 16 tokens 5.5 and 5.3, fp32 10.0 and 8.5)
    if (rows > 256 * 16) wide(k_q4_wide<T, G, WHOLE, WT, 2>, 2);
    else wide(k_q4_wide<T, G, WHOLE, WT, 1>, 1);
    return mhip::check_launch(c, "matvec_q4");
}

template <class T, int G, bool WHOLE>
int choose(mhip_ctx *c, int type, T *out, int ldo, const void *w, const void *s, int rows, int cols,
           int n, void *ws, const T *x, int ldx) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;
    if (n <= FEW && (size_t)(cols + CHUNK - 1) / CHUNK * CHUNK * n * P * 2 <= FEW_LDS) {
        const bool many = rows >= MANY_ROWS;
        if (n == 1)
            return many ? launch<T, G, WHOLE, 1, 1, 4, 1, 2>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx)
                        : launch<T, G, WHOLE, 1, 1, 1, 8, 1>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
        return many ? launch<T, G, WHOLE, FEW, 1, 4, 1, 2>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx)
                    : launch<T, G, WHOLE, FEW, 1, 1, 8, 1>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
    }
    if (n > 32) return many_tokens<T, G, WHOLE, 4>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
    if (n > 16) return many_tokens<T, G, WHOLE, 2>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
    return many_tokens<T, G, WHOLE, 1>(c, type, out, ldo, w, s, rows, cols, n, ws, x, ldx);
}

template <class T>
int run(mhip_ctx *c, int type, void *out, int ldo, const void *w, const void *s, int group,
        const void *x, int ldx, int rows, int cols, int n, void *ws) {
    // rows of whole chunks, a chunk's scales in one load
    const bool whole = cols % CHUNK == 0 && (uintptr_t)s % (2 * CHUNK / group) == 0;
    auto call = [&](auto f) { return f(c, type, (T *)out, ldo, w, s, rows, cols, n, ws, (const T *)x, ldx); };
    if (group == 32) return whole ? call(choose<T, 32, true>) : call(choose<T, 32, false>);
    if (group == 64) return whole ? call(choose<T, 64, true>) : call(choose<T, 64, false>);
    return whole ? call(choose<T, 128, true>) : call(choose<T, 128, false>);
}

}  // namespace

extern "C" {

int mhip_quantize_q4(mhip_ctx *c, const float *d_w, int rows, int cols, int group, void *d_codes,
                     void *d_scales) {
    if (check_q4(c, "quantize_q4", d_codes, d_scales, rows, cols, group)) return -1;
    if (!rows || !cols) return 0;
    if (!d_w) return mhip::fail(c, "quantize_q4: a null argument");
    if (mhip::use_device(c)) return -1;
    const size_t groups = (size_t)rows * (cols / group);
    k_quantize_q4<<<mhip::blocks_for(groups, 256), 256, 0, c->stream>>>(
        d_w, groups, group, (uint8_t *)d_codes, (uint16_t *)d_scales);
    return mhip::check_launch(c, "quantize_q4");
}

int mhip_dequantize_q4(mhip_ctx *c, const void *d_codes, const void *d_scales, int rows, int cols,
                       int group, float *d_w) {
    if (check_q4(c, "dequantize_q4", d_codes, d_scales, rows, cols, group)) return -1;
    if (!rows || !cols) return 0;
    if (!d_w) return mhip::fail(c, "dequantize_q4: a null argument");
    if (mhip::use_device(c)) return -1;
    const size_t n = (size_t)rows * cols;
    k_dequantize_q4<<<mhip::blocks_for(n / 8, 256), 256, 0, c->stream>>>(
        (const uint8_t *)d_codes, (const uint16_t *)d_scales, n, group, d_w);
    return mhip::check_launch(c, "dequantize_q4");
}

size_t mhip_matvec_q4_ws_bytes(int type, int cols, int n) {
    if (type < MHIP_F32 || type > MHIP_BF16 || cols <= 0 || cols > 1 << 24 || cols % 32 || n <= 0 || n > MOST_TOKENS)
        return 0;
    return tokens_of(type, cols, n).group * (size_t)((n + TG - 1) / TG);
}

int mhip_matvec_q4(mhip_ctx *c, int type, void *d_out, int ldo, const void *d_codes,
                   const void *d_scales, int group, const void *d_x, int ldx, int rows, int cols,
                   int n, void *d_ws) {
    if (check_q4(c, "matvec_q4", d_codes, d_scales, rows, cols, group)) return -1;
    if (type < MHIP_F32 || type > MHIP_BF16) return mhip::fail(c, "matvec_q4: type %d", type);
    if (n < 0 || ldx < cols || ldo < rows)
        return mhip::fail(c, "matvec_q4: %d tokens, rows %d and %d apart (%d columns, %d rows)", n,
                          ldx, ldo, cols, rows);
    if (rows > (1 << 28) - 32)  // (a launch holds less than 2^32 threads: 512 for two tiles of 16 rows)
        return mhip::fail(c, "matvec_q4: %d rows in one call", rows);
    if (!n || !rows) return 0;
    if (!cols) return mhip::fail(c, "matvec_q4: no columns");
    if (!d_out || !d_x || !d_ws) return mhip::fail(c, "matvec_q4: a null argument");
    const int esz = mhip::type_bytes(type);
    if ((uintptr_t)d_x % 16 || (size_t)ldx * esz % 16 || (uintptr_t)d_out % esz ||
        (uintptr_t)d_ws % 256)
        return mhip::fail(c, "matvec_q4: x rows must start on 16 bytes, the workspace on 256");
    if (n > MOST_TOKENS)
        return mhip::fail(c, "matvec_q4: %d tokens of %d columns in one call", n, cols);
    if (mhip::use_device(c)) return -1;
    if (type == MHIP_F32)
        return run<float>(c, type, d_out, ldo, d_codes, d_scales, group, d_x, ldx, rows, cols, n, d_ws);
    if (type == MHIP_F16)
        return run<_Float16>(c, type, d_out, ldo, d_codes, d_scales, group, d_x, ldx, rows, cols, n, d_ws);
    return run<__bf16>(c, type, d_out, ldo, d_codes, d_scales, group, d_x, ldx, rows, cols, n, d_ws);
}

}  // extern "C"
