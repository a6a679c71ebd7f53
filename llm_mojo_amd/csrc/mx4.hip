// Microscaled 4-bit floating point (include/llmq.h, llmq_mx4_*): blocks of 32
// values along the reduction axis, each an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4,
// 6 and a sign bit) times the block's power-of-two scale (e8m0: 2^(byte -
// 127), 255 NaN), as in the OCP Microscaling Formats specification 1.0.
//
// The products run on the block-scaled matrix instruction (16 x 16 outputs,
// 128 of the reduction axis a step): lane l holds the 32 values of row l % 16,
// block l / 16, one 16-byte load, and the block's scale byte.  Products of
// two codes are multiples of 1/4 up to 36 and the scales powers of two, so the only
// roundings are those of the float32 sums.
//
// Device layout of a matrix: rows in tiles of 16, codes [tile][step][lane][16
// bytes] (a wave's operand is 1 KB in one piece), scales [tile][step /
// 4][lane][4 bytes] (four steps' bytes a word, the instruction selects one).
// A tile has whole words of four steps; rows and blocks past the matrix's end
// are zero codes with scale 127.
#include <math.h>

#include <new>
#include <type_traits>
#include <vector>

#include "common.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// The scale byte of a block with largest magnitude m (any_bad: it holds a NaN
// or an infinity): floor(log2 m) - 2, the exponent that brings m into [4, 8),
// at least 2^-127.
__device__ __forceinline__ int scale_byte(float m, bool bad) {
    const int e = (int)(__float_as_uint(m) >> 23) - 2;
    return bad ? 255 : (e < 0 ? 0 : e);
}

// 2^(127 - e), the reciprocal of scale byte e < 254 (exact; byte 255 gives 2^-126, whose codes mean nothing).
__device__ __forceinline__ float inverse_scale(int e) {
    return __uint_as_float((uint32_t)(254 - (e > 253 ? 253 : e)) << 23);
}
__device__ __forceinline__ float scale_value(int e) {
    return e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(e == 0 ? 1u << 22 : (uint32_t)e << 23);
}

// Eight values as codes of a word, x0 lowest: nearest, ties to the even code, saturating at 6.
__device__ __forceinline__ uint32_t codes8(const float *x, float inv) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] * inv, x[1] * inv, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] * inv, x[3] * inv, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] * inv, x[5] * inv, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] * inv, x[7] * inv, 1.0f, 3);
    return w;
}

__device__ __forceinline__ uint4 quant_block(const float (&x)[32], int *scale) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        m = fmaxf(m, fabsf(x[i]));
        bad |= !(fabsf(x[i]) <= 3.402823466e38f);
    }
    const int e = scale_byte(m, bad);
    const float inv = inverse_scale(e);
    *scale = e;
    if (bad) return make_uint4(0, 0, 0, 0);
    return make_uint4(codes8(x, inv), codes8(x + 8, inv), codes8(x + 16, inv), codes8(x + 24, inv));
}

__device__ __forceinline__ float code_value(int c) {
    const int m = c & 7;
    const float v = m < 2 ? 0.5f * (float)m : (float)(2 + (m & 1)) * (float)(1 << (m >> 1)) * 0.25f;
    return c & 8 ? -v : v;
}

struct Float4 {
    float x[4];
} __attribute__((packed, aligned(4)));

// Largest magnitude over the four lanes of a block (quad permutes); NaN counts as above all.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
    return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
}

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ int scale_of_bits(uint32_t m) {
    const int e = (int)(m >> 23) - 2;
    return m >= 0x7f800000u ? 255 : (e < 0 ? 0 : e);
}

// One lane's quarter of a block: its 8 codes, and the block's scale byte.
__device__ __forceinline__ uint32_t quant_quarter(const float (&x)[8], int *scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    const int e = scale_of_bits(quad_max(m));
    *scale = e;
    return e == 255 ? 0u : codes8(x, inverse_scale(e));
}

// llmq_mx4_quantize: eight lanes a block, 4 values each, so that a wave's load
// is 1 KB in one piece; kQuant pairs of them a lane.  Two lanes' codes make a
// word, which the even lane stores for the first of a pair and the odd one
// for the second.  Bound by reading the floats, which pass the caches by:
// 4096 x 11008 36 us (5.7 TB/s of both sides; 52 by plain loads).  unit = K / 4
// lanes a row (0: the rows lie together).
constexpr int kQuant = 4;
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const float *__restrict__ x, int64_t ldx, uint32_t unit,
                                                           int64_t total, uint32_t *__restrict__ codes,
                                                           uint8_t *__restrict__ scales) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t i0 = ((int64_t)blockIdx.x * 4 + wave) * (128 * kQuant) + lane;
    Float4 v[2 * kQuant];
#pragma unroll
    for (int k = 0; k < 2 * kQuant; k++) {
        const int64_t i = i0 + 64 * k;
        if (i < total) llmq_load4_once(x + (unit ? (i / unit) * ldx + (i % unit) * 4 : i * 4), v[k].x);
    }
    const bool odd = threadIdx.x & 1;
#pragma unroll
    for (int k = 0; k < kQuant; k++) {
        uint32_t word[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const float *y = v[2 * k + s].x;
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
            m = quad_max(m);
            m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));  // row_half_mirror
            const int e = scale_of_bits(m);
            const float inv = inverse_scale(e);
            uint32_t c = 0;
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[0] * inv, y[1] * inv, 1.0f, 0);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2] * inv, y[3] * inv, 1.0f, 1);
            if (e == 255) c = 0;
            const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0xB1, 0xF, 0xF, false);
            word[s] = odd ? other | c << 16 : c | other << 16;
            const int64_t i = i0 + 64 * (2 * k + s);  // the eight lanes of a block are in or out together
            if ((threadIdx.x & 7) == 0 && i < total) scales[i >> 3] = (uint8_t)e;
        }
        const int64_t i = i0 + 64 * (2 * k + (odd ? 1 : 0));
        if (i < total) codes[i >> 1] = odd ? word[1] : word[0];
    }
}

// The same into a record: tokens in tiles of 16 laid out as a matrix's rows
// are, so that a product's operand is 1 KB in one piece (rows of packed codes
// 2 KB apart, at 4096 inputs, meet in few of L2's channels, and the scales
// that are gathered from them cost the product's kernel registers, 28 bytes of
// scratch a lane with 96 tokens: 2048 x 4096 x 11008 takes 94 us from those and
// 69 by way of a record, 2048 x 11008 x 4096 70 and 70).  A workgroup 16 tokens
// and a group of four steps, a wave a block of each step; tokens and blocks
// past the end become zeros with scale 127.  2048 x 4096 takes 9-12 us after a
// product (7 alone; 38 MB).
__global__ __launch_bounds__(256) void mx4_record_kernel(const float *__restrict__ x, int64_t T, int nb, int words,
                                                         uint32_t *__restrict__ codes, uint32_t *__restrict__ scales) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = lane >> 2, quarter = lane & 3, g = blockIdx.x;
    const int64_t tile = blockIdx.y, t = tile * 16 + row;
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int b = g * 16 + 4 * j + w;
        if (t < T && b < nb) {
            const float *p = x + (t * nb + b) * 32 + quarter * 8;
            const Float4 y = *reinterpret_cast<const Float4 *>(p), z = *reinterpret_cast<const Float4 *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[j][i] = y.x[i];
                v[j][4 + i] = z.x[i];
            }
        }
    }
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int b = g * 16 + 4 * j + w;
        int e = 127;
        uint32_t code = 0;
        if (t < T && b < nb) code = quant_quarter(v[j], &e);  // four lanes of a block: in or out together
        word |= (uint32_t)e << (8 * j);
        codes[(((tile * words + g) * 4 + j) * 64 + row + 16 * w) * 4 + quarter] = code;
    }
    if (quarter == 0) scales[(tile * words + g) * 64 + row + 16 * w] = word;
}

// llmq_mx4_dequantize: a thread kQuant words of codes, 32 bytes out of each.
// Bound by writing the floats: 4096 x 11008 36 us (5.6 TB/s; streaming stores,
// which leave lines half written, 74).
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, uint32_t unit,
                                                             int64_t total, float *__restrict__ out, int64_t ldo) {
    const int64_t i0 = (int64_t)blockIdx.x * (256 * kQuant) + threadIdx.x;
    uint32_t c[kQuant];
    float s[kQuant];
#pragma unroll
    for (int k = 0; k < kQuant; k++) {
        const int64_t i = i0 + 256 * k;
        if (i < total) {
            c[k] = codes[i];
            s[k] = scale_value(scales[i >> 2]);
        }
    }
#pragma unroll
    for (int k = 0; k < kQuant; k++) {
        const int64_t i = i0 + 256 * k;
        if (i >= total) continue;
        float *p = out + (unit ? (i / unit) * ldo + (i % unit) * 8 : i * 8);
        Float4 a, b;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            a.x[j] = code_value((c[k] >> (4 * j)) & 15) * s[k];
            b.x[j] = code_value((c[k] >> (4 * j + 16)) & 15) * s[k];
        }
        *reinterpret_cast<Float4 *>(p) = a;
        *reinterpret_cast<Float4 *>(p + 4) = b;
    }
}

// A weight matrix from floats: a thread a (row, block); with reduce_rows
// (source [IN, OUT]) neighbouring threads read neighbouring floats.
__global__ __launch_bounds__(256) void mx4_weights_kernel(const float *__restrict__ src, int64_t cols, int reduce_rows,
                                                          int64_t n, int64_t nb, int64_t words,
                                                          uint4 *__restrict__ codes, uint8_t *__restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * nb) return;
    const int64_t o = reduce_rows ? i % n : i / nb, b = reduce_rows ? i / n : i % nb;
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = reduce_rows ? src[(b * 32 + j) * cols + o] : src[o * cols + b * 32 + j];
    int e;
    const uint4 c = quant_block(v, &e);
    const int64_t tile = o >> 4, step = b >> 2;
    const int lane = (int)(o & 15) + 16 * (int)(b & 3);
    codes[(tile * words * 4 + step) * 64 + lane] = c;
    scales[((tile * words + (step >> 2)) * 64 + lane) * 4 + (step & 3)] = (uint8_t)e;
}

// GELU in its tanh form, 0.5 r (1 + tanh z) = r / (1 + e^-2z) with z =
// sqrt(2 / pi) (r + 0.044715 r^3): one exponential and a reciprocal, no branches
// and no cancellation for negative r.
__device__ __forceinline__ float gelu_of(float r) {
    const float u = fmaf(0.044715f * r * r, r, r);
    const float e = __builtin_amdgcn_exp2f(u * -2.302208198f);  // -2 sqrt(2 / pi) log2 e
    return r * __builtin_amdgcn_rcpf(1.0f + e);
}

// act(sum + bias) (+ what is there): the epilogue of every product here.
__device__ __forceinline__ void finish(float *p, float y, const float *bias, int64_t o, int flags) {
    if (flags & LLMQ_BIAS) y = y + bias[o];
    if (flags & LLMQ_GELU) y = gelu_of(y);
    if (flags & LLMQ_RESID) y = *p + y;
    *p = y;
}

// Four of a row's n floats from o on, zeros past its end, and back.
__device__ __forceinline__ v4f load_four(const float *p, int o, int n) {
    v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (o + 4 <= n) {
        v = __builtin_bit_cast(v4f, *reinterpret_cast<const Float4 *>(p + o));
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (o + i < n) v[i] = p[o + i];
    }
    return v;
}
__device__ __forceinline__ void store_four(float *p, const v4f &v, int o, int n) {
    if (o + 4 <= n) {
        *reinterpret_cast<Float4 *>(p + o) = __builtin_bit_cast(Float4, v);
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (o + i < n) p[o + i] = v[i];
    }
}

// Operands of a product: tokens in packed rows (codes K / 2 and scales K / 32
// bytes each; nb blocks) or a record, the matrix in its layout.
enum { kRows = 0, kRecord = 1, kFloats = 2 };  // how a kernel is given its tokens (kFloats: one)
struct Product {
    const uint8_t *xc, *xs;
    const uint8_t *wc;
    const uint32_t *ws;
    const float *x;  // one token's floats instead of xc, xs
    int64_t T;
    int n, nb, steps, words, ntiles;
    float *out;
    const float *bias;
    int flags;
};

__device__ __forceinline__ v4f mma(const uint4 &a, const uint4 &b, const v4f &c, int as, int bs, int sel) {
    const v8i x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0},
              y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    switch (sel) {  // a constant after unrolling
        case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, as, 0, bs);
        case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 1, as, 1, bs);
        case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 2, as, 2, bs);
        default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 3, as, 3, bs);
    }
}

// The scale bytes of blocks q, 4 + q, 8 + q, 12 + q of a token's 16 blocks
// from block 16 g, in one word (a step a byte).  Blocks past the row's end
// get 127: their weights are zeros, which a NaN there would spoil.
struct Bytes16 {
    uint32_t x[4];
} __attribute__((packed, aligned(1)));
__device__ __forceinline__ uint32_t pack_scales(const Bytes16 &s, int q) {
    const uint32_t sel = 0x0400u + 0x0101u * q;
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(s.x[3], s.x[2], sel),
                                 __builtin_amdgcn_perm(s.x[1], s.x[0], sel), 0x05040100u);
}
__device__ __forceinline__ uint32_t tail_scales(const uint8_t *row, int nb, int g, int q) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int b = g * 16 + 4 * j + q;
        w |= (b < nb ? (uint32_t)row[b] : 127u) << (8 * j);
    }
    return w;
}
__device__ __forceinline__ uint32_t token_scales(const uint8_t *row, int nb, int g, int q) {
    if (g * 16 + 16 > nb) return tail_scales(row, nb, g, q);
    return pack_scales(*reinterpret_cast<const Bytes16 *>(row + g * 16), q);
}

// Waves of a few-token workgroup at most: with four token tiles its registers hold half as many.
constexpr int few_most(int tt) { return tt < 4 ? 16 : 8; }

// Few tokens: a workgroup 16 outputs and TT tiles of 16 tokens, its waves
// taking groups of four steps (`per` each, in a row), their sums added in LDS
// in wave order: the matrix's few tiles become many waves with all of a
// group's operands asked for before its first product, and the next group's
// weights.  Bound by the weights for one token tile, then by the tokens'
// codes, which every workgroup reads (two tiles of outputs a workgroup halve
// that and were slower at every size measured: 64 x 4096 x 11008 14.9 us
// against 11.3).  kFloats: one token from its floats, quantized by every
// workgroup into LDS while its weights are on their way, in place of a launch
// that writes 17 / 32 K bytes.  4096 x 11008 for one token 5.4-6.3 us, the
// read of its 24 MB alone 5.6.
template <int TT, int X>
__global__ __launch_bounds__(64 * few_most(TT)) void mx4_few_kernel(Product p, int per) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4,
              c = lane & 15, waves = blockDim.x >> 6;
    const int tile = blockIdx.x;
    const int64_t t0 = (int64_t)blockIdx.y * (16 * TT);
    const auto rw = llmq_rsrc(p.wc + (int64_t)tile * p.words * 4096, (uint32_t)p.steps * 1024);
    const uint32_t *ws = p.ws + (int64_t)tile * p.words * 64 + lane;
    const int rowb = p.nb * 16;
    const int64_t left = p.T - t0;
    const int live = (int)(left < 16 * TT ? left : 16 * TT);
    const uint32_t tiles = (uint32_t)(live + 15) / 16;
    const auto rx = X == kRows     ? llmq_rsrc(p.xc + t0 * rowb, (uint32_t)live * rowb)
                    : X == kRecord ? llmq_rsrc(p.xc + t0 / 16 * p.words * 4096, tiles * p.words * 4096)
                                   : llmq_rsrc(p.wc, 0);
    uint8_t *fs = lds, *fc = lds + p.words * 16;  // kFloats: scales [group][q][step], codes

    uint4 a[4];
    uint32_t as;
    auto weights = [&](int g) {
#pragma unroll
        for (int j = 0; j < 4; j++)  // zeros past the last step, without reading them
            a[j] = llmq_bload16(rw, lane * 16 + (g * 4 + j) * 1024);
        as = ws[g * 64];
    };
    int g = w * per;
    const int end = min(g + per, p.words);
    if (g < end) weights(g);
    if constexpr (X == kFloats) {
        const int units = p.words * 64;  // quarters of blocks
        for (int i = tid; i < units; i += blockDim.x) {
            float v[8];
            int e = 127;
            uint32_t code = 0;
            if (i < p.nb * 4) {
                const Float4 x = *reinterpret_cast<const Float4 *>(p.x + i * 8),
                             y = *reinterpret_cast<const Float4 *>(p.x + i * 8 + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    v[j] = x.x[j];
                    v[4 + j] = y.x[j];
                }
                code = quant_quarter(v, &e);
            }
            reinterpret_cast<uint32_t *>(fc)[i] = code;
            const int blk = i >> 2;
            if ((i & 3) == 0) fs[(blk & ~15) + (blk & 3) * 4 + ((blk >> 2) & 3)] = (uint8_t)e;
        }
        __syncthreads();
    }
    v4f acc[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) acc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    for (; g < end; g++) {
        uint4 b[TT][4];
        uint32_t bs[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) {
            if constexpr (X == kFloats) {  // the token in every column
                bs[t] = *reinterpret_cast<const uint32_t *>(fs + g * 16 + q * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) b[t][j] = *reinterpret_cast<const uint4 *>(fc + (g * 4 + j) * 64 + q * 16);
            } else if constexpr (X == kRecord) {
                const int64_t at = t0 / 16 + min(t, (live - 1) / 16);
                bs[t] = reinterpret_cast<const uint32_t *>(p.xs)[(at * p.words + g) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; j++) b[t][j] = llmq_bload16(rx, ((t * p.words + g) * 4 + j) * 1024 + lane * 16);
            } else {
                const int row = min(16 * t + c, live - 1);
                bs[t] = token_scales(p.xs + (t0 + row) * p.nb, p.nb, g, q);
#pragma unroll
                for (int j = 0; j < 4; j++) b[t][j] = llmq_bload16(rx, row * rowb + q * 16 + (g * 4 + j) * 64);
            }
        }
        uint4 u[4];
        const uint32_t us = as;
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = a[j];
        if (g + 1 < end) weights(g + 1);
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int t = 0; t < TT; t++) acc[t] = mma(u[j], b[t][j], acc[t], (int)us, (int)bs[t], j);
    }
    // [wave][tile][token][output]
    float *sum = reinterpret_cast<float *>(lds);
    if constexpr (X == kFloats) __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; t++)
        if (X != kFloats || c == 0) *reinterpret_cast<v4f *>(sum + ((w * TT + t) * 16 + c) * 16 + 4 * q) = acc[t];
    __syncthreads();
    for (int i = tid; i < live * 16; i += blockDim.x) {
        const int o = tile * 16 + (i & 15);
        float y = sum[i];
        for (int k = 1; k < waves; k++) y += sum[k * TT * 256 + i];
        if (o < p.n) finish(p.out + (t0 + (i >> 4)) * p.n + o, y, p.bias, o, p.flags);
    }
}

// Many tokens: a workgroup 256 outputs and TT tiles of 16 tokens, a wave 64 of
// the outputs by all the tokens.  The tokens' codes are shared by the four
// waves: they are copied to LDS a group of four steps ahead, each fragment as
// the 1 KB that a wave reads of it, without passing through registers; their
// scales are put into words there a group ahead.  A wave's weights, which no
// other wave of the workgroup reads, come straight to its registers three
// steps ahead, 1 KB in one piece.  2048 x 4096 x 11008 takes 67 us
// (2750 TFLOP/s): the products 20 on full CUs (16 cycles each), its 90 MB of
// outputs 13 behind them, prologues, copies and barriers the rest; eight waves on
// twice the tokens, which read a third less from L2, took as long.  Tiles
// of 128 tokens need more than 256 registers.
constexpr int kOuts = 256;
template <int TT, int X>
__global__ __launch_bounds__(256, 2) void mx4_many_kernel(Product p, int gx, int gy) {
    constexpr int kTokens = 16 * TT;
    __shared__ __align__(16) uint8_t c0[TT * 4096], c1[TT * 4096];
    constexpr int NS = (TT + 3) / 4;  // words of the tokens' scales a thread
    __shared__ uint32_t s0[NS * 256], s1[NS * 256];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4,
              c = lane & 15;
    // an XCD takes neighbouring tiles, the tokens' fastest: it reads its part of the weights once
    const int all = gx * gy, xcd = blockIdx.x & 7, at = blockIdx.x >> 3, each = all >> 3, more = all & 7;
    const int pos = xcd * each + min(xcd, more) + at;
    const int bo = pos / gy, bt = pos % gy;
    const int64_t t0 = (int64_t)bt * kTokens;
    const int rowb = p.nb * 16;
    const int64_t left = p.T - t0;
    const int live = (int)(left < kTokens ? left : kTokens);
    const uint32_t tiles = (uint32_t)(live + 15) / 16;
    const auto rx = X == kRows ? llmq_rsrc(p.xc + t0 * rowb, (uint32_t)live * rowb)
                               : llmq_rsrc(p.xc + t0 / 16 * p.words * 4096, tiles * p.words * 4096);
    const int tile0 = bo * 16 + w * 4;
    int so[4];  // the wave's row tiles (its first again past the matrix's end)
    const int base = min(tile0, p.ntiles - 1);
#pragma unroll
    for (int r = 0; r < 4; r++) so[r] = (min(tile0 + r, p.ntiles - 1) - base);
    const auto rw = llmq_rsrc(p.wc + (int64_t)base * p.words * 4096,
                              (uint32_t)min(4, p.ntiles - base) * (uint32_t)p.words * 4096);
    const uint32_t *ws = p.ws + (int64_t)base * p.words * 64 + lane;
    const int groups = p.words;

    auto stage = [&](int g, uint8_t *dst) __attribute__((always_inline)) {  // wave w: step w of the group
#pragma unroll
        for (int t = 0; t < TT; t++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rx, (__attribute__((address_space(3))) void *)(dst + (w * TT + t) * 1024), 16,
                X == kRows ? (16 * t + c) * rowb + q * 16 + (g * 4 + w) * 64
                           : ((t * p.words + g) * 4 + w) * 1024 + lane * 16,
                0, 0, 0);
    };
    // the thread's tokens' scales: asked for at a group's start, put into words at its end
    const uint8_t *xs[NS];
#pragma unroll
    for (int k = 0; k < NS; k++) {
        if constexpr (X == kRows)
            xs[k] = p.xs + (t0 + min((w + 4 * k) * 16 + c, live - 1)) * p.nb;
        else
            xs[k] = p.xs + ((t0 / 16 + min(w + 4 * k, (live - 1) / 16)) * p.words * 64 + lane) * 4;
    }
    uint32_t raw[NS][4];
    auto ask = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NS; k++) {
            if constexpr (X == kRecord) {
                raw[k][0] = *reinterpret_cast<const uint32_t *>(xs[k] + (int64_t)g * 256);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) raw[k][j] = xs[k][min(g * 16 + 4 * j + q, p.nb - 1)];
            }
        }
    };
    auto put = [&](int g, uint32_t *dst) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NS; k++) {
            uint32_t word = raw[k][0];
            if constexpr (X == kRows) {  // 127 past the row's end, as in tail_scales
                word = 0;
#pragma unroll
                for (int j = 0; j < 4; j++) word |= (g * 16 + 4 * j + q < p.nb ? raw[k][j] : 127u) << (8 * j);
            }
            dst[tid + 256 * k] = word;
        }
    };
    v4f acc[4][TT];
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int t = 0; t < TT; t++) acc[r][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    uint4 a[4][4];
    auto weights = [&](int s, uint4 (&dst)[4]) __attribute__((always_inline)) {
        const int k = min(s, 4 * p.words - 1);  // (past the end: loaded and not used)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(rw, lane * 16, (so[r] * 4 * p.words + k) * 1024, 0);
            dst[r] = make_uint4(v[0], v[1], v[2], v[3]);
        }
    };
    uint32_t as[4], an[4];
#pragma unroll
    for (int r = 0; r < 4; r++) as[r] = ws[so[r] * p.words * 64];
    stage(0, c0);
    ask(0);
    put(0, s0);
#pragma unroll
    for (int s = 0; s < 3; s++) weights(s, a[s]);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the first group's copies, which fewer loads follow
    auto group = [&](int g, const uint8_t *cb, uint8_t *nb, const uint32_t *sb, uint32_t *ns)
        __attribute__((always_inline)) {
        // vmcnt(16), lgkmcnt(0): this wave's copies are in, behind which it has asked for the weights of the last
        // group's four steps only (4 loads each), and its reads are done
        __builtin_amdgcn_s_waitcnt(0x4070);
        llmq_lds_barrier();
        // (no branches here: at one, the compiler moves the accumulators about; the last group's next is itself)
        const int next = min(g + 1, groups - 1);
        stage(next, nb);
        ask(next);
#pragma unroll
        for (int r = 0; r < 4; r++) an[r] = ws[(so[r] * p.words + next) * 64];
        __builtin_amdgcn_sched_barrier(0);  // the weights' loads below stay behind the copies
        uint32_t bs[TT];
#pragma unroll
        for (int t = 0; t < TT; t++) bs[t] = sb[t * 64 + lane];
        // U of the tokens' fragments at a time, the next U read while these are multiplied
        constexpr int U = TT == 6 ? 3 : 4, H = TT / U;
        uint4 b[2][U];
        auto read = [&](int h) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < U; t++)
                b[h & 1][t] = *reinterpret_cast<const uint4 *>(cb + (h / H * TT + h % H * U + t) * 1024 + lane * 16);
        };
        read(0);
#pragma unroll
        for (int h = 0; h < 4 * H; h++) {
            const int j = h / H;
            if (h + 1 < 4 * H) read(h + 1);
            if (h % H == 0) weights(g * 4 + j + 3, a[(j + 3) % 4]);
            // (left to itself, the compiler asks for all of these where they are used)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < U; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    acc[r][h % H * U + t] =
                        mma(a[j][r], b[h & 1][t], acc[r][h % H * U + t], (int)as[r], (int)bs[h % H * U + t], j);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) as[r] = an[r];
        put(next, ns);
    };
    int g = 0;
    for (; g + 1 < groups; g += 2) {
        group(g, c0, c1, s0, s1);
        group(g + 1, c1, c0, s1, s0);
    }
    if (g < groups) group(g, c0, c1, s0, s1);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): no copy into LDS is left behind
    // Four outputs a load and a store, whatever their alignment: 2048 x 4096 x 11008 with GELU 67 us, with bias and
    // residual 75; an output at a time they took 106 and 155, and 1024 x 4096 x 11009 53 for 37.  (The waves of the
    // matrix's last outputs look at each four.)
    auto write = [&](auto whole) __attribute__((always_inline)) {
        const int n = decltype(whole)::value ? INT32_MAX : p.n;
        v4f bias[4] = {};
        if (p.flags & LLMQ_BIAS)
#pragma unroll
            for (int r = 0; r < 4; r++) bias[r] = load_four(p.bias, (tile0 + r) * 16 + 4 * q, n);
#pragma unroll
        for (int t = 0; t < TT; t++) {
            if (16 * t + c >= live) continue;
            float *row = p.out + (t0 + 16 * t + c) * p.n;
            v4f there[4];
            if (p.flags & LLMQ_RESID)
#pragma unroll
                for (int r = 0; r < 4; r++) there[r] = load_four(row, (tile0 + r) * 16 + 4 * q, n);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                v4f y = acc[r][t] + bias[r];
                if (p.flags & LLMQ_GELU)
#pragma unroll
                    for (int i = 0; i < 4; i++) y[i] = gelu_of(y[i]);
                if (p.flags & LLMQ_RESID) y = there[r] + y;
                store_four(row, y, (tile0 + r) * 16 + 4 * q, n);
            }
        }
    };
    if ((tile0 + 4) * 16 <= p.n)
        write(std::true_type{});
    else
        write(std::false_type{});
}

int check_shape(const char *name, int64_t rows, int64_t cols) {
    LLMQ_REQUIRE(rows > 0 && cols > 0, "%s: empty matrix", name);
    LLMQ_REQUIRE(cols % 32 == 0, "%s: %lld inputs are no whole blocks of 32", name, (long long)cols);
    LLMQ_REQUIRE(rows <= INT32_MAX - 512 && cols <= 1 << 24, "%s: %lld x %lld matrix (at most 2^24 inputs)", name,
                 (long long)rows, (long long)cols);
    return LLMQ_OK;
}

// A matrix is used on its own GPU, whose memory it is in.
int check_device(const char *name, const llmq_ctx *ctx, const llmq_mat *m) {
    LLMQ_REQUIRE(m->device == ctx->device, "%s: the matrix is on device %d, the context on %d", name, m->device,
                 ctx->device);
    return LLMQ_OK;
}

// Calls that allocate, or copy to or from host memory, cannot be part of a graph.
int check_no_capture(const char *name, const llmq_ctx *ctx) {
    LLMQ_REQUIRE(!ctx_capturing(ctx), "%s: not under graph capture", name);
    return LLMQ_OK;
}

int mx4_alloc(llmq_ctx *ctx, int64_t n, int64_t k, llmq_mat **out) {
    llmq_mat *m = new (std::nothrow) llmq_mat();
    if (!m) return llmq_set_error(LLMQ_ENOMEM, "from_f32_mx4: out of host memory");
    m->device = ctx->device;
    m->kind = MAT_MX4;
    m->bits = 4;
    m->n = n;
    m->k = k;
    m->group = m->group_param = 32;
    m->ntiles = (n + 15) / 16;
    m->CK = (k + 127) / 128;
    m->NG = (m->CK + 3) / 4;
    const size_t cb = (size_t)(m->ntiles * m->NG) * 4096, sb = (size_t)(m->ntiles * m->NG) * 256;
    if (hipMalloc(&m->codes, cb) != hipSuccess || hipMalloc(&m->scales, sb) != hipSuccess) {
        (void)hipGetLastError();
        llmq_mat_free(m);
        return llmq_set_error(LLMQ_ENOMEM, "from_f32_mx4: device allocation of %zu bytes failed", cb + sb);
    }
    if (hipMemsetAsync(m->codes, 0, cb, ctx->stream) != hipSuccess ||
        hipMemsetAsync(m->scales, 127, sb, ctx->stream) != hipSuccess) {
        llmq_mat_free(m);
        return llmq_set_error(LLMQ_EHIP, "from_f32_mx4: clearing the matrix failed");
    }
    *out = m;
    return LLMQ_OK;
}

// Where a matrix keeps row o's block b: index of its 16 code bytes, and of its scale byte.
struct Place {
    int64_t code, scale;
};
Place place_of(const llmq_mat *m, int64_t o, int64_t b) {
    const int64_t tile = o >> 4, step = b >> 2, lane = (o & 15) + 16 * (b & 3);
    return Place{(tile * m->NG * 4 + step) * 64 + lane, ((tile * m->NG + (step >> 2)) * 64 + lane) * 4 + (step & 3)};
}

int check_codes(const char *name, const llmq_ctx *ctx, const void *a, const void *codes, const void *scales, int64_t T,
                int64_t K) {
    LLMQ_REQUIRE(ctx && ((a && codes && scales) || T == 0), "%s: null argument", name);
    LLMQ_REQUIRE(T >= 0 && T <= INT32_MAX && K > 0 && K % 32 == 0 && K <= 1 << 24,
                 "%s: %lld rows of %lld (whole blocks of 32)", name, (long long)T, (long long)K);
    LLMQ_REQUIRE((uintptr_t)codes % 16 == 0, "%s: codes are 16-byte aligned", name);
    return LLMQ_OK;
}

// The grid of a kernel whose workgroups take `each` pieces of `values` values, and pieces a row (0: the rows
// lie together).
struct Pieces {
    int64_t total, grid;
    uint32_t unit;
};
int pieces(const char *name, int64_t T, int64_t K, int64_t ld, int values, int each, Pieces *out) {
    out->total = T * (K / values);
    out->grid = (out->total + each - 1) / each;
    out->unit = ld == K || T == 1 ? 0 : (uint32_t)(K / values);
    LLMQ_REQUIRE(out->grid <= INT32_MAX, "%s: %lld rows of %lld", name, (long long)T, (long long)K);
    return LLMQ_OK;
}

int launch_quantize(llmq_ctx *ctx, const float *x, int64_t ldx, int64_t T, int64_t K, uint8_t *codes,
                    uint8_t *scales) {
    Pieces u;
    RC(pieces("mx4_quantize", T, K, ldx, 4, 256 * 2 * kQuant, &u));
    hipLaunchKernelGGL(mx4_quantize_kernel, dim3((unsigned)u.grid), dim3(256), 0, ctx->stream, x, ldx, u.unit, u.total,
                       reinterpret_cast<uint32_t *>(codes), scales);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

// Waves of a few-token workgroup, and groups of steps each: a wave a group as far as they go.
int few_waves(const llmq_mat *w, int most, int *per) {
    *per = (int)((w->NG + most - 1) / most);
    return (int)((w->NG + *per - 1) / *per);
}

template <int TT, int X>
int launch_few(llmq_ctx *ctx, const Product &p, const llmq_mat *w, size_t front) {
    int per;
    const int waves = few_waves(w, few_most(TT), &per);
    const size_t sums = (size_t)waves * TT * 1024;
    const dim3 grid((unsigned)w->ntiles, (unsigned)((p.T + 16 * TT - 1) / (16 * TT)));
    hipLaunchKernelGGL((mx4_few_kernel<TT, X>), grid, dim3(64 * waves), sums > front ? sums : front, ctx->stream, p,
                       per);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

template <int TT, int X>
int launch_many(llmq_ctx *ctx, const Product &p) {
    const int64_t gx = ((int64_t)p.n + kOuts - 1) / kOuts, gy = (p.T + 16 * TT - 1) / (16 * TT);
    LLMQ_REQUIRE(gx * gy <= INT32_MAX, "mx4_linear: %lld tokens by %d outputs", (long long)p.T, p.n);
    hipLaunchKernelGGL((mx4_many_kernel<TT, X>), dim3((unsigned)(gx * gy)), dim3(256), 0, ctx->stream, p, (int)gx,
                       (int)gy);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

// The kernel by its time, whichever way the tokens are given (their sums are
// then in one order).  Few-token workgroups cost the same each, 1.5 to 3 ns a
// group of 512 inputs, however many there are; the others fill the CUs with few,
// a chain of 1.4 us a group behind 5.5 us.  300 x 4096 x 4096 30.6 us by the
// first and 17.1 by the others, 500 x 1024 x 1024 6.0 and 8.3, 32 x 4096 x 32000
// 25 and 16, 40 x 4096 x 11008 16.1 and 13.7 (a record 10.7 and 13.9): over 280
// sizes of 40 to 500 tokens 0.9 % behind the better of the two in the mean.  Of
// the two large tiles the one whose workgroups, a CU's share of them after one
// another, are done first: 2048 x 4096 x 11008 68 us with 96 tokens, 75.5 with
// 64; 2048 x 11008 x 4096 75 and 69.
template <int X>
int launch_tokens(llmq_ctx *ctx, const Product &p, const llmq_mat *w) {
    const int64_t work = w->ntiles * w->NG, bound = 650 * (w->NG + 3);
    if (p.T <= 16) return launch_few<1, X>(ctx, p, w, 0);
    if (p.T <= 32 && 2 * work <= 3 * bound) return launch_few<2, X>(ctx, p, w, 0);
    if (work * ((p.T + 63) / 64) <= bound) return launch_few<4, X>(ctx, p, w, 0);
    const int64_t gx = (w->n + kOuts - 1) / kOuts;
    auto cost = [&](int64_t tt) { return (gx * ((p.T + 16 * tt - 1) / (16 * tt)) + 255) / 256 * (5 * tt + 6); };
    return cost(6) < cost(4) ? launch_many<6, X>(ctx, p) : launch_many<4, X>(ctx, p);
}

// The product of tokens given as X says: packed rows, a record, or one token's floats x.
template <int X>
int launch_product(llmq_ctx *ctx, const uint8_t *codes, const uint8_t *scales, const float *x, const llmq_mat *w,
                   int64_t T, float *out, const float *bias, int flags) {
    Product p;
    p.xc = codes;
    p.xs = scales;
    p.x = x;
    p.wc = w->codes;
    p.ws = reinterpret_cast<const uint32_t *>(w->scales);
    p.T = T;
    p.n = (int)w->n;
    p.nb = (int)(w->k / 32);
    p.steps = (int)w->CK;
    p.words = (int)w->NG;
    p.ntiles = (int)w->ntiles;
    p.out = out;
    p.bias = bias;
    p.flags = flags;
    if constexpr (X == kFloats)
        return launch_few<1, kFloats>(ctx, p, w, (size_t)w->NG * (16 + 256));
    else
        return launch_tokens<X>(ctx, p, w);
}

int check_epilogue(const char *name, const float *out, const float *bias, int64_t T, int flags) {
    LLMQ_REQUIRE(out || T == 0, "%s: null output", name);
    LLMQ_REQUIRE(!(flags & ~(LLMQ_BIAS | LLMQ_GELU | LLMQ_RESID)), "%s: flags %d", name, flags);
    LLMQ_REQUIRE(!(flags & LLMQ_BIAS) || bias, "%s: null bias", name);
    return LLMQ_OK;
}

}  // namespace

// A record of T tokens of K inputs: whole tiles of 16 and groups of 512.
int64_t mx4_record_bytes(int64_t T, int64_t K) {
    const int64_t values = ((T + 15) / 16 * 16) * ((K + 511) / 512 * 512);
    return values / 2 + values / 32;
}

int launch_mx4_linear(llmq_ctx *ctx, const llmq_mat *w, const float *x, int64_t T, float *out, const float *bias,
                      int flags, void *rec, int64_t rec_cap) {
    RC(check_epilogue("linear", out, bias, T, flags));
    LLMQ_REQUIRE(T >= 0 && T <= INT32_MAX && (x || T == 0), "linear: %lld microscaled tokens", (long long)T);
    RC(check_device("linear", ctx, w));
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    // one token's row fits LDS beside the sums
    if (T == 1 && w->NG * (16 + 256) <= 65536)
        return launch_product<kFloats>(ctx, nullptr, nullptr, x, w, 1, out, bias, flags);
    const int64_t need = mx4_record_bytes(T, w->k);
    if (rec_cap < 0) {
        // the workspace is one for the context: two graphs that held it could not run side by side
        LLMQ_REQUIRE(!ctx_capturing(ctx),
                     "linear: under graph capture a microscaled matrix takes llmq_mx4_quantize and llmq_mx4_linear");
        RC(ctx_workspace(ctx, (size_t)need, &rec));
    } else {
        LLMQ_REQUIRE(need <= rec_cap,
                     "linear_noalloc: %lld tokens x %lld inputs need %lld bytes of scratch, the maximum is %lld",
                     (long long)T, (long long)w->k, (long long)need, (long long)rec_cap);
    }
    const int64_t tiles = (T + 15) / 16;
    uint8_t *codes = static_cast<uint8_t *>(rec), *scales = codes + tiles * w->NG * 4096;
    for (int64_t done = 0; done < tiles; done += 65535) {
        const int64_t some = tiles - done < 65535 ? tiles - done : 65535;
        hipLaunchKernelGGL(mx4_record_kernel, dim3((unsigned)w->NG, (unsigned)some), dim3(256), 0, ctx->stream,
                           x + done * 16 * w->k, T - done * 16, (int)(w->k / 32), (int)w->NG,
                           reinterpret_cast<uint32_t *>(codes + done * w->NG * 4096),
                           reinterpret_cast<uint32_t *>(scales + done * w->NG * 256));
        LLMQ_HIP(hipGetLastError());
    }
    return launch_product<kRecord>(ctx, codes, scales, nullptr, w, T, out, bias, flags);
}

int mx4_dequant_row(llmq_ctx *ctx, const llmq_mat *m, int64_t row, float *dst) {
    RC(check_device("dequant_row", ctx, m));
    RC(check_no_capture("dequant_row", ctx));
    DeviceGuard guard(ctx);
    try {
        const int64_t nb = m->k / 32, tile = row >> 4, r = row & 15;
        std::vector<uint8_t> c((size_t)m->NG * 4096), s((size_t)m->NG * 256);
        LLMQ_HIP(hipMemcpyAsync(c.data(), m->codes + tile * m->NG * 4096, c.size(), hipMemcpyDeviceToHost,
                                ctx->stream));
        LLMQ_HIP(hipMemcpyAsync(s.data(), reinterpret_cast<const uint8_t *>(m->scales) + tile * m->NG * 256, s.size(),
                                hipMemcpyDeviceToHost, ctx->stream));
        LLMQ_HIP(hipStreamSynchronize(ctx->stream));
        static const float val[16] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f,
                                      -0.0f, -0.5f, -1.0f, -1.5f, -2.0f, -3.0f, -4.0f, -6.0f};
        for (int64_t b = 0; b < nb; b++) {
            const Place at = place_of(m, r, b);  // the row within its own tile
            const int e = s[(size_t)at.scale];
            const float sc = e == 255 ? NAN : ldexpf(1.0f, e - 127);
            for (int j = 0; j < 32; j++)
                dst[b * 32 + j] = val[(c[(size_t)at.code * 16 + j / 2] >> (4 * (j & 1))) & 15] * sc;
        }
    } catch (const std::bad_alloc &) {
        return llmq_set_error(LLMQ_ENOMEM, "dequant_row: out of host memory");
    }
    return LLMQ_OK;
}

extern "C" {

int llmq_mx4_quantize(llmq_ctx *ctx, const float *x, int64_t ldx, int64_t T, int64_t K, uint8_t *codes,
                      uint8_t *scales) {
    RC(check_codes("mx4_quantize", ctx, x, codes, scales, T, K));
    LLMQ_REQUIRE(ldx >= K, "mx4_quantize: rows of %lld floats %lld apart", (long long)K, (long long)ldx);
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    return launch_quantize(ctx, x, ldx, T, K, codes, scales);
}

int llmq_mx4_dequantize(llmq_ctx *ctx, const uint8_t *codes, const uint8_t *scales, int64_t T, int64_t K, float *out,
                        int64_t ldo) {
    RC(check_codes("mx4_dequantize", ctx, out, codes, scales, T, K));
    LLMQ_REQUIRE(ldo >= K, "mx4_dequantize: rows of %lld floats %lld apart", (long long)K, (long long)ldo);
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    Pieces u;
    RC(pieces("mx4_dequantize", T, K, ldo, 8, 256 * kQuant, &u));
    hipLaunchKernelGGL(mx4_dequantize_kernel, dim3((unsigned)u.grid), dim3(256), 0, ctx->stream,
                       reinterpret_cast<const uint32_t *>(codes), scales, u.unit, u.total, out, ldo);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

int llmq_mat_from_f32_mx4_device(llmq_ctx *ctx, const float *src, int64_t rows, int64_t cols, int reduce_rows,
                                 llmq_mat **out) {
    LLMQ_REQUIRE(ctx && src && out, "from_f32_mx4: null argument");
    const int64_t n = reduce_rows ? cols : rows, k = reduce_rows ? rows : cols;
    RC(check_shape("from_f32_mx4", n, k));
    const int64_t nb = k / 32, grid = (n * nb + 255) / 256;
    LLMQ_REQUIRE(grid <= INT32_MAX, "from_f32_mx4: %lld x %lld matrix", (long long)n, (long long)k);
    RC(check_no_capture("from_f32_mx4", ctx));
    DeviceGuard guard(ctx);
    llmq_mat *m = nullptr;
    RC(mx4_alloc(ctx, n, k, &m));
    hipLaunchKernelGGL(mx4_weights_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, src, cols, reduce_rows, n,
                       nb, m->NG, reinterpret_cast<uint4 *>(m->codes), reinterpret_cast<uint8_t *>(m->scales));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        llmq_mat_free(m);
        return llmq_set_error(LLMQ_EHIP, "from_f32_mx4: %s", hipGetErrorString(e));
    }
    *out = m;
    return LLMQ_OK;
}

int llmq_mat_from_f32_mx4(llmq_ctx *ctx, const float *src, int64_t rows, int64_t cols, int reduce_rows,
                          llmq_mat **out) {
    LLMQ_REQUIRE(ctx && src && out, "from_f32_mx4: null argument");
    RC(check_shape("from_f32_mx4", reduce_rows ? cols : rows, reduce_rows ? rows : cols));
    RC(check_no_capture("from_f32_mx4", ctx));
    DeviceGuard guard(ctx);
    float *d = nullptr;
    const size_t bytes = sizeof(float) * (size_t)rows * (size_t)cols;
    if (hipMalloc(&d, bytes) != hipSuccess) {
        (void)hipGetLastError();
        return llmq_set_error(LLMQ_ENOMEM, "from_f32_mx4: staging %zu bytes", bytes);
    }
    int rc = LLMQ_OK;
    if (hipMemcpyAsync(d, src, bytes, hipMemcpyHostToDevice, ctx->stream) != hipSuccess)
        rc = llmq_set_error(LLMQ_EHIP, "from_f32_mx4: copy to the device failed");
    llmq_mat *m = nullptr;
    if (rc == LLMQ_OK) rc = llmq_mat_from_f32_mx4_device(ctx, d, rows, cols, reduce_rows, &m);
    const hipError_t e = hipStreamSynchronize(ctx->stream);
    if (rc == LLMQ_OK && e != hipSuccess) {
        llmq_mat_free(m);
        rc = llmq_set_error(LLMQ_EHIP, "from_f32_mx4: %s", hipGetErrorString(e));
    }
    hipFree(d);
    if (rc == LLMQ_OK) *out = m;
    return rc;
}

int llmq_mat_restore_mx4(llmq_ctx *ctx, int64_t rows, int64_t cols, const uint8_t *codes, const uint8_t *scales,
                         llmq_mat **out) {
    LLMQ_REQUIRE(ctx && codes && scales && out, "restore_mx4: null argument");
    RC(check_shape("restore_mx4", rows, cols));
    RC(check_no_capture("restore_mx4", ctx));
    DeviceGuard guard(ctx);
    llmq_mat *m = nullptr;
    RC(mx4_alloc(ctx, rows, cols, &m));
    int rc = LLMQ_OK;
    try {
        const int64_t nb = cols / 32;
        std::vector<uint8_t> c((size_t)(m->ntiles * m->NG) * 4096, 0), s((size_t)(m->ntiles * m->NG) * 256, 127);
        for (int64_t o = 0; o < rows; o++)
            for (int64_t b = 0; b < nb; b++) {
                const Place at = place_of(m, o, b);
                for (int j = 0; j < 16; j++) c[(size_t)at.code * 16 + j] = codes[(o * nb + b) * 16 + j];
                s[(size_t)at.scale] = scales[o * nb + b];
            }
        if (hipMemcpyAsync(m->codes, c.data(), c.size(), hipMemcpyHostToDevice, ctx->stream) != hipSuccess ||
            hipMemcpyAsync(m->scales, s.data(), s.size(), hipMemcpyHostToDevice, ctx->stream) != hipSuccess ||
            hipStreamSynchronize(ctx->stream) != hipSuccess)
            rc = llmq_set_error(LLMQ_EHIP, "restore_mx4: copy to the device failed");
    } catch (const std::bad_alloc &) {
        rc = llmq_set_error(LLMQ_ENOMEM, "restore_mx4: out of host memory");
    }
    if (rc != LLMQ_OK) {
        llmq_mat_free(m);
        return rc;
    }
    *out = m;
    return LLMQ_OK;
}

int llmq_mat_export_mx4(llmq_ctx *ctx, const llmq_mat *m, uint8_t *codes, uint8_t *scales) {
    LLMQ_REQUIRE(ctx && m && m->kind == MAT_MX4, "export_mx4: not a microscaled matrix");
    RC(check_device("export_mx4", ctx, m));
    RC(check_no_capture("export_mx4", ctx));
    DeviceGuard guard(ctx);
    try {
        std::vector<uint8_t> c((size_t)(m->ntiles * m->NG) * 4096), s((size_t)(m->ntiles * m->NG) * 256);
        LLMQ_HIP(hipMemcpyAsync(c.data(), m->codes, c.size(), hipMemcpyDeviceToHost, ctx->stream));
        LLMQ_HIP(hipMemcpyAsync(s.data(), m->scales, s.size(), hipMemcpyDeviceToHost, ctx->stream));
        LLMQ_HIP(hipStreamSynchronize(ctx->stream));
        const int64_t nb = m->k / 32;
        for (int64_t o = 0; o < m->n; o++)
            for (int64_t b = 0; b < nb; b++) {
                const Place at = place_of(m, o, b);
                if (codes)
                    for (int j = 0; j < 16; j++) codes[(o * nb + b) * 16 + j] = c[(size_t)at.code * 16 + j];
                if (scales) scales[o * nb + b] = s[(size_t)at.scale];
            }
    } catch (const std::bad_alloc &) {
        return llmq_set_error(LLMQ_ENOMEM, "export_mx4: out of host memory");
    }
    return LLMQ_OK;
}

int llmq_mx4_linear(llmq_ctx *ctx, float *out, const uint8_t *codes, const uint8_t *scales, const llmq_mat *w,
                    const float *bias, int64_t T, int64_t IN, int64_t OUT, int flags) {
    LLMQ_REQUIRE(w && w->kind == MAT_MX4, "mx4_linear: not a microscaled matrix");
    LLMQ_REQUIRE(w->k == IN && w->n == OUT, "mx4_linear: matrix is %lldx%lld, call says IN=%lld OUT=%lld",
                 (long long)w->n, (long long)w->k, (long long)IN, (long long)OUT);
    RC(check_codes("mx4_linear", ctx, out, codes, scales, T, IN));
    RC(check_device("mx4_linear", ctx, w));
    RC(check_epilogue("mx4_linear", out, bias, T, flags));
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    return launch_product<kRows>(ctx, codes, scales, nullptr, w, T, out, bias, flags);
}

}  // extern "C"
