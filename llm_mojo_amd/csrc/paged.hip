// A key / value cache in pages, and attention of one new token a sequence
// over it (include/llmq.h, llmq_pkv_*).
//
// Device layout, a layer and a page at a time: keys [head][position][hd],
// values [head][block][hd][slot] (paged_plan.h), and for int8 the float32
// scales of keys and values [head][position].
#include <math.h>

#include <new>
#include <type_traits>

#include "common.h"
#include "paged_plan.h"

struct llmq_pkv {
    int device = 0, type = 0, n_layer = 0, page = 0, n_kv = 0, hd = 0;
    int64_t n_pages = 0;
    uint8_t *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;  // int8 only
    int elem() const { return type == LLMQ_PKV_INT8 ? 1 : 2; }
    int64_t rows() const { return (int64_t)n_layer * n_pages * n_kv * page; }  // positions x heads held
};

namespace {

constexpr int B = pkv::kBlock;

// One layer of a cache as a kernel takes it.
struct Layer {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;
    int64_t width, pages;
    int page, n_kv;
};

// int8 codes are kept plus 128: 0x64 above such a byte is the float16 1024 +
// code + 128, which is how the attention widens them.
constexpr int kBias = 128;

// A head's row (position 0 of its page) in units of positions.
__device__ __forceinline__ int64_t head_row(const Layer &c, int page, int head) {
    return ((int64_t)page * c.n_kv + head) * c.page;
}

// QuantKV.store's quantisation of a row (kvcache.mojo:333-342), but for the
// last bit of a scale: s = max|x| / 127 as a product with the rounded 1 / 127,
// codes round(x (1 / s)) away from zero at ties, kept plus kBias.  A row with a
// NaN or an infinity (largest: infinity) gets the scale NaN; one below 2^-120,
// whose reciprocal scale is infinite, is a row of zeros.  Their scale is 0, not
// QuantKV's 1: the attention's weights carry the scales relative to the
// largest, beside which those of small values would vanish.
__device__ __forceinline__ float row_scale(float largest) {
    if (largest == INFINITY) return __uint_as_float(0x7fc00000u);
    return largest < 0x1p-120f ? 0.0f : largest * (1.0f / 127.0f);
}
__device__ __forceinline__ float inverse_of(float scale) { return scale > 0.0f ? 1.0f / scale : 0.0f; }
// Truncating after adding the float below a half, with the sign of y, rounds
// any |y| < 2^22 as roundf does (a half itself would round 0.5 - 2^-25 up), in
// a third of its instructions: storing 17.7k x 8 x 128 takes 40.8 us, 42.8 with roundf.
__device__ __forceinline__ int row_code(float x, float inv) {
    const float y = x * inv;
    return (int)__builtin_amdgcn_fmed3f(y + copysignf(0.49999997f, y), -127.0f, 127.0f) + kBias;  // (NaN: -127)
}

__device__ __forceinline__ uint16_t half_bits(float x) {
    // nearest even; finite values past the range become its ends
    const float lim = fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    return __half_as_ushort(__float2half_rn(lim));
}

// A row's codes (int8, or float16 bits) and scale, dimensions lane + 64 i.
template <int HD, int ELEM>
__device__ __forceinline__ float encode_row(const float (&x)[HD / 64], int (&code)[HD / 64]) {
    if constexpr (ELEM == 1) {
        float m = 0.0f, bad = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 64; i++) {
            m = fmaxf(m, fabsf(x[i]));
            bad += x[i] - x[i];  // NaN for NaN and infinities
        }
        m = llmq_wave_max_all(bad != 0.0f || bad != bad ? INFINITY : m);
        const float s = row_scale(m), inv = inverse_of(s);
#pragma unroll
        for (int i = 0; i < HD / 64; i++) code[i] = row_code(x[i], inv);
        return s;
    } else {
#pragma unroll
        for (int i = 0; i < HD / 64; i++) code[i] = half_bits(x[i]);
        return 1.0f;
    }
}

// One wave writes the key and value row of (token, head); the codes stay with it.
template <int HD, int ELEM>
struct NewRow {
    int k[HD / 64], v[HD / 64];
    float ks, vs;
};
template <int HD, int ELEM>
__device__ __forceinline__ NewRow<HD, ELEM> store_row(const Layer &c, int page, int off, int head,
                                                      const float (&kx)[HD / 64], const float (&vx)[HD / 64],
                                                      int lane) {
    const int64_t row = head_row(c, page, head) + off;
    const int64_t vrow = (head_row(c, page, head) + off / B * B) * HD;  // the block's first element
    const int slot = pkv::value_slot(off % B);
    NewRow<HD, ELEM> x;
    x.ks = encode_row<HD, ELEM>(kx, x.k);
    x.vs = encode_row<HD, ELEM>(vx, x.v);
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        const int64_t kat = row * HD + lane + 64 * i, vat = vrow + (int64_t)(lane + 64 * i) * B + slot;
        if constexpr (ELEM == 1) {
            c.k[kat] = (uint8_t)x.k[i];
            c.v[vat] = (uint8_t)x.v[i];
        } else {
            reinterpret_cast<uint16_t *>(c.k)[kat] = (uint16_t)x.k[i];
            reinterpret_cast<uint16_t *>(c.v)[vat] = (uint16_t)x.v[i];
        }
    }
    if (ELEM == 1 && lane == 0) {
        c.ks[row] = x.ks;
        c.vs[row] = x.vs;
    }
    return x;
}

// Rows of a call to or from the cache: a workgroup kRows rows of one head,
// eight lanes a row, the values through LDS so that both sides see whole
// lines: the floats a row at a time, the cache a dimension's slots at a time
// (neighbouring rows are mostly neighbouring positions).
constexpr int kRows = 32, kLanes = 8;

// Where row t's position is: its first element in the keys (units of rows),
// and in the values the element of dimension 0; -1: nowhere.
struct Dest {
    int64_t row, value;
};
template <int HD>
__device__ __forceinline__ Dest dest_of(const Layer &c, const int32_t *seq, const int32_t *pos, int64_t n_seq,
                                        int64_t t, int64_t T, int head) {
    Dest d{-1, -1};
    if (t >= T) return d;
    const int s = seq[t], p = pos[t];
    if (s < 0 || s >= n_seq) return d;
    const int page = pkv::page_of(c.table + s * c.width, c.width, c.page, c.pages, p);
    if (page < 0) return d;
    const int off = p % c.page;
    d.row = head_row(c, page, head) + off;
    d.value = (d.row - off % B) * HD + pkv::value_slot(off % B);
    return d;
}

// The rows of workgroup i: from the first row of its kRows that begins a
// block or does not follow the row before, to the next workgroup's first such.
// So a block whose positions are neighbouring rows is one workgroup's, which
// writes its lines whole, wherever the rows begin.  At most 2 kRows - 1 of
// them: neighbouring rows begin a block every kRows.
struct Span {
    int64_t lo, hi;
};
__device__ __forceinline__ Span rows_of(const int32_t *seq, const int32_t *pos, int64_t i, int64_t T, int lane) {
    static_assert(kRows == B, "a workgroup's rows and a block's");
    const int64_t t = i * kRows + lane;
    bool first = false;
    if (t < T) {
        const int p = pos[t];
        first = t == 0 || p % B == 0 || seq[t - 1] != seq[t] || (uint32_t)pos[t - 1] + 1u != (uint32_t)p;
    }
    const uint64_t all = __ballot(first);
    const uint32_t here = (uint32_t)all, next = (uint32_t)(all >> 32);
    const int64_t end = (i + 1) * kRows;
    Span s;
    s.hi = next ? end + __ffs(next) - 1 : (end + kRows < T ? end + kRows : T);
    s.lo = here ? i * kRows + __ffs(here) - 1 : s.hi;
    if (s.hi > T) s.hi = T;
    return s;
}

// Maximum over the eight lanes of a row.
__device__ __forceinline__ float eighth_max(float v) {
    v = fmaxf(v, llmq_dppf<0xB1>(v));
    v = fmaxf(v, llmq_dppf<0x4E>(v));
    return fmaxf(v, llmq_dppf<0x141>(v));  // row_half_mirror
}

struct Floats4 {
    float x[4];
} __attribute__((packed, aligned(4)));

// llmq_pkv_store.  Bound by reading the floats and writing the cache: 17.7k
// positions x 8 x 128 to float16 49 us (218 MB, 4.4 TB/s; 62 with plain loads),
// 476 x 12 x 64 to int8 5.
template <int HD, int ELEM>
__global__ __launch_bounds__(kRows *kLanes) void pkv_store_kernel(Layer c, const float *__restrict__ k,
                                                                  const float *__restrict__ v, int64_t ld, int64_t T,
                                                                  const int32_t *__restrict__ seq,
                                                                  const int32_t *__restrict__ pos, int64_t n_seq) {
    constexpr int NP = HD / 32, STRIDE = HD * ELEM + 4;  // fours of a lane; bytes of a row in LDS
    __shared__ __align__(4) uint8_t vt[kRows * STRIDE];
    __shared__ int64_t at[kRows];
    const int tid = threadIdx.x, row = tid / kLanes, j = tid % kLanes, head = blockIdx.y;
    const Span span = rows_of(seq, pos, blockIdx.x, T, tid & 63);
    for (int64_t begin = span.lo; begin < span.hi; begin += kRows) {
        if (begin > span.lo) __syncthreads();  // the rows before are through
        const int64_t t = begin + row;
        const Dest d = dest_of<HD>(c, seq, pos, n_seq, t, span.hi, head);
        if (j == 0) at[row] = d.value;
        if (d.row >= 0) {
            const float *src[2] = {k + t * ld + head * HD, v + t * ld + head * HD};
            float x[2][NP][4];
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < NP; i++)
                    llmq_load4_once(src[s] + 32 * i + 4 * j, x[s][i]);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint8_t *keys = s == 0 ? c.k + d.row * HD * ELEM : vt + row * STRIDE;
                if constexpr (ELEM == 1) {
                    float m = 0.0f, bad = 0.0f;
#pragma unroll
                    for (int i = 0; i < NP; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            m = fmaxf(m, fabsf(x[s][i][e]));
                            bad += x[s][i][e] - x[s][i][e];  // NaN for NaN and infinities
                        }
                    m = eighth_max(bad != 0.0f || bad != bad ? INFINITY : m);
                    const float scale = row_scale(m), inv = inverse_of(scale);
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        uint32_t u = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) u |= (uint32_t)row_code(x[s][i][e], inv) << (8 * e);
                        *reinterpret_cast<uint32_t *>(keys + 32 * i + 4 * j) = u;
                    }
                    if (j == 0) (s == 0 ? c.ks : c.vs)[d.row] = scale;
                } else {
#pragma unroll
                    for (int i = 0; i < NP; i++) {
                        uint32_t *u = reinterpret_cast<uint32_t *>(keys + 64 * i + 8 * j);
                        u[0] = half_bits(x[s][i][0]) | (uint32_t)half_bits(x[s][i][1]) << 16;
                        u[1] = half_bits(x[s][i][2]) | (uint32_t)half_bits(x[s][i][3]) << 16;
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < kRows * HD; i += kRows * kLanes) {
            const int e = i % kRows, dim = i / kRows;
            if (at[e] < 0) continue;
            if constexpr (ELEM == 1)
                c.v[at[e] + dim * B] = vt[e * STRIDE + dim];
            else
                reinterpret_cast<uint16_t *>(c.v)[at[e] + dim * B] =
                    *reinterpret_cast<const uint16_t *>(vt + e * STRIDE + 2 * dim);
        }
    }
}

// llmq_pkv_fetch; zeros where the cache has no row.  The same rows back: 39 us
// (5.5 TB/s) and 4.3.
template <int HD, int ELEM>
__global__ __launch_bounds__(kRows *kLanes) void pkv_fetch_kernel(Layer c, float *__restrict__ k,
                                                                  float *__restrict__ v, int64_t ld, int64_t T,
                                                                  const int32_t *__restrict__ seq,
                                                                  const int32_t *__restrict__ pos, int64_t n_seq) {
    constexpr int NP = HD / 32, STRIDE = HD * ELEM + 4;
    __shared__ __align__(4) uint8_t vt[kRows * STRIDE];
    __shared__ int64_t at[kRows];
    const int tid = threadIdx.x, row = tid / kLanes, j = tid % kLanes, head = blockIdx.y;
    const Span span = rows_of(seq, pos, blockIdx.x, T, tid & 63);
    for (int64_t begin = span.lo; begin < span.hi; begin += kRows) {
        if (begin > span.lo) __syncthreads();  // the rows before are through
        const int64_t t = begin + row;
        const Dest d = dest_of<HD>(c, seq, pos, n_seq, t, span.hi, head);
        if (j == 0) at[row] = d.value;
        uint32_t key[NP][ELEM];
        float ks = 1.0f, vs = 1.0f;
        if (d.row >= 0) {
#pragma unroll
            for (int i = 0; i < NP; i++)
#pragma unroll
                for (int e = 0; e < ELEM; e++)
                    key[i][e] = *reinterpret_cast<const uint32_t *>(c.k + (d.row * HD + 32 * i + 4 * j) * ELEM + 4 * e);
            if constexpr (ELEM == 1) {
                ks = c.ks[d.row];
                vs = c.vs[d.row];
            }
        }
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < kRows * HD; i += kRows * kLanes) {
            const int e = i % kRows, dim = i / kRows;
            if (at[e] < 0) continue;
            if constexpr (ELEM == 1)
                vt[e * STRIDE + dim] = c.v[at[e] + dim * B];
            else
                *reinterpret_cast<uint16_t *>(vt + e * STRIDE + 2 * dim) =
                    reinterpret_cast<const uint16_t *>(c.v)[at[e] + dim * B];
        }
        __syncthreads();
        if (t >= span.hi) continue;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            Floats4 x{}, y{};
            if (d.row >= 0)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int dim = 32 * i + 4 * j + e;
                    if constexpr (ELEM == 1) {
                        x.x[e] = (float)((int)((key[i][0] >> (8 * e)) & 255) - kBias) * ks;
                        y.x[e] = (float)((int)vt[row * STRIDE + dim] - kBias) * vs;
                    } else {
                        x.x[e] = __half2float(__ushort_as_half((uint16_t)(key[i][e >> 1] >> (16 * (e & 1)))));
                        y.x[e] = __half2float(
                            __ushort_as_half(*reinterpret_cast<const uint16_t *>(vt + row * STRIDE + 2 * dim)));
                    }
                }
            *reinterpret_cast<Floats4 *>(k + t * ld + head * HD + 32 * i + 4 * j) = x;
            *reinterpret_cast<Floats4 *>(v + t * ld + head * HD + 32 * i + 4 * j) = y;
        }
    }
}

struct Attend {
    float *out;
    int64_t ldo;
    const float *q, *k, *v;  // k, v: the new token's rows (step), or null
    int64_t ldq;
    const int32_t *len;  // positions a row attends to (step: its new token's position, -1 for no token)
    int n_head;
    float scale, cap;
    const float *slopes;
    int rows, tiles, columns;  // columns 0: a workgroup a row
    uint32_t least;            // of the plan
    int2 *meta;   // [row]: first slot, segments
    float2 *ml;   // [slot][head]: reference, sum
    float *sums;  // [slot][head][hd]
};

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;
// Cache policy of loads whose lines are read once (nt): 342 MB of float16 64.4 us with it, 70.5 without; 1118 MB of
// int8 221 and 226.
constexpr int kOnce = 2;

// Eight int8 codes as float16, exactly: byte u = code + 128 under the
// exponent byte 0x64 is 1024 + u, less 1152.
__device__ __forceinline__ h8 halves(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        h2 h[4];
        h8 v;
    } r;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - off;
    return r.v;
}

__device__ __forceinline__ h8 as_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    union {
        uint32_t u[4];
        h8 v;
    } r;
    r.u[0] = a;
    r.u[1] = b;
    r.u[2] = c;
    r.u[3] = d;
    return r.v;
}

// tanh without branches, to 2^-23 of 1: ref_tanhf's polynomial below 0.625,
// 1 - 2 / (e^(2|y|) + 1) above.
__device__ __forceinline__ float tanh_select(float y) {
    const float a = fabsf(y), s = y * y;
    float p = 0.002148991f;
    p = fmaf(p, s, -0.00818467f);
    p = fmaf(p, s, 0.021704003f);
    p = fmaf(p, s, -0.053947456f);
    p = fmaf(p, s, 0.13333212f);
    p = fmaf(p, s, -0.3333333f);
    p = fmaf(p * s, a, a);
    const float e = __builtin_amdgcn_exp2f(a * (2.0f * kLog2e));
    const float t = fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return copysignf(a < 0.625f ? p : t, y);
}

// Maximum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quarters_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x),
                   hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ int64_t row_len(const Layer &c, const Attend &a, int64_t r) {
    const int64_t n = a.len[r];
    return pkv::clamp_len(a.k ? n + 1 : n, c.width, c.page);
}

// Sums over a wave's lanes up to each (row_shr 1, 2, 4, 8, then the rows before).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31
}

// The segment of a slot: blocks b0 .. b1 - 1 of a row of `count` segments
// (none: b0 = b1 = 0).  Every wave finds it by itself from the rows' lengths
// (a.rows <= kPlanRows), a lane the same number of neighbouring rows.
struct Part {
    int row, b0, b1, count;
};
__device__ __forceinline__ Part find_part(const Layer &c, const Attend &a, uint32_t slot, int lane) {
    constexpr int N = pkv::kPlanRows / 64;
    const int each = (a.rows + 63) >> 6;
    uint32_t nb[N], segs[N], sum = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i >= each) break;
        const int r = lane * each + i;
        nb[i] = r < a.rows ? (uint32_t)((row_len(c, a, r) + B - 1) / B) : 0;
        sum += nb[i];
    }
    const uint32_t per = pkv::per_of(__builtin_amdgcn_readlane(wave_scan(sum), 63), a.columns, a.least);
    sum = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i >= each) break;
        segs[i] = pkv::segments_of(nb[i], per);
        sum += segs[i];
    }
    const uint32_t end = wave_scan(sum);
    const uint64_t who = __ballot(slot < end && slot >= end - sum);
    Part p{0, 0, 0, 0};
    if (who == 0) return p;
    uint32_t left = slot - (end - sum), row = 0, n = 0, segments = 1, index = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i >= each) break;
        if (!found && left < segs[i]) {
            found = true;
            row = lane * each + i;
            n = nb[i];
            segments = segs[i];
            index = left;
        }
        left -= segs[i];  // (not looked at once found)
    }
    const int l = __ffsll((unsigned long long)who) - 1;
    n = __builtin_amdgcn_readlane(n, l);
    const uint32_t size = pkv::segment_blocks(n, __builtin_amdgcn_readlane(segments, l));
    const uint32_t lo = __builtin_amdgcn_readlane(index, l) * size;
    if (lo >= n) return p;
    p.row = __builtin_amdgcn_readlane(row, l);
    p.b0 = (int)lo;
    p.b1 = (int)(n < lo + size ? n : lo + size);
    p.count = (int)pkv::segments_of(n, size);
    return p;
}

struct Float8 {
    float x[8];
} __attribute__((packed, aligned(4)));

// A table entry by a scalar load, which does not wait for the vector loads in flight.
__device__ __forceinline__ int table_at(const int32_t *p) {
    return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p;
}

// Attention of one token over what a column has of the rows: up to 8 query
// heads of one cached head, on the fp16 matrix cores.
//
// Scores: K (16 positions x 32 dimensions) times the queries as 16 columns,
// columns 0-7 their float16 roundings and 8-15 what those leave times 2^11
// (the keys are exact), so columns n and n ^ 8 add up to a score, in lane n
// for positions 4 (lane / 16) + 0..3 of the tile.  A head's queries are put by
// a power of two to where the largest is just below float16's end, 2^15: each
// is held to 2^-23 of itself, and to 2^-50 of the largest.  Values:
// the weights are already where the second product wants its rows: row n
// holds head n's weights as float16, row n ^ 8 what is left times 2^11, and
// the slots of paged_plan.h give the values in the same order, so nothing is
// moved between lanes.  For int8 a weight is p times the value's scale.
//
// Weights are put near float16's upper end by a power of two: for float16 a
// constant, for int8 one a head that follows its largest weight so far (not
// its largest scale: a large value behind a low score would take the bits of
// all others).  So a weight is held to 2^-22 of itself, and to 2^-48 of its
// head's largest.
//
// The reference of a head's exponentials is moved (and the sums rescaled)
// only when a score passes it by 1, which is rare after the first blocks, as
// is a weight that outgrows its power of two by 4.
// Scores are compared and taken by their difference from it, which is exact
// where it matters: the reference times log2 e would be off by whole units
// from 2^24 on, and infinite above 2.3e38.
// Each wave keeps its own and reads every fourth block; they are put
// together through LDS.  A wave's next keys are on their way while it forms
// the weights, its next values while it scores.
//
// Bound by reading the cache: 4 rows of 9001-32768 float16 positions, 8 heads
// of 128 and 32 queries, 342 MB in 57.5 us (5.9 TB/s); 64 rows of 130-16384
// int8, 1118 MB in 198 (5.6; a plain read of as many bytes 187).  One row of
// 477 and 12 heads of 64 takes 8.3, a chain of loads: lengths and table, keys,
// values.  Eight waves a workgroup were slower (75 and 254 us beside the 64
// and 221 of four), as were blocks of 64 int8 positions (260 registers).
template <int HD, int ELEM>
__global__ __launch_bounds__(64 * pkv::kWaves, 3) void pkv_attend_kernel(Layer c, Attend a) {
    constexpr int NT = B / 16, NC = HD * ELEM / 64, NF = HD / 32, ND = HD / 16, NV = 2 * ELEM;
    constexpr int kBytes = B * HD * ELEM;  // of a block's keys, and of its values
    __shared__ __align__(16) uint8_t fresh[2][HD * ELEM];  // the new token's key and value
    __shared__ float2 wml[pkv::kWaves][8];
    __shared__ float wsum[pkv::kWaves][8][HD];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15,
              q = lane >> 4;
    const int kvh = blockIdx.y / a.tiles, G = a.n_head / c.n_kv, t0 = blockIdx.y % a.tiles * 8;
    const int h0 = kvh * G + t0, hn = min(8, G - t0);
    const int bpp = c.page / B;
    const bool low = n >= 8;

    const uint32_t slot = blockIdx.z * 8 + blockIdx.x;
    int64_t r = slot;
    int b0 = 0, b1 = 0, count = 0;
    if (a.columns) {
        const Part part = find_part(c, a, slot, lane);
        r = __builtin_amdgcn_readfirstlane(part.row);
        b0 = __builtin_amdgcn_readfirstlane(part.b0);
        b1 = __builtin_amdgcn_readfirstlane(part.b1);
        count = __builtin_amdgcn_readfirstlane(part.count);
        if (b0 == b1) return;  // the same for the whole workgroup
    } else if (r >= a.rows) {
        return;
    }
    const int32_t *table = c.table + r * c.width;
    const int64_t told = (int64_t)a.len[r] + (a.k ? 1 : 0), len = uniform64(pkv::clamp_len(told, c.width, c.page));
    const int nb = (int)((len + B - 1) / B);
    if (!a.columns) b1 = nb;
    const bool whole = b0 == 0 && b1 == nb;
    if (b0 == b1) {  // a row of none
        for (int i = tid; i < hn * HD; i += 64 * pkv::kWaves) a.out[r * a.ldo + (int64_t)h0 * HD + i] = 0.0f;
        return;
    }

    // the lane's part of its column's query: the column's plane of its dimensions
    float x[NF][8];
    {
        const float *src = a.q + r * a.ldq + (int64_t)(h0 + min(n & 7, hn - 1)) * HD;
#pragma unroll
        for (int f = 0; f < NF; f++)
            *reinterpret_cast<Float8 *>(x[f]) = *reinterpret_cast<const Float8 *>(
                src + (ELEM == 1 ? (f >> 1) * 64 + q * 16 + (f & 1) * 8 : f * 32 + q * 8));
    }
    const bool bias = a.slopes != nullptr;
    float slope = bias ? a.slopes[h0 + min(n & 7, hn - 1)] : 0.0f;
    // the new token's row, by the wave whose last block holds it
    const bool mine = a.k && told == len && b1 == nb && (nb - 1 - b0) % pkv::kWaves == w;
    float kx[HD / 64], vx[HD / 64];
    if (mine) {
        const int64_t from = r * a.ldq + kvh * HD + lane;
#pragma unroll
        for (int i = 0; i < HD / 64; i++) {
            kx[i] = a.k[from + 64 * i];
            vx[i] = a.v[from + 64 * i];
        }
    }
    // a block: its page (page 0 in the place of one that is none, with no live positions) and its rows there
    int b = b0 + w;
    int pi = min(b, b1 - 1) / bpp, off = min(b, b1 - 1) - pi * bpp;
    uint32_t kr[NT * NC][4], vr[ND][NV];
    v4f ks[NT], vs[NT];
    int64_t at = 0;  // the block's first row
    auto find = [&]() -> int {
        const int page = table_at(table + __builtin_amdgcn_readfirstlane(pi));
        const bool ok = page >= 0 && page < c.pages;
        at = uniform64(((int64_t)(ok ? page : 0) * c.n_kv + kvh) * c.page + off * B);
        const int64_t left = len - (int64_t)b * B;
        return __builtin_amdgcn_readfirstlane(ok ? (int)(left < B ? left : B) : 0);
    };
    auto load_k = [&]() {
        const auto rk = llmq_rsrc(c.k + at * HD * ELEM, kBytes);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b128(rk, n * HD * ELEM + q * 16,
                                                                     t * 16 * HD * ELEM + i * 64, kOnce);
#pragma unroll
                for (int e = 0; e < 4; e++) kr[t * NC + i][e] = y[e];
            }
        if constexpr (ELEM == 1) {
            const auto rs = llmq_rsrc(c.ks + at, 4 * B);
#pragma unroll
            for (int t = 0; t < NT; t++)
                ks[t] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * q, 64 * t, 0));
        }
    };
    auto load_v = [&]() {
        const auto rv = llmq_rsrc(c.v + at * HD * ELEM, kBytes);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const int vo = (n * B + q * 8) * ELEM, so = d * 16 * B * ELEM;
            if constexpr (ELEM == 1) {
                const auto y = __builtin_amdgcn_raw_buffer_load_b64(rv, vo, so, kOnce);
                vr[d][0] = y[0];
                vr[d][1] = y[1];
            } else {
                const auto y = __builtin_amdgcn_raw_buffer_load_b128(rv, vo, so, kOnce);
#pragma unroll
                for (int e = 0; e < 4; e++) vr[d][e] = y[e];
            }
        }
        if constexpr (ELEM == 1) {
            const auto rs = llmq_rsrc(c.vs + at, 4 * B);
#pragma unroll
            for (int t = 0; t < NT; t++)
                vs[t] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * q, 64 * t, 0));
        }
    };
    // the first block's rows are asked for before the query is taken apart
    // (a wave without a block asks for another's and leaves them)
    int live = find();
    load_k();
    load_v();
    h8 qf[NF];
    float mul, big = 1.0f;  // a score's factors
    {
        float m = 0.0f;
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if ((n & 7) >= hn) x[f][i] = 0.0f;
                m = fmaxf(m, fabsf(x[f][i]));
            }
        m = quarters_max(m);
        const int e = max((int)(__float_as_uint(m) >> 23) - (127 + 14), -112);  // (mul stays a normal float)
        mul = ldexpf(a.scale, e);
        if (ELEM == 1 && e >= 0) {  // large queries: not with a key's scale, beside which it might overflow
            big = mul;
            mul = 1.0f;
        }
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = ldexpf(x[f][i], -e);
                const _Float16 hi = (_Float16)y;
                qf[f][i] = low ? (_Float16)((y - (float)hi) * 2048.0f) : hi;
            }
    }
    const float own = low ? 0x1p-11f * big : big, oth = low ? big : 0x1p-11f * big;  // a score from the two columns
    const float wg = low ? 2048.0f : 1.0f, wr = low ? -2048.0f : 0.0f;     // a weight to its row's share
    const float icap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    asm volatile("" : "+v"(slope));  // waited for here, not behind the loop's loads

    // the new token's row goes to the cache (the tiles of a group store the
    // same bytes), and into the wave's last block as it came from memory
    int fb = -1;
    float fks = 0.0f, fvs = 0.0f;
    if (mine) {
        const int p = (int)(len - 1), page = table_at(table + __builtin_amdgcn_readfirstlane(p / c.page));
        if (page >= 0 && page < c.pages) {
            const NewRow<HD, ELEM> y = store_row<HD, ELEM>(c, page, p % c.page, kvh, kx, vx, lane);
#pragma unroll
            for (int i = 0; i < HD / 64; i++) {
                if constexpr (ELEM == 1) {
                    fresh[0][lane + 64 * i] = (uint8_t)y.k[i];
                    fresh[1][lane + 64 * i] = (uint8_t)y.v[i];
                } else {
                    reinterpret_cast<uint16_t *>(fresh[0])[lane + 64 * i] = (uint16_t)y.k[i];
                    reinterpret_cast<uint16_t *>(fresh[1])[lane + 64 * i] = (uint16_t)y.v[i];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            fks = y.ks;
            fvs = y.vs;
            fb = nb - 1;
        }
    }
    fb = __builtin_amdgcn_readfirstlane(fb);

    v4f acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = kLowest, l = 0.0f;
    // the weights' power of two: p is at most e (e 2^14 < 65504), a weight for int8 below 2^(ve + 2); top is where it
    // would be by the sums so far, which rising scores bring down by less than a power at a time
    constexpr int kTop = ELEM == 1 ? 13 : 14, kLeast = -100;
    int ve = ELEM == 1 ? kLeast : 0;
    float top = kLeast;

    // one block; LAST: the wave's last, which may hold the new token and the
    // row's end (the others are whole, or in a page that is none)
    auto block = [&](auto last) {
        constexpr bool LAST = decltype(last)::value;
        const int j0 = b * B, have = live;
        if (LAST && b == fb) {
            const int o = (int)(len - 1) - j0, ft = o >> 4, fq = (o >> 2) & 3, fi = o & 3;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                if (t != ft) continue;
                if (n == (o & 15))
#pragma unroll
                    for (int i = 0; i < NC; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            kr[t * NC + i][e] =
                                *reinterpret_cast<const uint32_t *>(&fresh[0][i * 64 + q * 16 + 4 * e]);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (ELEM == 1 && i == fi && q == fq) {
                        ks[t][i] = fks;
                        vs[t][i] = fvs;
                    }
            }
            const int word = (ft * 4 + fi) * ELEM / 4, sh = (ft * 4 + fi) * ELEM % 4 * 8;
            const uint32_t keep = ~((ELEM == 1 ? 0xffu : 0xffffu) << sh);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const uint32_t code = ELEM == 1 ? fresh[1][16 * d + n]
                                                : reinterpret_cast<const uint16_t *>(fresh[1])[16 * d + n];
#pragma unroll
                for (int i = 0; i < NV; i++)
                    if (i == word && q == fq) vr[d][i] = (vr[d][i] & keep) | code << sh;
            }
        }
        if constexpr (!LAST) {
            b += pkv::kWaves;
            for (off += pkv::kWaves; off >= bpp; off -= bpp) pi++;
            live = find();
        }
        // scores
        v4f s[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const uint32_t *y = kr[t * NC + i];
                if constexpr (ELEM == 1) {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(y[0], y[1]), qf[2 * i], s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(y[2], y[3]), qf[2 * i + 1], s[t], 0, 0, 0);
                } else {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(y[0], y[1], y[2], y[3]), qf[i], s[t], 0, 0,
                                                                  0);
                }
            }
        }
        float sv[NT * 4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y = s[t][i] * own + llmq_dppf<0x128>(s[t][i]) * oth;  // row_ror:8
                sv[4 * t + i] = y * (ELEM == 1 ? ks[t][i] * mul : mul);
            }
        if constexpr (!LAST) load_k();
        if (a.cap > 0.0f)
#pragma unroll
            for (int i = 0; i < NT * 4; i++) sv[i] = a.cap * tanh_select(sv[i] * icap);
        if (bias) {
            const float base = (float)(j0 + 4 * q - (len - 1));
#pragma unroll
            for (int i = 0; i < NT * 4; i++) sv[i] = fmaf(slope, base + (float)(16 * (i >> 2) + (i & 3)), sv[i]);
        }
        if (!LAST && have == 0) {
#pragma unroll
            for (int i = 0; i < NT * 4; i++) sv[i] = -INFINITY;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < NV; i++) vr[d][i] = 0;
            if constexpr (ELEM == 1) vs[0] = vs[1] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (LAST && have < B) {
#pragma unroll
            for (int i = 0; i < NT * 4; i++) {
                const bool in = 16 * (i >> 2) + 4 * q + (i & 3) < have;
                sv[i] = in ? sv[i] : -INFINITY;
                if constexpr (ELEM == 1) vs[i >> 2][i & 3] = in ? vs[i >> 2][i & 3] : 0.0f;
            }
            if constexpr (ELEM == 2) {  // what lies there may be NaN
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int p = 16 * (i >> 1) + 4 * q + 2 * (i & 1);
                    const uint32_t keep = p + 1 < have ? 0xffffffffu : (p < have ? 0xffffu : 0u);
#pragma unroll
                    for (int d = 0; d < ND; d++) vr[d][i] &= keep;
                }
            }
        }
        float mx = sv[0];
#pragma unroll
        for (int i = 1; i < NT * 4; i++) mx = fmaxf(mx, sv[i]);
        mx = quarters_max(mx);
        const bool moves = __any(mx - ref > 1.0f);
        float down = 0.0f;  // log2 of what the sums so far are multiplied by
        if (moves) {
            const float to = fmaxf(ref, mx);
            down = ref == to ? 0.0f : (ref - to) * kLog2e;
            ref = to;
            l *= exp2f(down);
        }
        float wm = 0.0f;
#pragma unroll
        for (int i = 0; i < NT * 4; i++) {
            const float p = __builtin_amdgcn_exp2f((sv[i] - ref) * kLog2e);
            l += p;
            sv[i] = ELEM == 1 ? p * vs[i >> 2][i & 3] : p;
            if constexpr (ELEM == 1) wm = fmaxf(wm, sv[i]);
        }
        int e = 0;
        if constexpr (ELEM == 1) e = (int)(__float_as_uint(quarters_max(wm)) >> 23) - 127;
        if (moves || (ELEM == 1 && __any(e > ve + 1))) {
            int to = ve;
            if constexpr (ELEM == 1) {
                top = fmaxf(fmaxf(top + fmaxf(down, -400.0f), (float)e), (float)kLeast);
                to = (int)floorf(top);
            }
            const float f = ldexpf(exp2f(down), ve - to);
            ve = to;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float y = __shfl(f, 4 * q + i);  // of row 4 q + i
#pragma unroll
                for (int d = 0; d < ND; d++) acc[d][i] *= y;
            }
        }
        const float unit = ldexpf(1.0f, kTop - ve);
        h8 wf;
#pragma unroll
        for (int i = 0; i < NT * 4; i++) {
            float y = sv[i] * unit;
            // rounded to 32 bits once, for both rows: the product straight to 16 bits would now and then be another
            // float16 than the one below, and the rows no longer add up
            asm volatile("" : "+v"(y));
            const float hi = (float)(_Float16)y;
            // row n: y rounded; row n ^ 8: what that leaves times 2^11 (exact)
            wf[i] = (_Float16)fmaf(hi, wr, y * wg);
        }
        // values
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const h8 y = ELEM == 1 ? halves(vr[d][0], vr[d][1])
                                   : as_h8(vr[d][0], vr[d][1], vr[d][NV - 2], vr[d][NV - 1]);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf, y, acc[d], 0, 0, 0);
        }
        if constexpr (!LAST) load_v();
    };
    while (b + pkv::kWaves < b1) block(std::false_type{});
    if (b < b1) block(std::true_type{});
    // the waves' results
    l = quarters_sum(l);
    if (lane < 8) wml[w][n] = make_float2(ref, l);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int e = ELEM == 1 ? __shfl(ve, 4 * q + i) : 0;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const float y = acc[d][i], z = __shfl_xor(y, 32);  // rows 4 q + i and 4 q + i + 8
            if (q < 2) wsum[w][4 * q + i][16 * d + n] = ldexpf(fmaf(z, 0x1p-11f, y), e - kTop);
        }
    }
    __syncthreads();
    if (tid == 0 && blockIdx.y == 0 && a.columns && b0 == 0) a.meta[r] = make_int2(slot, count);
    for (int i = tid; i < hn * HD; i += 64 * pkv::kWaves) {
        const int h = i / HD, d = i % HD;
        float R = kLowest, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int k = 0; k < pkv::kWaves; k++) R = fmaxf(R, wml[k][h].x);
#pragma unroll
        for (int k = 0; k < pkv::kWaves; k++) {
            const float f = exp2f((wml[k][h].x - R) * kLog2e);
            L = fmaf(wml[k][h].y, f, L);
            o = fmaf(wsum[k][h][d], f, o);
        }
        if (whole) {
            a.out[r * a.ldo + (int64_t)(h0 + h) * HD + d] = L == 0.0f ? 0.0f : o / L;
        } else {
            const int64_t at = (int64_t)slot * a.n_head + h0 + h;
            a.sums[at * HD + d] = o;
            if (d == 0) a.ml[at] = make_float2(R, L);
        }
    }
}

// The segments of a row put together, in their order: a workgroup a (head,
// row), all of a row's parts asked for at once up to 32.  5-6 us, of which the
// launch is most: 4 x 32 of 65 parts 5.4, 64 x 32 of 1-4 parts 6.0.
constexpr int kJoinWaves = 4;
template <int HD>
__global__ __launch_bounds__(64 * kJoinWaves) void pkv_join_kernel(Layer c, Attend a) {
    __shared__ float2 wl[kJoinWaves];
    __shared__ float ws[kJoinWaves][HD];
    const int64_t r = blockIdx.y;
    const int h = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int2 m = a.meta[r];
    if (row_len(c, a, r) == 0) {  // in no slot
        if (threadIdx.x < HD) a.out[r * a.ldo + (int64_t)h * HD + threadIdx.x] = 0.0f;
        return;
    }
    if (m.y == 1) return;  // in one, which has written it
    const float2 *ml = a.ml + (int64_t)m.x * a.n_head + h;
    const float *sums = a.sums + ((int64_t)m.x * a.n_head + h) * HD;
    const int n = m.y;
    // a wave every fourth segment, kAtOnce of them asked for together
    constexpr int kAtOnce = 8;
    float R = kLowest, L = 0.0f, o[HD / 64] = {};
    for (int i0 = w; i0 < n; i0 += kJoinWaves * kAtOnce) {
        float2 x[kAtOnce];
        float s[kAtOnce][HD / 64];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const int i = i0 + kJoinWaves * k;
            x[k] = make_float2(kLowest, 0.0f);
            if (i < n) {
                x[k] = ml[(int64_t)i * a.n_head];
#pragma unroll
                for (int d = 0; d < HD / 64; d++) s[k][d] = sums[(int64_t)i * a.n_head * HD + lane + 64 * d];
            } else {
#pragma unroll
                for (int d = 0; d < HD / 64; d++) s[k][d] = 0.0f;
            }
        }
        float to = R;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) to = fmaxf(to, x[k].x);
        const float f = exp2f((R - to) * kLog2e);
        R = to;
        L *= f;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] *= f;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const float g = exp2f((x[k].x - R) * kLog2e);
            L = fmaf(x[k].y, g, L);
#pragma unroll
            for (int d = 0; d < HD / 64; d++) o[d] = fmaf(s[k][d], g, o[d]);
        }
    }
    if (lane == 0) wl[w] = make_float2(R, L);
#pragma unroll
    for (int d = 0; d < HD / 64; d++) ws[w][lane + 64 * d] = o[d];
    __syncthreads();
    if (threadIdx.x < HD) {
        const int d = threadIdx.x;
        float to = kLowest, all = 0.0f, s = 0.0f;
#pragma unroll
        for (int k = 0; k < kJoinWaves; k++) to = fmaxf(to, wl[k].x);
#pragma unroll
        for (int k = 0; k < kJoinWaves; k++) {
            const float g = exp2f((wl[k].x - to) * kLog2e);
            all = fmaf(wl[k].y, g, all);
            s = fmaf(ws[k][d], g, s);
        }
        a.out[r * a.ldo + (int64_t)h * HD + d] = all == 0.0f ? 0.0f : s / all;
    }
}

template <class F>
int dispatch(const llmq_pkv *kv, F &&f) {
    if (kv->hd == 64) return kv->elem() == 1 ? f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{})
                                             : f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
    return kv->elem() == 1 ? f(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{})
                           : f(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{});
}

// Checks of every call on `rows` rows; none of their pointers is needed for none.
int check_cache(const char *name, const llmq_ctx *ctx, const llmq_pkv *kv, int layer, const void *table,
                int64_t width, int64_t rows) {
    LLMQ_REQUIRE(ctx && kv && (table || rows == 0), "%s: null argument", name);
    LLMQ_REQUIRE(kv->device == ctx->device, "%s: the cache is on device %d, the context on %d", name,
                 kv->device, ctx->device);
    LLMQ_REQUIRE(layer >= 0 && layer < kv->n_layer, "%s: layer %d of %d", name, layer, kv->n_layer);
    LLMQ_REQUIRE(width >= 1 && width <= INT32_MAX / kv->page, "%s: a table row of %lld pages", name, (long long)width);
    return LLMQ_OK;
}

Layer layer_of(const llmq_pkv *kv, int layer, const int32_t *table, int64_t width) {
    const int64_t at = (int64_t)layer * kv->n_pages * kv->n_kv * kv->page;
    Layer c;
    c.k = kv->k + at * kv->hd * kv->elem();
    c.v = kv->v + at * kv->hd * kv->elem();
    c.ks = kv->ks ? kv->ks + at : nullptr;
    c.vs = kv->vs ? kv->vs + at : nullptr;
    c.table = table;
    c.width = width;
    c.pages = kv->n_pages;
    c.page = kv->page;
    c.n_kv = kv->n_kv;
    return c;
}

// Shared checks of the row-wise calls: T rows of n_kv * hd floats, ld apart.
int check_rows(const char *name, const llmq_pkv *kv, const void *k, const void *v, int64_t ld, int64_t T,
               const void *seq, const void *pos, int64_t n_seq) {
    LLMQ_REQUIRE((k && v && seq && pos) || T == 0, "%s: null argument", name);
    LLMQ_REQUIRE(T >= 0 && T <= INT32_MAX, "%s: %lld rows", name, (long long)T);
    LLMQ_REQUIRE(n_seq >= 0, "%s: %lld sequences", name, (long long)n_seq);
    LLMQ_REQUIRE(ld >= (int64_t)kv->n_kv * kv->hd, "%s: rows of %lld floats hold no %d heads of %d", name,
                 (long long)ld, kv->n_kv, kv->hd);
    return LLMQ_OK;
}

int attend(const char *name, llmq_ctx *ctx, const llmq_pkv *kv, int layer, Attend a, int64_t rows,
           const int32_t *table, int64_t width, void *work, int64_t work_bytes) {
    RC(check_cache(name, ctx, kv, layer, table, width, rows));
    LLMQ_REQUIRE((a.out && a.q && a.len && work) || rows == 0, "%s: null argument", name);
    LLMQ_REQUIRE(rows >= 0 && rows <= 65535, "%s: %lld rows (at most 65535)", name, (long long)rows);
    LLMQ_REQUIRE(a.n_head > 0 && a.n_head % kv->n_kv == 0 && a.n_head <= 65535, "%s: %d query heads over %d cached",
                 name, a.n_head, kv->n_kv);
    const int64_t need = (int64_t)a.n_head * kv->hd;
    LLMQ_REQUIRE(a.ldo >= need && a.ldq >= need, "%s: row strides %lld, %lld below %lld", name, (long long)a.ldo,
                 (long long)a.ldq, (long long)need);
    LLMQ_REQUIRE(a.scale == a.scale && (a.cap == 0.0f || (a.cap >= 1.2e-38f && a.cap <= 3.0e38f)),
                 "%s: scale %g, cap %g", name, a.scale, a.cap);  // (1 / cap is finite)
    const int64_t want = llmq_pkv_work_bytes(kv, rows, a.n_head);
    LLMQ_REQUIRE(work_bytes >= want, "%s: %lld bytes of work, %lld needed", name, (long long)work_bytes,
                 (long long)want);
    if (rows == 0) return LLMQ_OK;
    LLMQ_REQUIRE((uintptr_t)work % 16 == 0, "%s: work is 16-byte aligned", name);
    DeviceGuard guard(ctx);
    const Layer c = layer_of(kv, layer, table, width);
    const pkv::Plan p = pkv::plan_of(rows, a.n_head, kv->n_kv);
    const pkv::Work at = pkv::work_of(p, rows, a.n_head, kv->hd);
    LLMQ_REQUIRE((int64_t)kv->n_kv * p.tiles <= 65535, "%s: %d query heads", name, a.n_head);
    a.rows = (int)rows;
    a.tiles = p.tiles;
    a.meta = static_cast<int2 *>(work);
    a.ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(work) + at.ml);
    a.sums = reinterpret_cast<float *>(static_cast<uint8_t *>(work) + at.sums);
    const bool join = p.columns && width * (kv->page / B) > (int64_t)p.uncut;
    a.columns = join ? p.columns : 0;
    a.least = p.least;
    // eight slots, one an XCD, of every head after one another: a slot's tiles share their XCD's L2, and the
    // slots without a segment, the last, are the last to start
    const int64_t slots = join ? pkv::slots_of(p, rows) : rows;
    LLMQ_REQUIRE(!join || rows * width * (kv->page / B) < pkv::kMaxBlocks, "%s: %lld table rows of %lld pages", name,
                 (long long)rows, (long long)width);
    return dispatch(kv, [&](auto hd, auto elem) -> int {
        const dim3 grid(8, (unsigned)(kv->n_kv * p.tiles), (unsigned)((slots + 7) / 8));
        hipLaunchKernelGGL((pkv_attend_kernel<decltype(hd)::value, decltype(elem)::value>), grid,
                           dim3(64 * pkv::kWaves), 0, ctx->stream, c, a);
        if (join)
            hipLaunchKernelGGL((pkv_join_kernel<decltype(hd)::value>), dim3((unsigned)a.n_head, (unsigned)rows),
                               dim3(64 * kJoinWaves), 0, ctx->stream, c, a);
        LLMQ_HIP(hipGetLastError());
        return LLMQ_OK;
    });
}

}  // namespace

extern "C" {

int llmq_pkv_create(llmq_ctx *ctx, int type, int n_layer, int64_t n_pages, int page, int n_kv, int head_dim,
                    llmq_pkv **out) {
    LLMQ_REQUIRE(ctx && out, "pkv_create: null argument");
    LLMQ_REQUIRE(type == LLMQ_PKV_INT8 || type == LLMQ_PKV_F16, "pkv_create: type %d", type);
    LLMQ_REQUIRE(n_layer > 0 && n_pages > 0 && n_pages <= INT32_MAX && n_kv > 0 && n_kv <= 65535,
                 "pkv_create: %d layers, %lld pages, %d heads", n_layer, (long long)n_pages, n_kv);
    LLMQ_REQUIRE(page >= 64 && page <= 4096 && page % 64 == 0,
                 "pkv_create: pages of %d positions (64 to 4096, a multiple of 64)", page);
    if (head_dim != 64 && head_dim != 128)
        return llmq_set_error(LLMQ_EUNSUPPORTED, "pkv_create: head_dim %d (64 or 128)", head_dim);
    LLMQ_REQUIRE(!ctx_capturing(ctx), "pkv_create: not under graph capture");
    const double total = (double)n_layer * (double)n_pages * n_kv * page * head_dim * 2.0;
    LLMQ_REQUIRE(total < 1e15, "pkv_create: %g elements", total);
    llmq_pkv *kv = new (std::nothrow) llmq_pkv();
    if (!kv) return llmq_set_error(LLMQ_ENOMEM, "pkv_create: out of host memory");
    kv->device = ctx->device;
    kv->type = type;
    kv->n_layer = n_layer;
    kv->n_pages = n_pages;
    kv->page = page;
    kv->n_kv = n_kv;
    kv->hd = head_dim;
    DeviceGuard guard(ctx);
    const size_t n = (size_t)kv->rows() * head_dim * kv->elem(), ns = (size_t)kv->rows() * 4;
    const bool scales = type == LLMQ_PKV_INT8;
    if (hipMalloc(&kv->k, n) != hipSuccess || hipMalloc(&kv->v, n) != hipSuccess ||
        (scales && (hipMalloc(&kv->ks, ns) != hipSuccess || hipMalloc(&kv->vs, ns) != hipSuccess))) {
        (void)hipGetLastError();
        llmq_pkv_free(kv);
        return llmq_set_error(LLMQ_ENOMEM, "pkv_create: allocation of %zu bytes failed", 2 * n + (scales ? 2 * ns : 0));
    }
    const int zero = scales ? kBias : 0;  // the code of 0
    if (hipMemsetAsync(kv->k, zero, n, ctx->stream) != hipSuccess ||
        hipMemsetAsync(kv->v, zero, n, ctx->stream) != hipSuccess ||
        (scales && (hipMemsetAsync(kv->ks, 0, ns, ctx->stream) != hipSuccess ||
                    hipMemsetAsync(kv->vs, 0, ns, ctx->stream) != hipSuccess)) ||
        hipStreamSynchronize(ctx->stream) != hipSuccess) {  // other streams may use it at once
        llmq_pkv_free(kv);
        return llmq_set_error(LLMQ_EHIP, "pkv_create: clearing the cache failed");
    }
    *out = kv;
    return LLMQ_OK;
}

int llmq_pkv_free(llmq_pkv *kv) {
    if (!kv) return LLMQ_OK;
    DeviceGuard guard(kv->device);
    hipFree(kv->k);  // (waits for the device; the context may be gone)
    hipFree(kv->v);
    hipFree(kv->ks);
    hipFree(kv->vs);
    delete kv;
    return LLMQ_OK;
}

int64_t llmq_pkv_nbytes(const llmq_pkv *kv) {
    if (!kv) return 0;
    return 2 * kv->rows() * (kv->hd * kv->elem() + (kv->type == LLMQ_PKV_INT8 ? 4 : 0));
}

int llmq_pkv_store(llmq_ctx *ctx, llmq_pkv *kv, int layer, const float *k, const float *v, int64_t ld, int64_t T,
                   const int32_t *seq, const int32_t *pos, const int32_t *table, int64_t n_seq, int64_t width) {
    RC(check_cache("pkv_store", ctx, kv, layer, table, width, T));
    RC(check_rows("pkv_store", kv, k, v, ld, T, seq, pos, n_seq));
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    const Layer c = layer_of(kv, layer, table, width);
    return dispatch(kv, [&](auto hd, auto elem) -> int {
        hipLaunchKernelGGL((pkv_store_kernel<decltype(hd)::value, decltype(elem)::value>),
                           dim3((unsigned)((T + kRows - 1) / kRows), (unsigned)kv->n_kv), dim3(kRows * kLanes), 0,
                           ctx->stream, c, k, v, ld, T, seq, pos, n_seq);
        LLMQ_HIP(hipGetLastError());
        return LLMQ_OK;
    });
}

int llmq_pkv_fetch(llmq_ctx *ctx, const llmq_pkv *kv, int layer, float *k, float *v, int64_t ld, int64_t T,
                   const int32_t *seq, const int32_t *pos, const int32_t *table, int64_t n_seq, int64_t width) {
    RC(check_cache("pkv_fetch", ctx, kv, layer, table, width, T));
    RC(check_rows("pkv_fetch", kv, k, v, ld, T, seq, pos, n_seq));
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    const Layer c = layer_of(kv, layer, table, width);
    return dispatch(kv, [&](auto hd, auto elem) -> int {
        hipLaunchKernelGGL((pkv_fetch_kernel<decltype(hd)::value, decltype(elem)::value>),
                           dim3((unsigned)((T + kRows - 1) / kRows), (unsigned)kv->n_kv), dim3(kRows * kLanes), 0,
                           ctx->stream, c, k, v, ld, T, seq, pos, n_seq);
        LLMQ_HIP(hipGetLastError());
        return LLMQ_OK;
    });
}

int64_t llmq_pkv_work_bytes(const llmq_pkv *kv, int64_t rows, int n_head) {
    if (!kv || rows < 0 || rows > 65535 || n_head <= 0 || n_head > 65535) return -1;
    if (n_head % kv->n_kv) return -1;
    return pkv::work_of(pkv::plan_of(rows, n_head, kv->n_kv), rows, n_head, kv->hd).bytes;
}

int llmq_pkv_attend(llmq_ctx *ctx, const llmq_pkv *kv, int layer, float *out, int64_t ldo, const float *q, int64_t ldq,
                    int64_t rows, int n_head, const int32_t *len, const int32_t *table, int64_t width, float scale,
                    float cap, const float *slopes, void *work, int64_t work_bytes) {
    const Attend a{out, ldo, q, nullptr, nullptr, ldq, len, n_head, scale, cap, slopes, 0, 0, 0, 0, nullptr, nullptr,
                   nullptr};
    return attend("pkv_attend", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

int llmq_pkv_step(llmq_ctx *ctx, llmq_pkv *kv, int layer, float *out, int64_t ldo, const float *q, const float *k,
                  const float *v, int64_t ld, int64_t rows, int n_head, const int32_t *pos, const int32_t *table,
                  int64_t width, float scale, float cap, const float *slopes, void *work, int64_t work_bytes) {
    LLMQ_REQUIRE((k && v) || rows == 0, "pkv_step: null argument");
    const Attend a{out, ldo, q, k, v, ld, pos, n_head, scale, cap, slopes, 0, 0, 0, 0, nullptr, nullptr, nullptr};
    return attend("pkv_step", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

}  // extern "C"
