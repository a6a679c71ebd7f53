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
    llmq_ctx *ctx = nullptr;
    int type = 0, n_layer = 0, page = 0, n_kv = 0, hd = 0;
    int64_t n_pages = 0;
    uint8_t *k = nullptr, *v = nullptr;
    float *ks = nullptr, *vs = nullptr;  // int8 only
    int elem() const { return type == LLMQ_PKV_INT8 ? 1 : 2; }
    int64_t rows() const { return (int64_t)n_layer * n_pages * n_kv * page; }  // positions x heads held
};

namespace {

// One layer of a cache as a kernel takes it.
struct Layer {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;
    int64_t width, pages;
    int page, n_kv;
};

// A head's row (position 0 of its page) in units of positions.
__device__ __forceinline__ int64_t head_row(const Layer &c, int page, int head) {
    return ((int64_t)page * c.n_kv + head) * c.page;
}

// QuantKV.store's quantisation of one row (kvcache.mojo:333-342) over a wave,
// HD / 64 dimensions a lane: s = max|x| / 127 (1 for a row of zeros), codes
// round(x / s) away from zero at ties.  A row with a NaN or an infinity gets
// the scale NaN; one below 2^-120, whose reciprocal scale is infinite, is a row of zeros.
template <int HD>
__device__ __forceinline__ float quant_row(const float (&x)[HD / 64], int (&code)[HD / 64]) {
    float m = 0.0f, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        m = fmaxf(m, fabsf(x[i]));
        bad += x[i] - x[i];  // NaN for NaN and infinities
    }
    m = llmq_wave_max_all(m);
    const bool none = __any(bad != 0.0f || bad != bad);
    const float s = m < 0x1p-120f ? 1.0f : m / 127.0f;
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < HD / 64; i++) code[i] = none ? 0 : llmq_to_int(roundf(x[i] * inv));
    return none ? __uint_as_float(0x7fc00000u) : s;
}

__device__ __forceinline__ uint16_t half_bits(float x) {
    // nearest even; finite values past the range become its ends
    const float lim = fabsf(x) <= 3.0e38f ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    return __half_as_ushort(__float2half_rn(lim));
}

// One wave writes the key and value row of (token, head).
template <int HD, int ELEM>
__device__ __forceinline__ void store_row(const Layer &c, int page, int off, int head, const float *k, const float *v,
                                          int lane) {
    const int64_t row = head_row(c, page, head) + off;
    const int B = pkv::block_positions(ELEM), blk = off / B;
    const int64_t vrow = (head_row(c, page, head) + (int64_t)blk * B) * HD;  // the block's first element
    const int slot = pkv::value_slot(ELEM, off % B);
    float kx[HD / 64], vx[HD / 64];
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        kx[i] = k[lane + 64 * i];
        vx[i] = v[lane + 64 * i];
    }
    if constexpr (ELEM == 1) {
        int kc[HD / 64], vc[HD / 64];
        const float s = quant_row<HD>(kx, kc), t = quant_row<HD>(vx, vc);
#pragma unroll
        for (int i = 0; i < HD / 64; i++) {
            c.k[row * HD + lane + 64 * i] = (uint8_t)kc[i];
            c.v[vrow + (int64_t)(lane + 64 * i) * B + slot] = (uint8_t)vc[i];
        }
        if (lane == 0) {
            c.ks[row] = s;
            c.vs[row] = t;
        }
    } else {
        uint16_t *ck = reinterpret_cast<uint16_t *>(c.k), *cv = reinterpret_cast<uint16_t *>(c.v);
#pragma unroll
        for (int i = 0; i < HD / 64; i++) {
            ck[row * HD + lane + 64 * i] = half_bits(kx[i]);
            cv[vrow + (int64_t)(lane + 64 * i) * B + slot] = half_bits(vx[i]);
        }
    }
}

// Element (lane + 64 i) of a cached key / value row.
template <int HD, int ELEM>
__device__ __forceinline__ void load_row(const Layer &c, int page, int off, int head, float (&k)[HD / 64],
                                         float (&v)[HD / 64], int lane) {
    const int64_t row = head_row(c, page, head) + off;
    const int B = pkv::block_positions(ELEM), blk = off / B;
    const int64_t vrow = (head_row(c, page, head) + (int64_t)blk * B) * HD;
    const int slot = pkv::value_slot(ELEM, off % B);
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        const int d = lane + 64 * i;
        if constexpr (ELEM == 1) {
            k[i] = (float)(int8_t)c.k[row * HD + d] * c.ks[row];
            v[i] = (float)(int8_t)c.v[vrow + (int64_t)d * B + slot] * c.vs[row];
        } else {
            k[i] = __half2float(__ushort_as_half(reinterpret_cast<const uint16_t *>(c.k)[row * HD + d]));
            v[i] = __half2float(
                __ushort_as_half(reinterpret_cast<const uint16_t *>(c.v)[vrow + (int64_t)d * B + slot]));
        }
    }
}

// llmq_pkv_store: one wave a (token, head).
template <int HD, int ELEM>
__global__ __launch_bounds__(64) void pkv_store_kernel(Layer c, const float *__restrict__ k,
                                                       const float *__restrict__ v, int64_t ld,
                                                       const int32_t *__restrict__ seq,
                                                       const int32_t *__restrict__ pos, int64_t n_seq) {
    const int64_t t = blockIdx.x;
    const int head = blockIdx.y, s = seq[t];
    if (s < 0 || s >= n_seq) return;
    const int page = pkv::page_of(c.table + s * c.width, c.width, c.page, c.pages, pos[t]);
    if (page < 0) return;
    store_row<HD, ELEM>(c, page, pos[t] % c.page, head, k + t * ld + head * HD, v + t * ld + head * HD, threadIdx.x);
}

// llmq_pkv_fetch: one wave a (token, head); zeros where the cache has no row.
template <int HD, int ELEM>
__global__ __launch_bounds__(64) void pkv_fetch_kernel(Layer c, float *__restrict__ k, float *__restrict__ v,
                                                       int64_t ld, const int32_t *__restrict__ seq,
                                                       const int32_t *__restrict__ pos, int64_t n_seq) {
    const int64_t t = blockIdx.x;
    const int head = blockIdx.y, s = seq[t], lane = threadIdx.x;
    int page = -1;
    if (s >= 0 && s < n_seq) page = pkv::page_of(c.table + s * c.width, c.width, c.page, c.pages, pos[t]);
    float kx[HD / 64], vx[HD / 64];
#pragma unroll
    for (int i = 0; i < HD / 64; i++) kx[i] = vx[i] = 0.0f;
    if (page >= 0) load_row<HD, ELEM>(c, page, pos[t] % c.page, head, kx, vx, lane);
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        k[t * ld + head * HD + lane + 64 * i] = kx[i];
        v[t * ld + head * HD + lane + 64 * i] = vx[i];
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
    int rows, tiles, shift;
    int2 *meta;    // [row]: first split, number of splits
    float2 *ml;    // [split][head]: reference (log2), sum
    float *sums;   // [split][head][hd]
};

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

// Eight int8 codes as float16, exactly: byte u = code + 128 under the
// exponent byte 0x64 is 1024 + u, less 1152.
__device__ __forceinline__ h8 halves(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        h2 h[4];
        h8 v;
    } r;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - off;
    return r.v;
}

__device__ __forceinline__ h8 as_h8(const uint4 &x) {
    union {
        uint4 u;
        h8 v;
    } r;
    r.u = x;
    return r.v;
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

__device__ __forceinline__ int64_t row_len(const Layer &c, const Attend &a, int64_t r) {
    const int64_t n = a.len[r];
    return pkv::clamp_len(a.k ? n + 1 : n, c.width, c.page);
}

// Which part of which row workgroup column `slot` takes; every wave finds it
// by itself from the rows' lengths (a.rows <= kPlanRows).
struct Part {
    int row, split, count, first;  // row -1: nothing
    int64_t blocks;                // blocks a split
};
__device__ __forceinline__ Part find_part(const Layer &c, const Attend &a, int B, int slot, int lane) {
    constexpr int N = pkv::kPlanRows / 64;
    uint32_t nb[N];
    int64_t total = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int r = 64 * i + lane;
        nb[i] = r < a.rows ? (uint32_t)((row_len(c, a, r) + B - 1) / B) : 0;
        total += nb[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
    Part p;
    p.blocks = pkv::split_blocks(total, a.shift);
    p.row = -1;
    uint32_t before = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (64 * i >= a.rows) break;
        const uint32_t mine = 64 * i + lane < a.rows ? pkv::row_splits(nb[i], (uint32_t)p.blocks) : 0;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(incl, o);
            if (lane >= o) incl += up;
        }
        const uint32_t all = __shfl(incl, 63);
        if (p.row < 0 && (uint32_t)slot < before + all) {
            const int at = __popcll(__ballot(before + incl <= (uint32_t)slot));  // < 64
            const uint32_t end = __shfl(incl, at), n = __shfl(mine, at);
            p.row = 64 * i + at;
            p.count = (int)n;
            p.first = (int)(before + end - n);
            p.split = slot - p.first;
        }
        before += all;
    }
    return p;
}

// Attention of one token over a row's pages, or a split of it: 4 waves, up to
// 8 query heads of one cached head, on the fp16 matrix cores.
//
// Scores: K (16 positions x 32 dimensions) times the queries as 16 columns,
// columns 0-7 their float16 roundings and 8-15 what those leave times 2^11
// (22 bits in all; the keys are exact), so column n and n ^ 8 add up to a
// score, in lane n for positions 4 (lane / 16) + 0..3 of the tile.  Values:
// the weights are already where the second product wants its rows: row n
// holds head n's weights as float16, row n ^ 8 what is left times 2^11, and
// the slots of paged_plan.h give the values in the same order, so nothing is
// moved between lanes.  For int8 a weight is p times the value's scale over a
// power of two near the largest scale so far.
//
// The reference of a head's exponentials is moved (and the sums rescaled)
// only when a score passes it by 2^6, which is rare after the first blocks.
// Each wave keeps its own and reads every fourth block; the four are put
// together through LDS.  A wave's next keys are on their way while it forms
// the weights, its next values while it scores.
template <int HD, int ELEM>
__global__ __launch_bounds__(256, 2) void pkv_attend_kernel(Layer c, Attend a) {
    constexpr int B = ELEM == 1 ? 64 : 32, NT = B / 16, NC = HD * ELEM / 64, NF = HD / 32, ND = HD / 16;
    constexpr int kBlock = HD * 64;  // bytes of a block's keys, and of its values
    __shared__ __align__(16) _Float16 qp[16][HD];
    __shared__ float qexp[8];
    __shared__ float2 wml[pkv::kWaves][8];
    __shared__ float wsum[pkv::kWaves][8][HD];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = lane & 15, q = lane >> 4;
    const int kvh = blockIdx.y / a.tiles, G = a.n_head / c.n_kv, t0 = blockIdx.y % a.tiles * 8;
    const int h0 = kvh * G + t0, hn = min(8, G - t0);

    Part part;
    if (a.shift >= 0) {
        part = find_part(c, a, B, blockIdx.x, lane);
        if (part.row < 0) return;  // the same for the whole workgroup
    } else {
        part = Part{(int)blockIdx.x, 0, 1, 0, 0x7fffffff};
    }
    const int64_t r = __builtin_amdgcn_readfirstlane(part.row);
    const int32_t *table = c.table + r * c.width;
    const int64_t len = row_len(c, a, r);
    const int nb = (int)((len + B - 1) / B);
    const int64_t e64 = (part.split + 1) * part.blocks;
    const int b0 = __builtin_amdgcn_readfirstlane((int)(part.split * part.blocks)),
              b1 = __builtin_amdgcn_readfirstlane((int)(e64 < nb ? e64 : nb));
    const int count = __builtin_amdgcn_readfirstlane(part.count);

    // the new token's rows, by the workgroups whose split ends with it (the
    // tiles of a group write the same bytes, and each reads its own)
    if (a.k && len > 0 && b1 == nb && w == pkv::kWaves - 1) {
        const int64_t p = len - 1;
        const int page = a.len[r] == p ? pkv::page_of(table, c.width, c.page, c.pages, p) : -1;
        if (page >= 0)
            store_row<HD, ELEM>(c, page, (int)(p % c.page), kvh, a.k + r * a.ldq + kvh * HD, a.v + r * a.ldq + kvh * HD,
                                lane);
    }
    // queries to their planes: heads 2 w and 2 w + 1
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int h = 2 * w + i;
        float x[HD / 64], m = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) {
            x[d] = h < hn ? a.q[r * a.ldq + (int64_t)(h0 + h) * HD + lane + 64 * d] : 0.0f;
            m = fmaxf(m, fabsf(x[d]));
        }
        m = llmq_wave_max_all(m);
        const int e = m > 0.0f ? (int)(__float_as_uint(m) >> 23) - 127 : 0;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) {
            const float y = ldexpf(x[d], -e);
            const _Float16 hi = (_Float16)y;
            qp[h][lane + 64 * d] = hi;
            qp[h + 8][lane + 64 * d] = (_Float16)((y - (float)hi) * 2048.0f);
        }
        if (lane == 0) qexp[h] = ldexpf(a.scale, e);
    }
    __syncthreads();
    h8 qf[NF];
#pragma unroll
    for (int f = 0; f < NF; f++) {
        const int d = ELEM == 1 ? (f >> 1) * 64 + q * 16 + (f & 1) * 8 : f * 32 + q * 8;
        qf[f] = *reinterpret_cast<const h8 *>(&qp[n][d]);
    }
    const bool low = n >= 8;
    const float mul = qexp[n & 7];
    const float own = low ? 0x1p-11f : 1.0f, oth = low ? 1.0f : 0x1p-11f;  // a score from the two columns
    const float wg = low ? 2048.0f : 1.0f, wr = low ? -2048.0f : 0.0f;     // a weight to its row's share
    const float slope = a.slopes && (n & 7) < hn ? a.slopes[h0 + (n & 7)] : 0.0f;
    const bool bias = a.slopes != nullptr;

    const int bpp = c.page / B;
    const int64_t head_bytes = (int64_t)c.page * HD * ELEM;
    const uint32_t koff = (uint32_t)(n * HD * ELEM + q * 16), voff = (uint32_t)(n * 64 + q * 16);
    struct Where {
        const uint8_t *k, *v;
        const float *ks, *vs;
        int live;
    };
    auto where = [&](int b) {
        Where x;
        const int p = __builtin_amdgcn_readfirstlane(b / bpp), o = b - p * bpp;
        const int page = __builtin_amdgcn_readfirstlane(table[p]);
        const bool ok = page >= 0 && page < c.pages;
        const int64_t hr = (int64_t)(ok ? page : 0) * c.n_kv + kvh;
        x.k = c.k + hr * head_bytes + (int64_t)o * kBlock;
        x.v = c.v + hr * head_bytes + (int64_t)o * kBlock;
        x.ks = ELEM == 1 ? c.ks + hr * c.page + o * B : nullptr;
        x.vs = ELEM == 1 ? c.vs + hr * c.page + o * B : nullptr;
        const int64_t left = len - (int64_t)b * B;
        x.live = ok ? (int)(left < B ? left : B) : 0;
        return x;
    };
    uint4 kr[NT * NC], vr[ND];
    float4 ks[NT], vs[NT];
    auto load_k = [&](const Where &x) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
#pragma unroll
            for (int i = 0; i < NC; i++)
                kr[t * NC + i] = *reinterpret_cast<const uint4 *>(x.k + koff + t * 16 * HD * ELEM + i * 64);
            if constexpr (ELEM == 1) {
                ks[t] = *reinterpret_cast<const float4 *>(x.ks + 16 * t + 4 * q);
                vs[t] = *reinterpret_cast<const float4 *>(x.vs + 16 * t + 4 * q);
            }
        }
    };
    auto load_v = [&](const Where &x) {
#pragma unroll
        for (int d = 0; d < ND; d++) vr[d] = *reinterpret_cast<const uint4 *>(x.v + voff + d * 1024);
    };

    v4f acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = kLowest, ref2 = kLowest, l = 0.0f;  // ref2 = ref log2 e, rounded once
    int ve = ELEM == 1 ? -100 : 0;                   // the weights' power of two

    int b = b0 + w;
    Where cur{};
    if (b < b1) {
        cur = where(b);
        load_k(cur);
        load_v(cur);
    }
    for (; b < b1; b += pkv::kWaves) {
        const int live = cur.live, j0 = b * B;
        const bool more = b + pkv::kWaves < b1;
        Where next{};
        if (more) next = where(b + pkv::kWaves);
        // scores
        v4f s[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const uint4 x = kr[t * NC + i];
                if constexpr (ELEM == 1) {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(x.x, x.y), qf[2 * i], s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(x.z, x.w), qf[2 * i + 1], s[t], 0, 0, 0);
                } else {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(x), qf[i], s[t], 0, 0, 0);
                }
            }
        }
        float sv[NT * 4], vsc[NT * 4];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x = s[t][i] * own + llmq_dppf<0x128>(s[t][i]) * oth;  // row_ror:8
                if constexpr (ELEM == 1) {
                    x *= reinterpret_cast<const float *>(&ks[t])[i];
                    vsc[4 * t + i] = reinterpret_cast<const float *>(&vs[t])[i];
                }
                sv[4 * t + i] = x * mul;
            }
        if (more) load_k(next);
        if (a.cap > 0.0f)
#pragma unroll
            for (int i = 0; i < NT * 4; i++) sv[i] = a.cap * ref_tanhf(sv[i] / a.cap);
        if (bias) {
            const float base = (float)(j0 + 4 * q - (len - 1));
#pragma unroll
            for (int i = 0; i < NT * 4; i++) sv[i] = fmaf(slope, base + (float)(16 * (i >> 2) + (i & 3)), sv[i]);
        }
        if (live < B) {  // the row's end, or a page that is none
#pragma unroll
            for (int i = 0; i < NT * 4; i++) {
                const bool in = 16 * (i >> 2) + 4 * q + (i & 3) < live;
                sv[i] = in ? sv[i] : -INFINITY;
                if constexpr (ELEM == 1) vsc[i] = in ? vsc[i] : 0.0f;
            }
            if constexpr (ELEM == 2) {  // what lies there may be NaN
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    uint32_t *u = reinterpret_cast<uint32_t *>(&vr[d]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int p = 16 * (i >> 1) + 4 * q + 2 * (i & 1);
                        u[i] &= p + 1 < live ? 0xffffffffu : (p < live ? 0xffffu : 0u);
                    }
                }
            }
        }
        float mx = sv[0], vm = 0.0f;
#pragma unroll
        for (int i = 1; i < NT * 4; i++) mx = fmaxf(mx, sv[i]);
        mx = quarters_max(mx);
        int nve = ve;
        if constexpr (ELEM == 1) {
#pragma unroll
            for (int i = 0; i < NT * 4; i++) vm = fmaxf(vm, vsc[i]);
            vm = quarters_max(vm);
            nve = max(ve, (int)(__float_as_uint(vm) >> 23) - 127);
        }
        if (__any(mx > ref + 4.0f || nve > ve)) {  // 4 log2 e < 6
            const float to = fmaxf(ref, mx), to2 = to * kLog2e;
            const float f = ref == to ? 1.0f : exp2f(ref2 - to2), fl = ldexpf(f, ve - nve);
            ref = to;
            ref2 = ref == kLowest ? kLowest : to2;
            ve = nve;
            l *= f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = __shfl(fl, 4 * q + i);  // of row 4 q + i
#pragma unroll
                for (int d = 0; d < ND; d++) acc[d][i] *= x;
            }
        }
        const float unit = ldexpf(1.0f, 8 - ve);
        h8 wf[NT / 2];
#pragma unroll
        for (int i = 0; i < NT * 4; i++) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sv[i], kLog2e, -ref2));
            l += p;
            const float x = ELEM == 1 ? p * (vsc[i] * unit) : p * unit;
            const float hi = (float)(_Float16)x;
            // row n: x rounded; row n ^ 8: what that leaves times 2^11 (exact)
            wf[i >> 3][i & 7] = (_Float16)fmaf(hi, wr, x * wg);
        }
        // values
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const uint4 x = vr[d];
            if constexpr (ELEM == 1) {
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[0], halves(x.x, x.y), acc[d], 0, 0, 0);
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[1], halves(x.z, x.w), acc[d], 0, 0, 0);
            } else {
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[0], as_h8(x), acc[d], 0, 0, 0);
            }
        }
        if (more) {
            load_v(next);
            cur = next;
        }
    }
    // the four waves' results
    l = quarters_sum(l);
    if (lane < 8) wml[w][n] = make_float2(ref2, l);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = acc[d][i], y = __shfl_xor(x, 32);  // rows 4 q + i and 4 q + i + 8
            if (q < 2) wsum[w][4 * q + i][16 * d + n] = ldexpf(fmaf(y, 0x1p-11f, x), ve - 8);
        }
    __syncthreads();
    if (tid == 0 && blockIdx.y == 0 && part.split == 0 && a.shift >= 0) a.meta[r] = make_int2(part.first, count);
    for (int i = tid; i < hn * HD; i += 256) {
        const int h = i / HD, d = i % HD;
        float R = kLowest, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int k = 0; k < pkv::kWaves; k++) R = fmaxf(R, wml[k][h].x);
#pragma unroll
        for (int k = 0; k < pkv::kWaves; k++) {
            const float f = exp2f(wml[k][h].x - R);
            L = fmaf(wml[k][h].y, f, L);
            o = fmaf(wsum[k][h][d], f, o);
        }
        if (count == 1) {
            a.out[r * a.ldo + (int64_t)(h0 + h) * HD + d] = L == 0.0f ? 0.0f : o / L;
        } else {
            const int64_t at = (int64_t)blockIdx.x * a.n_head + h0 + h;
            a.sums[at * HD + d] = o;
            if (d == 0) a.ml[at] = make_float2(R, L);
        }
    }
}

// The splits of a row put together, in their order: a workgroup a (head, row).
template <int HD>
__global__ __launch_bounds__(256) void pkv_join_kernel(Attend a) {
    __shared__ float wl[pkv::kWaves], ws[pkv::kWaves][HD];
    const int64_t r = blockIdx.y;
    const int h = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int2 m = a.meta[r];
    if (m.y <= 1) return;
    const float2 *ml = a.ml + (int64_t)m.x * a.n_head + h;
    const float *sums = a.sums + ((int64_t)m.x * a.n_head + h) * HD;
    float R = kLowest;
    for (int i = lane; i < m.y; i += 64) R = fmaxf(R, ml[(int64_t)i * a.n_head].x);
    R = llmq_wave_max_all(R);
    float L = 0.0f, o[HD / 64] = {};
#pragma unroll 4
    for (int i = w; i < m.y; i += pkv::kWaves) {
        const float2 x = ml[(int64_t)i * a.n_head];
        const float f = exp2f(x.x - R);
        L = fmaf(x.y, f, L);
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] = fmaf(sums[(int64_t)i * a.n_head * HD + lane + 64 * d], f, o[d]);
    }
    if (lane == 0) wl[w] = L;
#pragma unroll
    for (int d = 0; d < HD / 64; d++) ws[w][lane + 64 * d] = o[d];
    __syncthreads();
    if (threadIdx.x < HD) {
        const int d = threadIdx.x;
        const float all = (wl[0] + wl[1]) + (wl[2] + wl[3]), s = (ws[0][d] + ws[1][d]) + (ws[2][d] + ws[3][d]);
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
    LLMQ_REQUIRE(kv->ctx->device == ctx->device, "%s: the cache is on device %d, the context on %d", name,
                 kv->ctx->device, ctx->device);
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
    LLMQ_REQUIRE(a.scale == a.scale && a.cap >= 0.0f && a.cap <= 3.0e38f, "%s: scale %g, cap %g", name, a.scale, a.cap);
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
    a.shift = p.shift;
    a.meta = static_cast<int2 *>(work);
    a.ml = reinterpret_cast<float2 *>(static_cast<uint8_t *>(work) + at.ml);
    a.sums = reinterpret_cast<float *>(static_cast<uint8_t *>(work) + at.sums);
    // tables too short for a second split need no joining
    const bool join = p.shift >= 0 && width * kv->page > (int64_t)pkv::kMinBlocks * pkv::block_positions(kv->elem());
    // columns a multiple of the 8 XCDs: the tiles of one cached head land on one
    const int64_t cols = p.shift >= 0 ? ((join ? p.slots : rows) + 7) / 8 * 8 : rows;
    return dispatch(kv, [&](auto hd, auto elem) -> int {
        hipLaunchKernelGGL((pkv_attend_kernel<decltype(hd)::value, decltype(elem)::value>),
                           dim3((unsigned)cols, (unsigned)(kv->n_kv * p.tiles)), dim3(256), 0, ctx->stream, c, a);
        if (join)
            hipLaunchKernelGGL((pkv_join_kernel<decltype(hd)::value>), dim3((unsigned)a.n_head, (unsigned)rows),
                               dim3(256), 0, ctx->stream, a);
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
    const double total = (double)n_layer * (double)n_pages * n_kv * page * head_dim * 2.0;
    LLMQ_REQUIRE(total < 1e15, "pkv_create: %g elements", total);
    llmq_pkv *kv = new (std::nothrow) llmq_pkv();
    if (!kv) return llmq_set_error(LLMQ_ENOMEM, "pkv_create: out of host memory");
    kv->ctx = ctx;
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
    if (hipMemsetAsync(kv->k, 0, n, ctx->stream) != hipSuccess ||
        hipMemsetAsync(kv->v, 0, n, ctx->stream) != hipSuccess ||
        (scales && (hipMemsetAsync(kv->ks, 0, ns, ctx->stream) != hipSuccess ||
                    hipMemsetAsync(kv->vs, 0, ns, ctx->stream) != hipSuccess))) {
        llmq_pkv_free(kv);
        return llmq_set_error(LLMQ_EHIP, "pkv_create: clearing the cache failed");
    }
    *out = kv;
    return LLMQ_OK;
}

int llmq_pkv_free(llmq_pkv *kv) {
    if (!kv) return LLMQ_OK;
    DeviceGuard guard(kv->ctx);
    hipStreamSynchronize(kv->ctx->stream);
    hipFree(kv->k);
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
                           dim3((unsigned)T, (unsigned)kv->n_kv), dim3(64), 0, ctx->stream, c, k, v, ld, seq, pos,
                           n_seq);
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
                           dim3((unsigned)T, (unsigned)kv->n_kv), dim3(64), 0, ctx->stream, c, k, v, ld, seq, pos,
                           n_seq);
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
    Attend a{out, ldo, q, nullptr, nullptr, ldq, len, n_head, scale, cap, slopes, 0, 0, 0, nullptr, nullptr, nullptr};
    return attend("pkv_attend", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

int llmq_pkv_step(llmq_ctx *ctx, llmq_pkv *kv, int layer, float *out, int64_t ldo, const float *q, const float *k,
                  const float *v, int64_t ld, int64_t rows, int n_head, const int32_t *pos, const int32_t *table,
                  int64_t width, float scale, float cap, const float *slopes, void *work, int64_t work_bytes) {
    LLMQ_REQUIRE((k && v) || rows == 0, "pkv_step: null argument");
    Attend a{out, ldo, q, k, v, ld, pos, n_head, scale, cap, slopes, 0, 0, 0, nullptr, nullptr, nullptr};
    return attend("pkv_step", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

}  // extern "C"
