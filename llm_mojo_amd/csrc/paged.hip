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
};

// One wave a (row, query head), a position at a time, with the running
// maximum and sum of the softmax; lane = dimension.
template <int HD, int ELEM>
__global__ __launch_bounds__(64) void pkv_attend_kernel(Layer c, Attend a) {
    const int64_t r = blockIdx.y;
    const int h = blockIdx.x, kvh = h / (a.n_head / c.n_kv), lane = threadIdx.x;
    const int32_t *row = c.table + r * c.width;
    int64_t len = a.len[r];
    if (a.k) {
        const int64_t p = len;
        len = p < 0 ? 0 : p + 1;
        const int page = pkv::page_of(row, c.width, c.page, c.pages, p);
        // every query head of the group writes the same bytes, which its own wave reads below
        if (page >= 0)
            store_row<HD, ELEM>(c, page, (int)(p % c.page), kvh, a.k + r * a.ldq + kvh * HD, a.v + r * a.ldq + kvh * HD,
                                lane);
        __threadfence_block();
    }
    len = pkv::clamp_len(len, c.width, c.page);
    float q[HD / 64], o[HD / 64], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 64; i++) {
        q[i] = a.q[r * a.ldq + h * HD + lane + 64 * i];
        o[i] = 0.0f;
    }
    const float slope = a.slopes ? a.slopes[h] : 0.0f;
    for (int64_t j = 0; j < len; j++) {
        const int page = pkv::page_of(row, c.width, c.page, c.pages, j);
        if (page < 0) continue;
        float k[HD / 64], v[HD / 64], s = 0.0f;
        load_row<HD, ELEM>(c, page, (int)(j % c.page), kvh, k, v, lane);
#pragma unroll
        for (int i = 0; i < HD / 64; i++) s = fmaf(q[i], k[i], s);
        s = llmq_wave_sum_all(s) * a.scale;
        if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
        s += slope * (float)(j - (len - 1));
        const float mn = fmaxf(m, s), old = m == mn ? 1.0f : expf(m - mn), e = expf(s - mn);
        m = mn;
        l = l * old + e;
#pragma unroll
        for (int i = 0; i < HD / 64; i++) o[i] = fmaf(e, v[i], o[i] * old);
    }
#pragma unroll
    for (int i = 0; i < HD / 64; i++)
        a.out[r * a.ldo + h * HD + lane + 64 * i] = l == 0.0f ? 0.0f : o[i] / l;
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

int attend(const char *name, llmq_ctx *ctx, const llmq_pkv *kv, int layer, const Attend &a, int64_t rows,
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
    DeviceGuard guard(ctx);
    const Layer c = layer_of(kv, layer, table, width);
    return dispatch(kv, [&](auto hd, auto elem) -> int {
        hipLaunchKernelGGL((pkv_attend_kernel<decltype(hd)::value, decltype(elem)::value>),
                           dim3((unsigned)a.n_head, (unsigned)rows), dim3(64), 0, ctx->stream, c, a);
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
    return 256;
}

int llmq_pkv_attend(llmq_ctx *ctx, const llmq_pkv *kv, int layer, float *out, int64_t ldo, const float *q, int64_t ldq,
                    int64_t rows, int n_head, const int32_t *len, const int32_t *table, int64_t width, float scale,
                    float cap, const float *slopes, void *work, int64_t work_bytes) {
    Attend a{out, ldo, q, nullptr, nullptr, ldq, len, n_head, scale, cap, slopes};
    return attend("pkv_attend", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

int llmq_pkv_step(llmq_ctx *ctx, llmq_pkv *kv, int layer, float *out, int64_t ldo, const float *q, const float *k,
                  const float *v, int64_t ld, int64_t rows, int n_head, const int32_t *pos, const int32_t *table,
                  int64_t width, float scale, float cap, const float *slopes, void *work, int64_t work_bytes) {
    LLMQ_REQUIRE((k && v) || rows == 0, "pkv_step: null argument");
    Attend a{out, ldo, q, k, v, ld, pos, n_head, scale, cap, slopes};
    return attend("pkv_step", ctx, kv, layer, a, rows, table, width, work, work_bytes);
}

}  // extern "C"
