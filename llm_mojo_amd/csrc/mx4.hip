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
// Rows and blocks past the matrix's end are zero codes with scale 127.
#include <math.h>

#include <new>
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

// llmq_mx4_quantize: a thread a block.
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const float *__restrict__ x, int64_t ldx, int64_t nb,
                                                           int64_t total, uint4 *__restrict__ codes,
                                                           uint8_t *__restrict__ scales) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const float *p = x + (i / nb) * ldx + (i % nb) * 32;
    float v[32];
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = p[j];
    int e;
    codes[i] = quant_block(v, &e);
    scales[i] = (uint8_t)e;
}

__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, int64_t nb,
                                                             int64_t total, float *__restrict__ out, int64_t ldo) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    float *p = out + (i / nb) * ldo + (i % nb) * 32;
    const float s = scale_value(scales[i]);
    for (int j = 0; j < 32; j++) p[j] = code_value((codes[i * 16 + j / 2] >> (4 * (j & 1))) & 15) * s;
}

// A weight matrix from floats: a thread a (row, block); with reduce_rows
// (source [IN, OUT]) neighbouring threads read neighbouring floats.
__global__ __launch_bounds__(256) void mx4_weights_kernel(const float *__restrict__ src, int64_t cols, int reduce_rows,
                                                          int64_t n, int64_t nb, int64_t steps, int64_t words,
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
    codes[(tile * steps + step) * 64 + lane] = c;
    scales[((tile * words + (step >> 2)) * 64 + lane) * 4 + (step & 3)] = (uint8_t)e;
}

// act(sum + bias) (+ what is there): the epilogue of every product here.
__device__ __forceinline__ void finish(float *p, float y, const float *bias, int64_t o, int flags) {
    if (flags & LLMQ_BIAS) y = y + bias[o];
    if (flags & LLMQ_GELU) y = gelu_ref(y);
    if (flags & LLMQ_RESID) y = *p + y;
    *p = y;
}

// One wave a (16 outputs, 16 tokens).
__global__ __launch_bounds__(64) void mx4_linear_kernel(const uint4 *__restrict__ xc, const uint8_t *__restrict__ xs,
                                                        const uint4 *__restrict__ wc, const uint32_t *__restrict__ ws,
                                                        int64_t T, int64_t n, int64_t nb, int64_t steps, int64_t words,
                                                        float *__restrict__ out, const float *__restrict__ bias,
                                                        int flags) {
    const int lane = threadIdx.x, q = lane >> 4;
    const int64_t tile = blockIdx.x, t = (int64_t)blockIdx.y * 16 + (lane & 15);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t s = 0; s < steps; s++) {
        const uint4 a = wc[(tile * steps + s) * 64 + lane];
        const int as = (int)(ws[(tile * words + (s >> 2)) * 64 + lane] >> (8 * (s & 3)));
        const int64_t b = s * 4 + q;
        const bool in = t < T && b < nb;
        const uint4 x = in ? xc[t * nb + b] : make_uint4(0, 0, 0, 0);
        const int bs = in ? xs[t * nb + b] : 127;
        const v8i av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0},
                  bv = {(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0};
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, as, 0, bs);
    }
    if (t >= T) return;
    for (int i = 0; i < 4; i++) {
        const int64_t o = tile * 16 + 4 * q + i;
        if (o < n) finish(out + t * n + o, acc[i], bias, o, flags);
    }
}

int check_shape(const char *name, int64_t rows, int64_t cols) {
    LLMQ_REQUIRE(rows > 0 && cols > 0, "%s: empty matrix", name);
    LLMQ_REQUIRE(cols % 32 == 0, "%s: %lld inputs are no whole blocks of 32", name, (long long)cols);
    LLMQ_REQUIRE(rows <= INT32_MAX - 64 && cols <= INT32_MAX - 1024, "%s: %lld x %lld matrix", name, (long long)rows,
                 (long long)cols);
    return LLMQ_OK;
}

int mx4_alloc(llmq_ctx *ctx, int64_t n, int64_t k, llmq_mat **out) {
    llmq_mat *m = new (std::nothrow) llmq_mat();
    if (!m) return llmq_set_error(LLMQ_ENOMEM, "from_f32_mx4: out of host memory");
    m->ctx = ctx;
    m->kind = MAT_MX4;
    m->bits = 4;
    m->n = n;
    m->k = k;
    m->group = m->group_param = 32;
    m->ntiles = (n + 15) / 16;
    m->CK = (k + 127) / 128;
    m->NG = (m->CK + 3) / 4;
    const size_t cb = (size_t)(m->ntiles * m->CK) * 1024, sb = (size_t)(m->ntiles * m->NG) * 256;
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
    return Place{(tile * m->CK + step) * 64 + lane, ((tile * m->NG + (step >> 2)) * 64 + lane) * 4 + (step & 3)};
}

int check_codes(const char *name, const llmq_ctx *ctx, const void *a, const void *codes, const void *scales, int64_t T,
                int64_t K) {
    LLMQ_REQUIRE(ctx && ((a && codes && scales) || T == 0), "%s: null argument", name);
    LLMQ_REQUIRE(T >= 0 && T <= INT32_MAX && K > 0 && K % 32 == 0 && K <= INT32_MAX - 1024,
                 "%s: %lld rows of %lld (whole blocks of 32)", name, (long long)T, (long long)K);
    LLMQ_REQUIRE((uintptr_t)codes % 16 == 0, "%s: codes are 16-byte aligned", name);
    return LLMQ_OK;
}

int launch_quantize(llmq_ctx *ctx, const float *x, int64_t ldx, int64_t T, int64_t K, uint8_t *codes,
                    uint8_t *scales) {
    const int64_t nb = K / 32, total = T * nb, grid = (total + 255) / 256;
    LLMQ_REQUIRE(grid <= INT32_MAX, "mx4_quantize: %lld rows of %lld", (long long)T, (long long)K);
    hipLaunchKernelGGL(mx4_quantize_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, x, ldx, nb, total,
                       reinterpret_cast<uint4 *>(codes), scales);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

int launch_product(llmq_ctx *ctx, const uint8_t *codes, const uint8_t *scales, const llmq_mat *w, int64_t T, float *out,
                   const float *bias, int flags) {
    const int64_t tt = (T + 15) / 16;
    LLMQ_REQUIRE(tt <= 65535, "mx4_linear: %lld tokens", (long long)T);
    hipLaunchKernelGGL(mx4_linear_kernel, dim3((unsigned)w->ntiles, (unsigned)tt), dim3(64), 0, ctx->stream,
                       reinterpret_cast<const uint4 *>(codes), scales, reinterpret_cast<const uint4 *>(w->codes),
                       reinterpret_cast<const uint32_t *>(w->scales), T, w->n, w->k / 32, w->CK, w->NG, out, bias,
                       flags);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

int check_epilogue(const char *name, const float *out, const float *bias, int64_t T, int flags) {
    LLMQ_REQUIRE(out || T == 0, "%s: null output", name);
    LLMQ_REQUIRE(!(flags & ~(LLMQ_BIAS | LLMQ_GELU | LLMQ_RESID)), "%s: flags %d", name, flags);
    LLMQ_REQUIRE(!(flags & LLMQ_BIAS) || bias, "%s: null bias", name);
    return LLMQ_OK;
}

}  // namespace

int64_t mx4_record_bytes(int64_t T, int64_t K) { return ((T * K / 2 + 255) & ~(int64_t)255) + T * K / 32; }

int launch_mx4_linear(llmq_ctx *ctx, const llmq_mat *w, const float *x, int64_t T, float *out, const float *bias,
                      int flags, void *rec, int64_t rec_cap) {
    RC(check_epilogue("linear", out, bias, T, flags));
    LLMQ_REQUIRE(T >= 0 && T <= INT32_MAX && (x || T == 0), "linear: %lld microscaled tokens", (long long)T);
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
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
    uint8_t *codes = static_cast<uint8_t *>(rec), *scales = codes + ((T * w->k / 2 + 255) & ~(int64_t)255);
    RC(launch_quantize(ctx, x, w->k, T, w->k, codes, scales));
    return launch_product(ctx, codes, scales, w, T, out, bias, flags);
}

int mx4_dequant_row(llmq_ctx *ctx, const llmq_mat *m, int64_t row, float *dst) {
    DeviceGuard guard(ctx);
    const int64_t nb = m->k / 32, tile = row >> 4, r = row & 15;
    std::vector<uint8_t> c((size_t)m->CK * 1024), s((size_t)m->NG * 256);
    LLMQ_HIP(hipMemcpyAsync(c.data(), m->codes + tile * m->CK * 1024, c.size(), hipMemcpyDeviceToHost, ctx->stream));
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
    const int64_t nb = K / 32, total = T * nb, grid = (total + 255) / 256;
    LLMQ_REQUIRE(grid <= INT32_MAX, "mx4_dequantize: %lld rows of %lld", (long long)T, (long long)K);
    hipLaunchKernelGGL(mx4_dequantize_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, codes, scales, nb, total,
                       out, ldo);
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
    DeviceGuard guard(ctx);
    llmq_mat *m = nullptr;
    RC(mx4_alloc(ctx, n, k, &m));
    hipLaunchKernelGGL(mx4_weights_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, src, cols, reduce_rows, n,
                       nb, m->CK, m->NG, reinterpret_cast<uint4 *>(m->codes), reinterpret_cast<uint8_t *>(m->scales));
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
    if (rc == LLMQ_OK) rc = llmq_mat_from_f32_mx4_device(ctx, d, rows, cols, reduce_rows, out);
    hipStreamSynchronize(ctx->stream);
    hipFree(d);
    return rc;
}

int llmq_mat_restore_mx4(llmq_ctx *ctx, int64_t rows, int64_t cols, const uint8_t *codes, const uint8_t *scales,
                         llmq_mat **out) {
    LLMQ_REQUIRE(ctx && codes && scales && out, "restore_mx4: null argument");
    RC(check_shape("restore_mx4", rows, cols));
    DeviceGuard guard(ctx);
    llmq_mat *m = nullptr;
    RC(mx4_alloc(ctx, rows, cols, &m));
    int rc = LLMQ_OK;
    try {
        const int64_t nb = cols / 32;
        std::vector<uint8_t> c((size_t)(m->ntiles * m->CK) * 1024, 0), s((size_t)(m->ntiles * m->NG) * 256, 127);
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
    DeviceGuard guard(ctx);
    try {
        std::vector<uint8_t> c((size_t)(m->ntiles * m->CK) * 1024), s((size_t)(m->ntiles * m->NG) * 256);
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
    RC(check_epilogue("mx4_linear", out, bias, T, flags));
    if (T == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    return launch_product(ctx, codes, scales, w, T, out, bias, flags);
}

}  // extern "C"
