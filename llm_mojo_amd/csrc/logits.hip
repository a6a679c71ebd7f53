// Rules on a head's logits and the greedy pick (include/llmq.h,
// llmq_adjust_logits): penalties for tokens a sequence holds already, biases,
// a grammar's mask.
//
// One pass over the logits.  A workgroup takes a row's next kChunk entries
// and counts the history's tokens that fall there in LDS (integer adds: the
// order does not matter), so no table of counts goes through memory; a
// history is read once a chunk, from the caches after the first.
#include <math.h>

#include "common.h"

namespace {

constexpr int kChunk = 4096, kThreads = 256;
constexpr int kPer = kChunk / kThreads;

struct Rules {
    const int32_t *hist;
    const int64_t *hist_off;
    int64_t hist_len;
    const float *rep, *pres, *freq;
    const int32_t *bias_ids;
    const float *bias;
    const int64_t *bias_off;
    int64_t bias_len;
    const uint32_t *mask;
    int64_t mask_ld;
};

// Entries lo .. hi - 1 of a list of len are row r's; offsets that lead
// outside the list are taken to its ends.
struct Span {
    int64_t lo, hi;
};
__device__ __forceinline__ Span span_of(const int64_t *off, int64_t len, int64_t r) {
    const int64_t lo = off[r], hi = off[r + 1];
    return Span{lo < 0 ? 0 : lo, hi > len ? len : hi};
}

struct Best {
    float v;
    int i;
};

// The larger value, the lower index between equals; index INT_MAX: none.
__device__ __forceinline__ void better(Best &a, float v, int i) {
    if (v > a.v || (v == a.v && i < a.i)) {
        a.v = v;
        a.i = i;
    }
}

__device__ __forceinline__ Best block_best(Best b, Best *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(b, __shfl_xor(b.v, o), __shfl_xor(b.i, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = b;
    __syncthreads();
    b = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) better(b, red[w].v, red[w].i);
    return b;
}

__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const float *__restrict__ in, int64_t ldi,
                                                                 float *__restrict__ out, int64_t ldo, int V, Rules u,
                                                                 Best *__restrict__ parts) {
    __shared__ int count[kChunk];
    __shared__ float add[kChunk];
    __shared__ Best red[kThreads / 64];
    const int64_t r = blockIdx.y;
    const int v0 = blockIdx.x * kChunk, tid = threadIdx.x;
    for (int i = tid; i < kChunk; i += kThreads) {
        count[i] = 0;
        add[i] = 0.0f;
    }
    __syncthreads();
    if (u.hist) {
        const Span s = span_of(u.hist_off, u.hist_len, r);
        for (int64_t i = s.lo + tid; i < s.hi; i += kThreads) {
            const uint32_t at = (uint32_t)u.hist[i] - (uint32_t)v0;
            if (at < (uint32_t)kChunk) atomicAdd(&count[at], 1);
        }
    }
    // biases of one token in the list's order: one thread adds them all
    if (u.bias_ids && tid == 0) {
        const Span s = span_of(u.bias_off, u.bias_len, r);
        for (int64_t i = s.lo; i < s.hi; i++) {
            const uint32_t at = (uint32_t)u.bias_ids[i] - (uint32_t)v0;
            if (at < (uint32_t)kChunk) add[at] += u.bias[i];
        }
    }
    __syncthreads();
    const float rep = u.rep ? u.rep[r] : 1.0f, pres = u.pres ? u.pres[r] : 0.0f, freq = u.freq ? u.freq[r] : 0.0f;
    Best b{-INFINITY, INT32_MAX};
    for (int i = tid; i < kChunk && v0 + i < V; i += kThreads) {
        const int v = v0 + i;
        float l = in[r * ldi + v];
        const int c = count[i];
        if (c > 0) {
            if (u.rep) l = l > 0.0f ? l / rep : l * rep;
            l = l - (freq * (float)c + pres);
        }
        if (u.bias_ids) l = l + add[i];
        if (u.mask && !((u.mask[r * u.mask_ld + (v >> 5)] >> (v & 31)) & 1)) l = -INFINITY;
        out[r * ldo + v] = l;
        if (l > b.v) {  // never for NaN and -inf
            b.v = l;
            b.i = v;
        }
    }
    if (!parts) return;
    b = block_best(b, red);
    if (tid == 0) parts[r * gridDim.x + blockIdx.x] = b;
}

__global__ __launch_bounds__(kThreads) void pick_kernel(const Best *__restrict__ parts, int n,
                                                        int64_t *__restrict__ pick) {
    __shared__ Best red[kThreads / 64];
    const Best *p = parts + (int64_t)blockIdx.x * n;
    Best b{-INFINITY, INT32_MAX};
    for (int i = threadIdx.x; i < n; i += kThreads) better(b, p[i].v, p[i].i);
    b = block_best(b, red);
    if (threadIdx.x == 0) pick[blockIdx.x] = b.i == INT32_MAX ? -1 : b.i;
}

}  // namespace

extern "C" {

int64_t llmq_adjust_logits_work_bytes(int64_t rows, int64_t V) {
    if (rows < 0 || rows > 65535 || V <= 0 || V > INT32_MAX / 2) return -1;
    return rows * ((V + kChunk - 1) / kChunk) * (int64_t)sizeof(Best) + 16;
}

int llmq_adjust_logits(llmq_ctx *ctx, float *out, int64_t ldo, const float *logits, int64_t ldl, int64_t rows,
                       int64_t V, const llmq_logit_rules *rules, int64_t *pick, void *work, int64_t work_bytes) {
    LLMQ_REQUIRE(ctx && ((out && logits) || rows == 0), "adjust_logits: null argument");
    LLMQ_REQUIRE(rows >= 0 && rows <= 65535, "adjust_logits: %lld rows (at most 65535)", (long long)rows);
    LLMQ_REQUIRE(V > 0 && V <= INT32_MAX / 2, "adjust_logits: a vocabulary of %lld", (long long)V);
    LLMQ_REQUIRE(ldo >= V && ldl >= V, "adjust_logits: row strides %lld, %lld below %lld", (long long)ldo,
                 (long long)ldl, (long long)V);
    Rules u{};
    if (rules) {
        const llmq_logit_rules &s = *rules;
        LLMQ_REQUIRE(s.history_len >= 0 && s.bias_len >= 0, "adjust_logits: lists of %lld and %lld entries",
                     (long long)s.history_len, (long long)s.bias_len);
        LLMQ_REQUIRE(s.history_len == 0 || (s.history && s.history_offsets), "adjust_logits: half a history");
        LLMQ_REQUIRE(s.bias_len == 0 || (s.bias_ids && s.bias && s.bias_offsets),
                     "adjust_logits: half a list of biases");
        LLMQ_REQUIRE(!s.mask || s.mask_ld >= (V + 31) / 32, "adjust_logits: mask rows of %lld words for %lld tokens",
                     (long long)s.mask_ld, (long long)V);
        // an empty list is none
        u = Rules{s.history_len ? s.history : nullptr, s.history_offsets, s.history_len, s.repetition, s.presence,
                  s.frequency, s.bias_len ? s.bias_ids : nullptr, s.bias, s.bias_offsets, s.bias_len, s.mask,
                  s.mask_ld};
    }
    const int64_t want = pick ? llmq_adjust_logits_work_bytes(rows, V) : 0;
    LLMQ_REQUIRE(!pick || rows == 0 || (work && work_bytes >= want), "adjust_logits: %lld bytes of work, %lld needed",
                 (long long)work_bytes, (long long)want);
    if (rows == 0) return LLMQ_OK;
    DeviceGuard guard(ctx);
    const int n = (int)((V + kChunk - 1) / kChunk);
    Best *parts = pick ? static_cast<Best *>(work) : nullptr;
    hipLaunchKernelGGL(adjust_logits_kernel, dim3((unsigned)n, (unsigned)rows), dim3(kThreads), 0, ctx->stream, logits,
                       ldl, out, ldo, (int)V, u, parts);
    if (pick)
        hipLaunchKernelGGL(pick_kernel, dim3((unsigned)rows), dim3(kThreads), 0, ctx->stream, parts, n, pick);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

}  // extern "C"
