// Rules on a head's logits and the greedy pick (include/llmq.h,
// llmq_adjust_logits): penalties for tokens a sequence holds already, biases,
// a grammar's mask.
//
// One pass over the logits, bound by reading and writing them.  A workgroup
// takes a row's next CHUNK entries into registers and, while they are on
// their way, counts the history's tokens that fall there in LDS (integer
// adds: the order does not matter), so no table of counts goes through
// memory; a history is read once a chunk, from the caches after the first.
// 256 rows x 50257 with histories of up to 2048 tokens, 64 biases and a mask
// take 28.9 us (106 MB, 3.7 TB/s), one row x 32000 5.2.
//
// Chunks of 2048 entries: 4096 took 37 us there, 512 threads 36.  Of 1024
// where larger ones would leave CUs without a workgroup.
#include <math.h>

#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 8;  // entries of the history a thread asks for at once
constexpr int kSmall = 1024, kLarge = 2048;  // entries of a workgroup

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
    return Span{lo < 0 ? 0 : (lo > len ? len : lo), hi > len ? len : hi};  // (positions past lo do not wrap)
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

__device__ __forceinline__ Best wave_best(Best b) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(b, __shfl_xor(b.v, o), __shfl_xor(b.i, o));
    return b;
}

__device__ __forceinline__ Best block_best(Best b, Best *red) {
    b = wave_best(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = b;
    __syncthreads();
    b = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) better(b, red[w].v, red[w].i);
    return b;
}

struct Float4 {
    float x[4];
} __attribute__((packed, aligned(4)));

template <int CHUNK>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(const float *in, int64_t ldi, float *out, int64_t ldo,
                                                                 int V, Rules u, Best *__restrict__ parts) {
    constexpr int N = CHUNK / (4 * kThreads);  // fours of entries a thread
    __shared__ __align__(16) int count[CHUNK];
    __shared__ __align__(16) float add[CHUNK];
    __shared__ __align__(16) int ids[kThreads + 4];  // (a batch's, then -1)
    __shared__ int from[kThreads / 64];
    __shared__ __align__(16) float val[kThreads + 4];
    __shared__ Best red[kThreads / 64];
    const int64_t r = blockIdx.y;
    const int v0 = blockIdx.x * CHUNK, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float *src = in + r * ldi;
    Float4 x[N];
    uint32_t bits[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int v = v0 + 4 * (tid + kThreads * k);
        bits[k] = 15;
        if (v + 4 <= V) {
            llmq_load4_once(src + v, x[k].x);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) x[k].x[i] = v + i < V ? src[v + i] : 0.0f;
        }
        if (u.mask && v < V) bits[k] = u.mask[r * u.mask_ld + (v >> 5)] >> (v & 31);
    }
    const float rep = u.rep ? u.rep[r] : 1.0f, pres = u.pres ? u.pres[r] : 0.0f, freq = u.freq ? u.freq[r] : 0.0f;
    const Span hist = u.hist ? span_of(u.hist_off, u.hist_len, r) : Span{0, 0};
    const Span bias = u.bias_ids ? span_of(u.bias_off, u.bias_len, r) : Span{0, 0};
    // the lists' first entries too, before anything waits
    int32_t h[kAhead], bid = -1;
    float bval = 0.0f;
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
        const int64_t i = hist.lo + tid + kThreads * k;
        h[k] = i < hist.hi ? u.hist[i] : -1;
    }
    if (bias.lo + tid < bias.hi) {
        bid = u.bias_ids[bias.lo + tid];
        bval = u.bias[bias.lo + tid];
    }
    if (hist.lo < hist.hi || bias.lo < bias.hi) {  // the same for the whole workgroup
#pragma unroll
        for (int k = 0; k < N; k++) {
            reinterpret_cast<int4 *>(count)[tid + kThreads * k] = make_int4(0, 0, 0, 0);
            reinterpret_cast<float4 *>(add)[tid + kThreads * k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        __syncthreads();
        auto seen = [&](int32_t id) {  // (a negative id is past every chunk)
            const uint32_t at = (uint32_t)id - (uint32_t)v0;
            if (at < (uint32_t)CHUNK) atomicAdd(&count[at], 1);
        };
#pragma unroll
        for (int k = 0; k < kAhead; k++) seen(h[k]);
        for (int64_t i = hist.lo + tid + kThreads * kAhead; i < hist.hi; i += kThreads) seen(u.hist[i]);
        // biases, a batch of kThreads at a time: those of this chunk go to
        // LDS in the list's order, and the first of each token adds up all
        // of its token's in that order
        for (int64_t i0 = bias.lo; i0 < bias.hi; i0 += kThreads) {
            const uint32_t at = (uint32_t)bid - (uint32_t)v0;
            const float b = bval;
            const bool in_chunk = at < (uint32_t)CHUNK;
            bid = -1;
            if (i0 + kThreads + tid < bias.hi) {
                bid = u.bias_ids[i0 + kThreads + tid];
                bval = u.bias[i0 + kThreads + tid];
            }
            const uint64_t who = __ballot(in_chunk);
            if (lane == 0) from[w] = __popcll(who);
            __syncthreads();
            int n = 0, first = 0;
#pragma unroll
            for (int k = 0; k < kThreads / 64; k++) {
                if (k == w) first = n;
                n += from[k];
            }
            if (in_chunk) {
                const int k = first + __popcll(who & ((1ull << lane) - 1));
                ids[k] = (int)at;
                val[k] = b;
            }
            if (tid < 4) ids[n + tid] = -1;
            __syncthreads();
            if (tid < n) {
                const int mine = ids[tid];
                int lead = -1;
                float s = add[mine];
                for (int k = 0; k < n; k += 4) {  // (the same for all lanes: four reads in one)
                    const int4 id = *reinterpret_cast<const int4 *>(ids + k);
                    const float4 b4 = *reinterpret_cast<const float4 *>(val + k);
                    const int is[4] = {id.x, id.y, id.z, id.w};
                    const float bs[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const bool same = is[j] == mine;
                        lead = same && lead < 0 ? k + j : lead;
                        s = same ? s + bs[j] : s;
                    }
                }
                if (lead == tid) add[mine] = s;
            }
            __syncthreads();
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int4 c4 = reinterpret_cast<const int4 *>(count)[tid + kThreads * k];
            const float4 a4 = reinterpret_cast<const float4 *>(add)[tid + kThreads * k];
            const int c[4] = {c4.x, c4.y, c4.z, c4.w};
            const float a[4] = {a4.x, a4.y, a4.z, a4.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float l = x[k].x[i];
                if (c[i] > 0) {
                    if (u.rep) l = l > 0.0f ? l / rep : l * rep;
                    l = l - (freq * (float)c[i] + pres);
                }
                x[k].x[i] = u.bias_ids ? l + a[i] : l;
            }
        }
    } else if (u.bias_ids) {  // what adding no bias does: -0 becomes 0
#pragma unroll
        for (int k = 0; k < N; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) x[k].x[i] += 0.0f;
    }
    Best b{-INFINITY, INT32_MAX};
    float *dst = out + r * ldo;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int v = v0 + 4 * (tid + kThreads * k);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!((bits[k] >> i) & 1)) x[k].x[i] = -INFINITY;
            if (x[k].x[i] > b.v && v + i < V) {  // never for NaN and -inf
                b.v = x[k].x[i];
                b.i = v + i;
            }
        }
        if (v + 4 <= V) {
            *reinterpret_cast<Float4 *>(dst + v) = x[k];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (v + i < V) dst[v + i] = x[k].x[i];
        }
    }
    if (!parts) return;
    b = block_best(b, red);
    if (tid == 0) parts[r * gridDim.x + blockIdx.x] = b;
}

// A row's chunks' picks put together: a wave a row (4 us for 256 rows of 25, most of it the launch).
__global__ __launch_bounds__(64) void pick_kernel(const Best *__restrict__ parts, int n, int64_t *__restrict__ pick) {
    const Best *p = parts + (int64_t)blockIdx.x * n;
    Best b{-INFINITY, INT32_MAX};
    for (int i = threadIdx.x; i < n; i += 64) better(b, p[i].v, p[i].i);
    b = wave_best(b);
    if (threadIdx.x == 0) pick[blockIdx.x] = b.i == INT32_MAX ? -1 : b.i;
}

}  // namespace

namespace {

// Small chunks where large ones would leave CUs without a workgroup.
int chunk_of(int64_t rows, int64_t V) { return rows * ((V + kLarge - 1) / kLarge) < 512 ? kSmall : kLarge; }

}  // namespace

extern "C" {

int64_t llmq_adjust_logits_work_bytes(int64_t rows, int64_t V) {
    if (rows < 0 || rows > 65535 || V <= 0 || V > INT32_MAX / 2) return -1;
    const int chunk = chunk_of(rows, V);
    return rows * ((V + chunk - 1) / chunk) * (int64_t)sizeof(Best) + 16;
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
    LLMQ_REQUIRE(!pick || (uintptr_t)work % 16 == 0, "adjust_logits: work is 16-byte aligned");
    DeviceGuard guard(ctx);
    const int chunk = chunk_of(rows, V), n = (int)((V + chunk - 1) / chunk);
    Best *parts = pick ? static_cast<Best *>(work) : nullptr;
    auto kernel = chunk == kSmall ? adjust_logits_kernel<kSmall> : adjust_logits_kernel<kLarge>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)n, (unsigned)rows), dim3(kThreads), 0, ctx->stream, logits, ldl, out, ldo,
                       (int)V, u, parts);
    if (pick)
        hipLaunchKernelGGL(pick_kernel, dim3((unsigned)rows), dim3(64), 0, ctx->stream, parts, n, pick);
    LLMQ_HIP(hipGetLastError());
    return LLMQ_OK;
}

}  // extern "C"
