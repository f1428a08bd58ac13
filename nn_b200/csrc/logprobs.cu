// Log probabilities of given tokens under rows of logits, with the entropy of each row and its most probable tokens.
//
//   lse = m + ln sum e^(x - m);  log p(t) = x_t - lse;  H = -sum p ln p = ln l - T / l,  l = sum e^(x - m), T = sum e^(x - m) (x - m)
//
// One pass over a row keeps the running maximum, l and T (every term of T has the same sign; a new maximum m' scales l by
// f = e^(m - m') and makes T f (T + (m - m') l)); exponents are taken to base 2. All of it is f32.
// A row is dealt to a cluster of CTAs where the rows are few, and every CTA's sums meet in the first one's shared memory, in order.
// The most probable tokens: the 32 warps' worth of threads (groups of threads with the same lane) have seen 32 disjoint parts of the
// CTA's slice, so at least 32 elements are not below the least of the 32 parts' maxima. A second pass, which finds the slice in L2,
// collects the elements from that bound on (some hundred of the real rows), whose ranks are counted; where they are more than there
// is room for (rows of equal values), the largest element below the one before is looked for `top` times. Order: larger value first, then
// the lower index.
// The reference turns logits into probabilities on the host (crates/nn-core/src/layers/generation/autoregressive_sampling.rs:14-21 and
// the samplers beside it).
#include <algorithm>

#include "kv_cache.cuh"
#include "tcgen05.cuh"

namespace nnq {

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32, kLpRoom = 1024, kLpTop = 32;
constexpr float kLpLog2E = 1.4426950408889634f, kLpLn2 = 0.6931471805599453f;

struct LogprobArgs {
    const void *x;
    const int32_t *token;
    float *logprob, *entropy, *top_logprob;
    int32_t *top_token;
    int64_t ld;
    int vocab, top, slice;   // slice: elements of a row that a CTA has, a multiple of 8
    int *status;
};

struct Stats {   // maximum, sum of 2^d and of 2^d d, d = (x - m) log2 e
    float m, l, t;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float m = fmaxf(a.m, b.m), r = finite_ref(m);
    const float da = (finite_ref(a.m) - r) * kLpLog2E, db = (finite_ref(b.m) - r) * kLpLog2E;
    // (a side without elements has sums of zero; its reference does not matter)
    const float fa = a.l == 0.0f ? 0.0f : exp2f(da), fb = b.l == 0.0f ? 0.0f : exp2f(db);
    return {m, fmaf(a.l, fa, b.l * fb), (a.l == 0.0f ? 0.0f : fa * fmaf(fmaxf(da, -1e4f), a.l, a.t)) + (b.l == 0.0f ? 0.0f : fb * fmaf(fmaxf(db, -1e4f), b.l, b.t))};
}

// order of logits as unsigned numbers; NaN above everything
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);   // (-0 equals 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, int i) { return (uint64_t)order_bits(x) << 32 | (0xFFFFFFFFu - (uint32_t)i); }

template <bool F32>
__device__ __forceinline__ float logit(const void *x, int64_t i) {
    if constexpr (F32) return reinterpret_cast<const float *>(x)[i];
    else return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i]);
}

// f(value, index in the row) for the elements [lo, hi) of a row: 16 bytes at a time from the first aligned one on
template <bool F32, typename F>
__device__ __forceinline__ void each_logit(const void *row, int lo, int hi, F f) {
    constexpr int V = F32 ? 4 : 8;
    const uint8_t *p = reinterpret_cast<const uint8_t *>(row);
    const int size = F32 ? 4 : 2, tid = threadIdx.x;
    const int head = min(hi, lo + (int)((16 - ((uintptr_t)(p + (int64_t)lo * size) & 15u)) % 16 / size));
    for (int i = lo + tid; i < head; i += kLpThreads) f(logit<F32>(row, i), i);
    const int vecs = (hi - head) / V;
    const uint4 *q = reinterpret_cast<const uint4 *>(p + (int64_t)head * size);
#pragma unroll 4
    for (int u = tid; u < vecs; u += kLpThreads) {
        const uint4 w = __ldg(q + u);
        const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float v = F32 ? __uint_as_float(c[e & 3]) : __uint_as_float(e & 1 ? c[e >> 1] & 0xFFFF0000u : c[e >> 1] << 16);
            f(v, head + u * V + e);
        }
    }
    for (int i = head + vecs * V + tid; i < hi; i += kLpThreads) f(logit<F32>(row, i), i);
}

template <bool F32>
__global__ void __launch_bounds__(kLpThreads) logprobs_kernel(const LogprobArgs a) {
    __shared__ Stats warp_stats[kLpWarps], cta_stats;
    __shared__ float part_max[kLpWarps][32];
    __shared__ float bound_s;
    __shared__ int found;
    __shared__ uint64_t room[kLpRoom];
    __shared__ uint64_t best[kLpTop];
    __shared__ uint64_t red[kLpWarps];
    pdl_prologue();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = gridDim.x, me = blockIdx.x;
    const int64_t row = blockIdx.y;
    const void *x = reinterpret_cast<const uint8_t *>(a.x) + row * a.ld * (F32 ? 4 : 2);
    const int lo = min(a.vocab, me * a.slice), hi = min(a.vocab, lo + a.slice);
    Stats s = {-INFINITY, 0.0f, 0.0f};
    each_logit<F32>(x, lo, hi, [&](float v, int) {
        if (v > s.m) {
            const float d = (finite_ref(s.m) - v) * kLpLog2E, f = s.l == 0.0f ? 0.0f : exp2f(d);
            s.t = s.l == 0.0f ? 0.0f : f * fmaf(fmaxf(d, -1e4f), s.l, s.t);
            s.l *= f;
            s.m = v;
        }
        const float d = (v - finite_ref(s.m)) * kLpLog2E, e = exp2f(d);
        s.l += e;
        s.t = fmaf(e, fmaxf(d, -1e4f), s.t);
    });
    const float mine = s.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.l, o), __shfl_xor_sync(0xFFFFFFFFu, s.t, o)});
    if (lane == 0) warp_stats[warp] = s;
    if (tid == 0) found = 0;
    part_max[warp][lane] = mine;
    __syncthreads();
    if (warp == 0) {
        s = lane < kLpWarps ? warp_stats[lane] : Stats{-INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s = join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.m, o), __shfl_xor_sync(0xFFFFFFFFu, s.l, o), __shfl_xor_sync(0xFFFFFFFFu, s.t, o)});
        if (lane == 0) cta_stats = s;
        float b = -INFINITY;   // maximum of the elements that the threads of this lane have seen
        for (int w = 0; w < kLpWarps; w++) b = fmaxf(b, part_max[w][lane]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) b = fminf(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
        if (lane == 0) bound_s = b;
    }
    __syncthreads();
    if (a.top > 0) {
        const float bound = bound_s;
        each_logit<F32>(x, lo, hi, [&](float v, int i) {
            if (!(v < bound)) {   // (a NaN as well)
                const int at = atomicAdd(&found, 1);
                if (at < kLpRoom) room[at] = order_key(v, i);
            }
        });
        if (tid < kLpTop) best[tid] = 0;   // below every key
        __syncthreads();
        const int n = found;
        if (n <= kLpRoom) {
            for (int i = tid; i < n; i += kLpThreads) {
                const uint64_t k = room[i];
                int rank = 0;
                for (int j = 0; j < n; j++) rank += room[j] > k;
                if (rank < a.top) best[rank] = k;
            }
        } else {
            uint64_t below = ~0ull;
            for (int i = 0; i < a.top; i++) {
                uint64_t b = 0;
                each_logit<F32>(x, lo, hi, [&](float v, int j) {
                    const uint64_t k = order_key(v, j);
                    if (k < below && k > b) b = k;
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
                __syncthreads();
                if (lane == 0) red[warp] = b;
                __syncthreads();
                for (int w = 0; w < kLpWarps; w++) b = max(b, red[w]);
                if (tid == 0) best[i] = b;
                below = b;
                if (b == 0) break;   // the slice has fewer elements
            }
        }
        __syncthreads();
    }
    if (ctas > 1) cluster_sync();
    if (me == 0) {
        const uint32_t stats_at = smem_u32(&cta_stats), best_at = smem_u32(best);
        s = cta_stats;
        for (int c = 1; c < ctas; c++) {
            Stats o;
            const uint32_t p = cluster_addr(stats_at, c);
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.m) : "r"(p) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.l) : "r"(p + 4) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o.t) : "r"(p + 8) : "memory");
            s = join(s, o);
        }
        const float log_l = log2f(s.l), r = finite_ref(s.m);
        const bool none = s.m == -INFINITY && s.l == 0.0f;   // no token has any probability
        auto log_prob = [&](float v) { return none ? v : fmaf(v - r, 1.0f, -log_l * kLpLn2); };
        if (tid == 0) {
            const int t = a.token ? a.token[row] : -1;
            if (t >= a.vocab) atomicExch(a.status, kStatusIndex);
            if (a.logprob) a.logprob[row] = t < 0 ? 0.0f : t >= a.vocab ? __int_as_float(0x7FFFFFFF) : log_prob(logit<F32>(x, t));
            if (a.entropy) a.entropy[row] = none ? 0.0f : (log_l - s.t / s.l) * kLpLn2;
        }
        if (a.top > 0) {
            __syncthreads();
            for (int i = tid; i < ctas * kLpTop; i += kLpThreads) {
                uint64_t k;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(cluster_addr(best_at + 8 * (i % kLpTop), i / kLpTop)) : "memory");
                room[i] = k;
            }
            __syncthreads();
            for (int i = tid; i < ctas * kLpTop; i += kLpThreads) {
                const uint64_t k = room[i];
                if (k == 0) continue;
                int rank = 0;
                for (int j = 0; j < ctas * kLpTop; j++) rank += room[j] > k;
                if (rank >= a.top) continue;
                const int idx = (int)(0xFFFFFFFFu - (uint32_t)k);
                if (a.top_token) a.top_token[row * a.top + rank] = idx;
                if (a.top_logprob) a.top_logprob[row * a.top + rank] = log_prob(logit<F32>(x, idx));
            }
        }
    }
    if (ctas > 1) cluster_sync();   // the other CTAs' shared memory has been read
}

}  // namespace nnq

using namespace nnq;

extern "C" {

nnq_status nnq_token_logprobs(nnq_ctx *ctx, const void *logits_dev, nnq_dtype dt, int64_t rows, int64_t vocab, int64_t ld, const int32_t *token_dev, int top,
                              float *logprob_dev, float *entropy_dev, int32_t *top_token_dev, float *top_logprob_dev, void *stream) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    if (dt != NNQ_F32 && dt != NNQ_BF16) return fail(ctx, NNQ_ERR_INVALID_ARG, "unknown dtype %d", (int)dt);
    if (rows < 0 || vocab < 1 || vocab > INT32_MAX / 2) return fail(ctx, NNQ_ERR_INVALID_ARG, "logits of %lld rows and %lld tokens", (long long)rows, (long long)vocab);
    if (ld < vocab) return fail(ctx, NNQ_ERR_SHAPE_MISMATCH, "rows of %lld logits lie %lld apart", (long long)vocab, (long long)ld);
    if (top < 0 || top > kLpTop || top > vocab) return fail(ctx, NNQ_ERR_UNSUPPORTED, "%d alternatives: at most %d and the vocabulary's size", top, kLpTop);
    if (rows == 0) return NNQ_OK;
    if (!logits_dev || (logprob_dev && !token_dev) || (top == 0 && !logprob_dev && !entropy_dev) || (top > 0 && !top_token_dev && !top_logprob_dev))
        return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor");
    if ((uintptr_t)logits_dev % (dt == NNQ_F32 ? 4 : 2)) return fail(ctx, NNQ_ERR_INVALID_ARG, "misaligned logits");
    nnq_status s = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice");
    if (s != NNQ_OK) return s;
    // CTAs of a row: as many as give every SM one, but no slices below 4096 elements
    int ctas = 1;
    while (ctas < 8 && rows * ctas < ctx->sm_count && vocab / (2 * ctas) >= 4096) ctas *= 2;
    const int slice = (int)(((vocab + ctas - 1) / ctas + 7) / 8 * 8);
    const int64_t most = 65535;   // rows of a launch
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        LogprobArgs a = {(const uint8_t *)logits_dev + r0 * ld * (dt == NNQ_F32 ? 4 : 2), token_dev ? token_dev + r0 : nullptr, logprob_dev ? logprob_dev + r0 : nullptr,
                         entropy_dev ? entropy_dev + r0 : nullptr, top_logprob_dev ? top_logprob_dev + r0 * top : nullptr, top_token_dev ? top_token_dev + r0 * top : nullptr,
                         ld, (int)vocab, top, slice, ctx->d_status};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas, (unsigned)std::min(most, rows - r0));
        cfg.blockDim = dim3(kLpThreads);
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim = {(unsigned)ctas, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        s = check_cuda(ctx, dt == NNQ_F32 ? cudaLaunchKernelEx(&cfg, logprobs_kernel<true>, a) : cudaLaunchKernelEx(&cfg, logprobs_kernel<false>, a), "log probabilities launch");
        if (s != NNQ_OK) return s;
        ctx->launches++;
    }
    return NNQ_OK;
}

}  // extern "C"
