// Log probabilities of given tokens under rows of logits, with the entropy of each row and its most probable tokens.
//
//   lse = m + ln sum e^(x - m);  log p(t) = x_t - lse;  H = -sum p ln p = ln l - T / l,  l = sum e^(x - m), T = sum e^(x - m) (x - m)
//
// One pass over a row keeps the running maximum m, l = sum 2^d and T = sum 2^d d with d = (x - m) log2 e, the difference formed first,
// so that logits of any size keep their digits (every term of T has the same sign; a new maximum scales l by f = 2^-delta and makes
// T f (T - delta l)). All of it is f32.
// A row is dealt to a cluster of CTAs where the rows are few, and every CTA's sums meet in the first one's shared memory, in order.
// The most probable tokens: the pass leaves the largest element of every group (four 16-byte vectors of a thread) in shared memory. The
// threads of each of 32 lanes have seen disjoint parts of the slice, so at least 32 elements are not below the least of these parts'
// maxima: the groups from there on (about a hundred) are ranked, and the `top` best are read again, element by element. Where one of these
// parts is all -inf (few tokens are allowed), all groups with anything above -inf are (64 rows of 151936 with 20 such tokens, 20 alternatives:
// 20 us as for other rows, 264 us by the search below). Where that
// meets more equal values than there is room for, or a NaN, the largest element below the one before is looked for `top` times. Order:
// larger value first, then the lower index.
// What bounds it: bf16 rows the issue of instructions (74 % of the slots used, special functions 57 %, logic pipe and FMA pipe 47 %: maxima, differences,
// clamps and the entropy's sums beside the exponentials); some hundred rows the search, which stands behind the reading in a CTA of its own SM;
// single rows the way through the cluster. Measured: 2000 bf16 rows of 128259 with one alternative 123 us (4.2 TB/s), 129 f32 rows of
// 151936 with 20 of them from memory 25 us (3.1 TB/s), one row 11 us.
// The reference turns logits into probabilities on the host (crates/nn-core/src/layers/generation/autoregressive_sampling.rs:14-21 and
// the samplers beside it).
#include <algorithm>
#include <cfloat>

#include "kv_cache.cuh"
#include "tcgen05.cuh"

namespace nnq {

constexpr int kLpRoom = 1024, kLpTop = 32, kLpUnroll = 4;
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

struct Stats {   // maximum (-inf: no element), sum of 2^d and of 2^d d
    float c, l, t;
};
__device__ __forceinline__ float finite_ref(float c) { return c == -INFINITY ? 0.0f : c; }
__device__ __forceinline__ float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float c = fmaxf(a.c, b.c), r = finite_ref(c);
    const float da = (finite_ref(a.c) - r) * kLpLog2E, db = (finite_ref(b.c) - r) * kLpLog2E;
    // (a side without elements has sums of zero; its reference does not matter)
    const float fa = a.l == 0.0f ? 0.0f : lp_ex2(da), fb = b.l == 0.0f ? 0.0f : lp_ex2(db);
    return {c, fmaf(a.l, fa, b.l * fb), (a.l == 0.0f ? 0.0f : fa * fmaf(fmaxf(da, -1e4f), a.l, a.t)) + (b.l == 0.0f ? 0.0f : fb * fmaf(fmaxf(db, -1e4f), b.l, b.t))};
}

// order of logits as unsigned numbers; NaN above everything
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0xFFFFFFFEu;   // (a key of all ones stands for none yet)
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);   // (-0 equals 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, int i) { return (uint64_t)order_bits(x) << 32 | (0xFFFFFFFFu - (uint32_t)i); }

template <bool F32>
__device__ __forceinline__ float logit(const void *x, int64_t i) {
    if constexpr (F32) return reinterpret_cast<const float *>(x)[i];
    else return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(x)[i]);
}

// A CTA's slice [lo, hi) of a row: elements up to the first 16-byte boundary, vectors, elements behind the last whole one.
template <bool F32, int kLpThreads>
struct Slice {
    static constexpr int V = F32 ? 4 : 8, SIZE = F32 ? 4 : 2;
    const void *row;
    int lo, hi, head, vecs;
    __device__ Slice(const void *row_, int lo_, int hi_) : row(row_), lo(lo_), hi(hi_) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row) + (uintptr_t)lo * SIZE;
        head = min(hi, lo + (int)((16 - (at & 15u)) % 16 / SIZE));
        vecs = (hi - head) / V;
    }
    __device__ const uint4 *vec() const { return reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(row) + (int64_t)head * SIZE); }
    __device__ int edges() const { return hi - lo - vecs * V; }                                         // elements outside the vectors
    __device__ int edge(int i) const { return i < head - lo ? lo + i : head + vecs * V + i - (head - lo); }
    __device__ int groups() const { return (vecs + kLpThreads * kLpUnroll - 1) / (kLpThreads * kLpUnroll); }   // of a thread
};

// f(value, index in the row) for all elements
template <bool F32, int kLpThreads, typename F>
__device__ __forceinline__ void each_logit(const Slice<F32, kLpThreads> &s, F f) {
    constexpr int V = Slice<F32, kLpThreads>::V;
    for (int i = threadIdx.x; i < s.edges(); i += kLpThreads) f(logit<F32>(s.row, s.edge(i)), s.edge(i));
    for (int u = threadIdx.x; u < s.vecs; u += kLpThreads)
        for (int e = 0; e < V; e++) f(logit<F32>(s.row, s.head + u * V + e), s.head + u * V + e);
}

template <bool F32, int kLpThreads>
__global__ void __launch_bounds__(kLpThreads, kLpThreads == 256 ? 4 : 2) logprobs_kernel(const LogprobArgs a) {
    extern __shared__ float group_max[];   // [groups of a thread][threads]
    constexpr int kLpWarps = kLpThreads / 32;
    __shared__ Stats warp_stats[kLpWarps], cta_stats;
    __shared__ float part_max[kLpWarps][32];
    __shared__ float bound_s;
    __shared__ uint32_t least_s;
    __shared__ int found, chosen;
    __shared__ uint64_t room[kLpRoom];
    __shared__ int pick[kLpRoom];
    __shared__ uint64_t best[kLpTop];
    __shared__ uint64_t red[kLpWarps];
    constexpr int V = Slice<F32, kLpThreads>::V;
    pdl_prologue();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = gridDim.x, me = blockIdx.x;
    const int64_t row = blockIdx.y;
    const void *x = reinterpret_cast<const uint8_t *>(a.x) + row * a.ld * Slice<F32, kLpThreads>::SIZE;
    const int lo = min(a.vocab, me * a.slice);
    const Slice<F32, kLpThreads> sl(x, lo, min(a.vocab, lo + a.slice));
    const int groups = sl.groups();
    const uint4 *vec = sl.vec();

    // ---- the pass
    float m = -INFINITY, ref = 0.0f;   // maximum; the same, or 0 before there is one
    float2 l = make_float2(0.0f, 0.0f), t = l;
    const float2 scale = make_float2(kLpLog2E, kLpLog2E);
    auto raise = [&](float top) {
        if (m != -INFINITY) {
            const float d = (m - top) * kLpLog2E, f = lp_ex2(d), dd = fmaxf(d, -1e4f);
            t = make_float2(f * fmaf(dd, l.x, t.x), f * fmaf(dd, l.y, t.y));
            l = make_float2(l.x * f, l.y * f);
        }
        m = ref = top;
    };
    auto add = [&](float2 v) {
        const float2 d = __fmul2_rn(__fadd2_rn(v, make_float2(-ref, -ref)), scale), e = make_float2(lp_ex2(d.x), lp_ex2(d.y));
        l = __fadd2_rn(l, e);
        t = __ffma2_rn(e, make_float2(fmaxf(d.x, -1e4f), fmaxf(d.y, -1e4f)), t);   // (0 times -inf would be NaN)
    };
    uint4 w[kLpUnroll], next[kLpUnroll];
    auto fetch = [&](int g, uint4 (&to)[kLpUnroll]) {
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) {
            const int u = (g * kLpUnroll + j) * kLpThreads + tid;
            const uint32_t none = F32 ? 0xFF800000u : 0xFF80FF80u;   // -inf
            to[j] = u < sl.vecs ? __ldg(vec + u) : make_uint4(none, none, none, none);
        }
    };
    fetch(0, next);
    for (int g = 0; g < groups; g++) {
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) w[j] = next[j];
        if (g + 1 < groups) fetch(g + 1, next);
        auto value = [&](int j, int i) {   // pair i of vector j
            const uint32_t q[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
            if constexpr (F32) return make_float2(__uint_as_float(q[2 * i]), __uint_as_float(q[2 * i + 1]));
            else return make_float2(__uint_as_float(q[i] << 16), __uint_as_float(q[i] & 0xFFFF0000u));
        };
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) top = fmaxf(top, fmaxf(value(j, i).x, value(j, i).y));
        if (a.top > 0) group_max[g * kLpThreads + tid] = top;
        if (top > m) raise(top);
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++)
#pragma unroll
            for (int i = 0; i < V / 2; i++) add(value(j, i));
    }
    const float mine = m;   // of the vectors alone
    for (int i = tid; i < sl.edges(); i += kLpThreads) {
        const float v = logit<F32>(x, sl.edge(i));
        if (v > m) raise(v);
        add(make_float2(v, -INFINITY));
    }
    Stats s = {m, l.x + l.y, t.x + t.y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.c, o), __shfl_xor_sync(0xFFFFFFFFu, s.l, o), __shfl_xor_sync(0xFFFFFFFFu, s.t, o)});
    if (lane == 0) warp_stats[warp] = s;
    if (tid == 0) {
        found = chosen = 0;
        least_s = 0xFFFFFFFFu;
    }
    if (tid < kLpTop) best[tid] = 0;   // below every key
    part_max[warp][lane] = mine;
    __syncthreads();
    if (warp == 0) {
        s = lane < kLpWarps ? warp_stats[lane] : Stats{-INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s = join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.c, o), __shfl_xor_sync(0xFFFFFFFFu, s.l, o), __shfl_xor_sync(0xFFFFFFFFu, s.t, o)});
        if (lane == 0) cta_stats = s;
    } else if (warp == 1) {
        float b = -INFINITY;   // maximum of the elements that the threads of this lane have seen
#pragma unroll
        for (int w = 0; w < kLpWarps; w++) b = fmaxf(b, part_max[w][lane]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) b = fminf(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
        if (lane == 0) bound_s = b;
    }
    __syncthreads();

    // ---- the slice's most probable tokens
    if (a.top > 0) {
        bool few = !(cta_stats.l != cta_stats.l);   // (a NaN hides from the groups' maxima)
        if (few) {
            // (a lane may have seen nothing but -inf, where few tokens are allowed: then every group with something above it)
            const float bound = fmaxf(bound_s, -FLT_MAX);
            const bool rest = bound_s == -INFINITY;
            for (int g = 0; g < groups; g++)
                if ((g * kLpUnroll * kLpThreads) + tid < sl.vecs && group_max[g * kLpThreads + tid] >= bound) {
                    const int at = atomicAdd(&found, 1);
                    if (at < kLpRoom) room[at] = order_key(group_max[g * kLpThreads + tid], g * kLpThreads + tid);
                }
            __syncthreads();
            const int n = found;
            few = n <= kLpRoom;
            if (few) {
                // the `top` best groups and their equals: the elements below the least of them are not among the best
                for (int i = tid; i < n; i += kLpThreads) {
                    const uint32_t k = (uint32_t)(room[i] >> 32);
                    int above = 0;
                    for (int j = 0; j < n; j++) above += (uint32_t)(room[j] >> 32) > k;
                    if (above < a.top) {
                        atomicMin(&least_s, k);
                        pick[atomicAdd(&chosen, 1)] = (int)(0xFFFFFFFFu - (uint32_t)room[i]);
                    }
                }
                __syncthreads();
                const uint32_t least = n >= a.top ? least_s : 0u;   // (with fewer groups than that everything counts)
                const int groups_read = chosen, per = kLpUnroll * V;
                if (tid == 0) found = 0;
                __syncthreads();
                auto offer = [&](int idx, bool masked) {
                    const float v = logit<F32>(x, idx);
                    if (order_bits(v) >= least && (v == -INFINITY) == masked) {
                        const int at = atomicAdd(&found, 1);
                        if (at < kLpRoom) room[at] = order_key(v, idx);
                    }
                };
#pragma unroll 2
                for (int i = tid; i < groups_read * per; i += kLpThreads) {
                    const int q = pick[i / per], e = i % per, u = (q / kLpThreads * kLpUnroll + e / V) * kLpThreads + q % kLpThreads;
                    if (u < sl.vecs) offer(sl.head + u * V + e % V, false);
                }
                for (int i = tid; i < sl.edges(); i += kLpThreads) offer(sl.edge(i), false);
                // fewer than `top` above -inf: the first ones at -inf, which are among the first `top` of the slice
                if (rest && sl.lo + tid < min(sl.hi, sl.lo + a.top)) offer(sl.lo + tid, true);
                __syncthreads();
                few = found <= kLpRoom;
            }
        }
        if (few) {
            const int n = found;
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
                each_logit(sl, [&](float v, int j) {
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

    // ---- the row
    if (ctas > 1) cluster_sync();
    if (me == 0) {
        const uint32_t stats_at = smem_u32(&cta_stats), best_at = smem_u32(best);
        s = lane < ctas ? cta_stats : Stats{-INFINITY, 0.0f, 0.0f};
        if (lane > 0 && lane < ctas) {
            const uint32_t p = cluster_addr(stats_at, lane);
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s.c) : "r"(p) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s.l) : "r"(p + 4) : "memory");
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(s.t) : "r"(p + 8) : "memory");
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s = join(s, {__shfl_xor_sync(0xFFFFFFFFu, s.c, o), __shfl_xor_sync(0xFFFFFFFFu, s.l, o), __shfl_xor_sync(0xFFFFFFFFu, s.t, o)});
        s = {__shfl_sync(0xFFFFFFFFu, s.c, 0), __shfl_sync(0xFFFFFFFFu, s.l, 0), __shfl_sync(0xFFFFFFFFu, s.t, 0)};
        const float log_l = log2f(s.l), r = finite_ref(s.c);
        const bool none = s.c == -INFINITY && s.l == 0.0f;   // no token has any probability
        auto log_prob = [&](float v) { return none ? v : fmaf(-log_l, kLpLn2, v - r); };
        if (tid == 0) {
            const int tok = a.token ? a.token[row] : -1;
            if (tok >= a.vocab) atomicExch(a.status, kStatusIndex);
            if (a.logprob) a.logprob[row] = tok < 0 ? 0.0f : tok >= a.vocab ? __int_as_float(0x7FFFFFFF) : log_prob(logit<F32>(x, tok));
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
    // CTAs of a row: as many as there are SMs for, but no slices below 4096 elements. us with as many / up to twice as many, rows from
    // memory: 30 bf16 rows of 151936 13.2 / 16.1, 140 bf16 rows of 32000 9.9 / 12.5, 19 f32 rows of 151936 13.9 / 15.9, but 80 of them 23.7 / 22.0;
    // rows in the L2 cache: 129 f32 rows 18.8 / 23.2. One row of 151936 by one CTA 15.8, by eight 10.9.
    int ctas = 1;
    while (ctas < 8 && rows * 2 * ctas <= ctx->sm_count && vocab / (2 * ctas) >= 4096) ctas *= 2;
    // threads: four CTAs of 256 on an SM are in different phases of their rows where there are many; a row's few parts are read faster by
    // 512 (us, 256 / 512: 2000 bf16 rows of 128259 123 / 145, 129 f32 rows of 151936 26.7 / 22.7 with two CTAs a row)
    const int threads = rows >= 2 * ctx->sm_count ? 256 : 512;
    auto kernel = dt == NNQ_F32 ? (threads == 256 ? logprobs_kernel<true, 256> : logprobs_kernel<true, 512>) : (threads == 256 ? logprobs_kernel<false, 256> : logprobs_kernel<false, 512>);
    const int slice = (int)(((vocab + ctas - 1) / ctas + 7) / 8 * 8), v = dt == NNQ_F32 ? 4 : 8;
    // shared memory: a float per thread and group of its vectors (vocabularies of many millions take more than there is)
    const int64_t groups = (slice / v + threads * kLpUnroll - 1) / (threads * kLpUnroll);
    const size_t smem = top > 0 ? (size_t)groups * threads * 4 : 0;
    constexpr size_t most_smem = 160 * 1024;
    static std::atomic<uint64_t> allowed[4];   // (one size for all calls: others of other threads may lie between asking and launching)
    if (smem > most_smem) return fail(ctx, NNQ_ERR_UNSUPPORTED, "alternatives among %lld tokens", (long long)vocab);
    if (smem > 16 * 1024 && (s = allow_smem(ctx, kernel, most_smem, allowed[(dt == NNQ_F32) * 2 + (threads == 256)])) != NNQ_OK) return s;
    const int64_t most = 65535;   // rows of a launch
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        LogprobArgs a = {(const uint8_t *)logits_dev + r0 * ld * (dt == NNQ_F32 ? 4 : 2), token_dev ? token_dev + r0 : nullptr, logprob_dev ? logprob_dev + r0 : nullptr,
                         entropy_dev ? entropy_dev + r0 : nullptr, top_logprob_dev ? top_logprob_dev + r0 * top : nullptr, top_token_dev ? top_token_dev + r0 * top : nullptr,
                         ld, (int)vocab, top, slice, ctx->d_status};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas, (unsigned)std::min(most, rows - r0));
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = (cudaStream_t)stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim = {(unsigned)ctas, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        s = check_cuda(ctx, cudaLaunchKernelEx(&cfg, kernel, a), "log probabilities launch");
        if (s != NNQ_OK) return s;
        ctx->launches++;
    }
    return NNQ_OK;
}

}  // extern "C"
