// Attention over the paged 8-bit cache (kv_cache.cuh) for few query vectors per key / value head: a decode step, draft tokens, and
// every size that the prompt kernel does not take.
//
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the positions that a row sees.
//
// What bounds it is the reading of the cache, 2 dim bytes per key and head once for all query heads of the group. The codes go from
// global memory to the operand registers of mma.sync (m16n8k16, f16) without a stop in shared memory:
//   scores   S^T [16 keys x 8 vectors] = K [16 x dim] Q^T: lane (g, t) of a warp reads 16 bytes of keys g and g + 8 at a time; which
//            dimension stands at which place of k is free as long as the queries agree.
//   values   O^T [dim x 8 vectors] += V^T [dim x 16 keys] P^T: lane (g, t) reads dim / 8 neighbouring bytes of the four keys whose
//            weights it holds, and a byte permutation puts two keys of a dimension side by side; the weights are turned by movmatrix.
// Keys as the 16 rows waste none of the tensor core on missing query vectors. Codes are exact in f16; a query vector enters under a
// power of two (one f16 term for bf16 queries, which is exact; two for f32), weights as two f16 terms (22 bits), so that scores, sums
// and outputs are of f32 accuracy. A block's scales stay outside: the key's multiplies the scores, the value's goes into the exponent
// of the weight, w = 2^(s - mv + e_v), which has a reference mv of its own beside the maximum m of the sum (l = sum 2^(s - m)): weights
// stay between 0 and 2^8 whatever the scales are. Both references move only when a score passes them by 8, so most steps have one vote
// in place of the maxima's exchange.
//
// Work is dealt in steps of 16 keys: all steps of all (request, head, vectors) items in one row, cut into equal parts, one for each
// CTA, whatever the requests' lengths are. An item inside one part is written directly; of an item that is cut every part leaves a
// record (m, mv, l, O), and kv_join_kernel joins them in their order.
#include <algorithm>

#include "kv_attn.cuh"

namespace nnq {

constexpr int kKvWarps = 8, kKvCols = 8, kKvStep = 16;
constexpr int kKvMinSteps = 2 * kKvWarps;   // of a CTA's part
constexpr int kFew = 32;   // see nnq_kv_attention
constexpr int kNothing = INT32_MIN;   // in place of a block: no key of the step is seen
constexpr float kKvLog2E = 1.4426950408889634f;
constexpr float kKvSlack = 8.0f;   // a score may pass the reference by this power of two: weights up to 256 in f16

// records: [part][began before, begins here][column]: m, mv, l, unused, then O[dim]
__host__ __device__ inline int kv_record_floats(int dim) { return 4 + dim; }

struct KvPlan {
    int64_t total, chunk;   // steps in all, steps of a part
    int64_t r;              // request of the first step of this part
    int64_t off;            // and the step's number within the request
};

// Steps of an item of the request (the same for all its heads and vectors), and its items of one head.
__device__ __forceinline__ int64_t item_steps(const KvAttn &a, const KvRequest &q) {
    if (q.rows == 0 || q.rows * a.group > a.few) return 0;
    const int64_t lo = row_first(a, max(row_pos(q, 0), (int64_t)0)), steps = ((q.length + kKvStep - 1) / kKvStep) - lo / kKvStep;
    return max(steps, (int64_t)1);
}
__device__ __forceinline__ int64_t item_count(const KvAttn &a, const KvRequest &q) { return ((int64_t)q.rows * a.group + kKvCols - 1) / kKvCols; }

__device__ __forceinline__ int64_t block_scan(int64_t &v, int64_t *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    long long x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long b = __shfl_up_sync(0xFFFFFFFFu, x, off);
        if (lane >= off) x += b;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < nw; w++) {
        if (w == warp) before = all;
        all += warp_sums[w];
    }
    v = before + x - v;
    return all;
}

// Every CTA sums the steps of all requests (twice, where there are more requests than threads) and finds where its part begins.
__device__ KvPlan kv_plan(const KvAttn &a, int parts) {
    __shared__ int64_t warp_sums[32], found[2];
    const int nt = blockDim.x, tid = threadIdx.x;
    auto steps_of = [&](int64_t r) -> int64_t {
        if (r >= a.requests) return 0;
        const KvRequest q = kv_request(a, r);
        return item_steps(a, q) * item_count(a, q) * a.kv_heads;
    };
    KvPlan p;
    p.total = 0;
    for (int64_t r0 = 0; r0 < a.requests; r0 += nt) {
        int64_t v = steps_of(r0 + tid);
        p.total += block_scan(v, warp_sums);
    }
    p.chunk = max((p.total + parts - 1) / parts, (int64_t)kKvMinSteps);
    const int64_t begin = p.chunk * blockIdx.x;
    p.r = p.off = 0;
    if (begin >= p.total) return p;
    int64_t done = 0;
    for (int64_t r0 = 0; r0 < a.requests && done <= begin; r0 += nt) {
        const int64_t mine = steps_of(r0 + tid);
        int64_t v = mine;
        const int64_t all = block_scan(v, warp_sums);
        if (begin >= done + v && begin < done + v + mine) {
            found[0] = r0 + tid;
            found[1] = begin - done - v;
        }
        done += all;
    }
    __syncthreads();
    p.r = found[0];
    p.off = found[1];
    return p;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Codes of 16 keys as a lane holds them, and the scales of their block.
template <int D>
struct KvStepData {
    uint4 k[2][D / 64];
    uint2 v[4][D / 64];
    int ke, ve;
    bool there;   // false: the table has no such block
};

template <int D>
__device__ __forceinline__ void load_step(const KvAttn &a, int blk, int64_t key0, int head, int lane, KvStepData<D> &s) {
    const int g = lane >> 2, t = lane & 3;
    s.there = blk >= 0 && blk < a.blocks;
    if (!s.there) return;
    const int64_t bh = (int64_t)blk * a.kv_heads + head;
    const int64_t at = ((bh << a.shift) + (key0 & ((1 << a.shift) - 1))) * D;
    const uint8_t *kp = a.k + at + g * D + t * 16, *vp = a.v + at + 2 * t * D + g * (D / 8);
#pragma unroll
    for (int c = 0; c < D / 64; c++) {
        s.k[0][c] = __ldg(reinterpret_cast<const uint4 *>(kp + c * 64));
        s.k[1][c] = __ldg(reinterpret_cast<const uint4 *>(kp + 8 * D + c * 64));
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint8_t *p = vp + ((i & 1) + (i >> 1) * 8) * D;
        if constexpr (D % 128 == 0) {
#pragma unroll
            for (int c = 0; c < D / 128; c++) {
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p) + c);
                s.v[i][2 * c] = make_uint2(x.x, x.y);
                s.v[i][2 * c + 1] = make_uint2(x.z, x.w);
            }
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; c++) s.v[i][c] = __ldg(reinterpret_cast<const uint2 *>(p) + c);
        }
    }
    s.ke = a.k_exp[bh];
    s.ve = a.v_exp[bh];
}

template <int FMT, int D, int QT>
__global__ void __launch_bounds__(kKvWarps * 32, D <= 128 ? 2 : 1) kv_attn_kernel(const KvAttn a, float *records) {
    extern __shared__ __align__(16) float sm[];   // a record of every warp and column
    typedef CodePairs<FMT> Codes;
    constexpr int REC = 4 + D;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_prologue();
    const KvPlan plan = kv_plan(a, gridDim.x);
    int64_t at = plan.chunk * blockIdx.x;
    const int64_t end = min(plan.total, at + plan.chunk);
    int64_t r = plan.r, off = plan.off;
    while (at < end) {
        // ---- the next request with steps left, the item and the part of it that is this CTA's
        const KvRequest rq = kv_request(a, r);
        const int64_t spi = item_steps(a, rq), cols = item_count(a, rq), of_request = spi * cols * a.kv_heads;
        if (off >= of_request) {
            off = 0;
            r++;
            continue;
        }
        const int64_t item = off / spi, s0 = off - item * spi, s1 = min(spi, s0 + end - at);
        const int head = (int)(item / cols), vec0 = (int)(item - (int64_t)head * cols) * kKvCols, vecs = min(kKvCols, rq.rows * a.group - vec0);
        const int64_t lo_all = row_first(a, max(row_pos(rq, 0), (int64_t)0)) / kKvStep * kKvStep;   // the item's step 0 begins here

        // ---- queries: lane (g, t) has vector g's dimensions c * 64 + t * 16 .. + 15 of every c, as the scores' second operand
        uint32_t qh[D / 16][2], ql[QT == 2 ? D / 16 : 1][2];
        float q_un = 1.0f;
        {
            float x[D / 64][16];
            const int v = vec0 + g, row = v / a.group, qhead = head * a.group + v % a.group;
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < D / 64; c++)
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    float y[8] = {};
                    const int64_t from = (int64_t)(rq.row0 + row) * a.q_ld + (int64_t)qhead * D + c * 64 + t * 16 + i;
                    if (g < vecs) {
                        if constexpr (QT == 2) {
                            const float4 u = __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + from));
                            const float4 w = __ldg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + from) + 1);
                            y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w; y[4] = w.x; y[5] = w.y; y[6] = w.z; y[7] = w.w;
                        } else {
                            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(a.q) + from));
                            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                y[2 * e] = __uint_as_float(w[e] << 16);
                                y[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[c][i + e] = y[e];
                        top = max(top, __float_as_uint(y[e]) & 0x7FFFFFFFu);
                    }
                }
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const float sc = kv_top_scale(top);
            q_un = kv_top_unscale(top);
#pragma unroll
            for (int c = 0; c < D / 64; c++)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t hi, lo;
                        kv_split(x[c][4 * j + 2 * e] * sc, x[c][4 * j + 2 * e + 1] * sc, hi, lo);
                        qh[4 * c + j][e] = hi;
                        if constexpr (QT == 2) ql[4 * c + j][e] = lo;
                    }
        }
        // this lane's two columns of the scores are vectors 2t and 2t + 1: factor, position and first position seen
        float fac[2];
        int64_t pos[2], low[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            fac[j] = a.scale * kKvLog2E * Codes::unscale * __shfl_sync(0xFFFFFFFFu, q_un, (2 * t + j) * 4);
            const int v = min(2 * t + j, vecs - 1);
            pos[j] = row_pos(rq, (vec0 + v) / a.group);
            low[j] = row_first(a, pos[j]);
        }
        // positions that every vector sees, and that some vector sees
        const int64_t first_pos = row_pos(rq, vec0 / a.group), last_pos = row_pos(rq, (vec0 + vecs - 1) / a.group);
        const int64_t lo_some = row_first(a, max(first_pos, (int64_t)0)), lo_every = row_first(a, max(last_pos, (int64_t)0));

        float acc[D / 16][4];
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = 0.0f;
        float m[2] = {0.0f, 0.0f}, mv[2] = {0.0f, 0.0f}, l[2] = {0.0f, 0.0f};
        float thr[2] = {-INFINITY, -INFINITY}, thv[2] = {-INFINITY, -INFINITY};   // references and what makes them move

        const int32_t *table = a.table + r * a.table_ld;
        auto key_of = [&](int64_t s) { return lo_all + s * kKvStep; };
        auto wanted = [&](int64_t s) { return s < s1 && key_of(s) <= last_pos && key_of(s) + kKvStep > lo_some; };
        auto block_of = [&](int64_t s) { return wanted(s) ? table[key_of(s) >> a.shift] : kNothing; };
        KvStepData<D> now, next;
        int blk = block_of(s0 + warp), blk1 = block_of(s0 + warp + kKvWarps);
        load_step<D>(a, blk, key_of(s0 + warp), head, lane, now);
        for (int64_t s = s0 + warp; s < s1; s += kKvWarps) {
            const int blk2 = block_of(s + 2 * kKvWarps);
            load_step<D>(a, blk1, key_of(s + kKvWarps), head, lane, next);
            if (now.there) {
                // ---- scores
                // (sums of 32 dimensions each: the tensor core cuts off what its f32 sums cannot hold, and long chains of that lean one way)
                float part[D / 32][4];
#pragma unroll
                for (int c = 0; c < D / 64; c++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) part[2 * c + (e >> 2)][e & 3] = 0.0f;
                    const uint32_t r0[4] = {now.k[0][c].x, now.k[0][c].y, now.k[0][c].z, now.k[0][c].w}, r1[4] = {now.k[1][c].x, now.k[1][c].y, now.k[1][c].z, now.k[1][c].w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t u = Codes::word(r0[j]), w = Codes::word(r1[j]);
                        const uint32_t x[4] = {Codes::low(u), Codes::low(w), Codes::high(u), Codes::high(w)};
                        if constexpr (QT == 2) mma_f16(part[2 * c + (j >> 1)], x, ql[4 * c + j][0], ql[4 * c + j][1]);
                        mma_f16(part[2 * c + (j >> 1)], x, qh[4 * c + j][0], qh[4 * c + j][1]);
                    }
                }
                float sc[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[i] = part[0][i] + part[1][i];
#pragma unroll
                    for (int c = 1; c < D / 64; c++) sc[i] += part[2 * c][i] + part[2 * c + 1][i];
                }
                const float kf = pow2_byte(now.ke), ve = (float)(now.ve - 127);
                const int64_t key0 = key_of(s);
#pragma unroll
                for (int i = 0; i < 4; i++) sc[i] = sc[i] * kf * fac[i & 1];
                if (key0 + kKvStep - 1 > first_pos || key0 < lo_every) {   // (the same for the whole warp)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int64_t j = key0 + g + (i >> 1) * 8;
                        if (j > pos[i & 1] || j < low[i & 1]) sc[i] = -INFINITY;
                    }
                }
                // ---- references
                const float big0 = fmaxf(sc[0], sc[2]), big1 = fmaxf(sc[1], sc[3]);
                if (__any_sync(0xFFFFFFFFu, big0 > thr[0] || big1 > thr[1] || big0 + ve > thv[0] || big1 + ve > thv[1])) {
                    float b[2] = {big0, big1};
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        b[0] = fmaxf(b[0], __shfl_xor_sync(0xFFFFFFFFu, b[0], o));
                        b[1] = fmaxf(b[1], __shfl_xor_sync(0xFFFFFFFFu, b[1], o));
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (b[j] == -INFINITY) continue;   // nothing seen yet or here
                        const bool none = thr[j] == -INFINITY;   // a first reference: the sums are zero
                        const float mn = none ? b[j] : fmaxf(m[j], b[j]), vn = none ? b[j] + ve : fmaxf(mv[j], b[j] + ve);
                        const float f = none ? 1.0f : exp2f(mv[j] - vn);
                        l[j] *= none ? 1.0f : exp2f(m[j] - mn);
#pragma unroll
                        for (int i = 0; i < D / 16; i++) {
                            acc[i][j] *= f;
                            acc[i][j + 2] *= f;
                        }
                        m[j] = mn;
                        mv[j] = vn;
                        thr[j] = mn + kKvSlack;
                        thv[j] = vn + kKvSlack;
                    }
                }
                // ---- weights
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    l[i & 1] += kv_ex2(sc[i] - m[i & 1]);
                    w[i] = kv_ex2(sc[i] + (ve - mv[i & 1]));
                }
                uint32_t h0, l0, h1, l1;
                kv_split(w[0], w[1], h0, l0);
                kv_split(w[2], w[3], h1, l1);
                h0 = turn8x8(h0);
                h1 = turn8x8(h1);
                l0 = turn8x8(l0);
                l1 = turn8x8(l1);
                // ---- values: 8 dimensions (four MMA rows each of g and g + 8) per two words of four keys
#pragma unroll
                for (int c = 0; c < D / 64; c++)
#pragma unroll
                    for (int hw = 0; hw < 2; hw++) {
                        const uint32_t k0 = Codes::word(hw ? now.v[0][c].y : now.v[0][c].x), k1 = Codes::word(hw ? now.v[1][c].y : now.v[1][c].x);
                        const uint32_t k2 = Codes::word(hw ? now.v[2][c].y : now.v[2][c].x), k3 = Codes::word(hw ? now.v[3][c].y : now.v[3][c].x);
                        const uint32_t a01 = __byte_perm(k0, k1, 0x5140), b01 = __byte_perm(k0, k1, 0x7362), a23 = __byte_perm(k2, k3, 0x5140), b23 = __byte_perm(k2, k3, 0x7362);
                        const uint32_t x0[4] = {Codes::low(a01), Codes::high(a01), Codes::low(a23), Codes::high(a23)};
                        const uint32_t x1[4] = {Codes::low(b01), Codes::high(b01), Codes::low(b23), Codes::high(b23)};
                        mma_f16(acc[4 * c + 2 * hw], x0, l0, l1);
                        mma_f16(acc[4 * c + 2 * hw + 1], x1, l0, l1);
                        mma_f16(acc[4 * c + 2 * hw], x0, h0, h1);
                        mma_f16(acc[4 * c + 2 * hw + 1], x1, h0, h1);
                    }
            } else if (blk != kNothing && lane == 0) {
                atomicExch(a.status, kStatusIndex);
            }
            now = next;
            blk = blk1;
            blk1 = blk2;
        }

        // ---- the warps' sums in shared memory: a record per warp and column (m = -inf: nothing seen)
        __syncthreads();
        {
            float *mine = sm + warp * kKvCols * REC;
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xFFFFFFFFu, l[j], o);
                float *rec = mine + (2 * t + j) * REC;
                if (g == 0) {
                    rec[0] = thr[j] > -INFINITY ? m[j] : (l[j] == 0.0f ? -INFINITY : l[j]);   // (scores that are all NaN move no reference)
                    rec[1] = mv[j];
                    rec[2] = l[j];
                }
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    rec[4 + g * (D / 8) + 2 * i] = acc[i][j];
                    rec[4 + g * (D / 8) + 2 * i + 1] = acc[i][j + 2];
                }
            }
        }
        __syncthreads();
        const bool whole = s0 == 0 && s1 == spi;
        for (int u = tid; u < vecs * D; u += kKvWarps * 32) {
            const int col = u / D, d = u - col * D;
            float mm = -INFINITY, mvv = -INFINITY;
#pragma unroll
            for (int w = 0; w < kKvWarps; w++) {
                const float *rec = sm + (w * kKvCols + col) * REC;
                if (rec[0] == -INFINITY) continue;
                mm = fmaxf(mm, rec[0]);
                mvv = fmaxf(mvv, rec[1]);
                if (rec[0] != rec[0]) mm = mvv = rec[0];
            }
            float ll = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < kKvWarps; w++) {
                const float *rec = sm + (w * kKvCols + col) * REC;
                if (rec[0] == -INFINITY) continue;
                ll += rec[2] * exp2f(rec[0] - mm);
                o += rec[4 + d] * exp2f(rec[1] - mvv);
            }
            if (whole) {
                const int v = vec0 + col;
                const int64_t to = (int64_t)(rq.row0 + v / a.group) * a.y_ld + (int64_t)(head * a.group + v % a.group) * D + d;
                // (the values' factor of e4m3 codes; exponents of both references are far inside the range)
                const float y = mm == -INFINITY ? 0.0f : o * (exp2f(mvv - mm) * Codes::unscale) / ll;
                if (a.y_dt == NNQ_F32) reinterpret_cast<float *>(a.y)[to] = y;
                else reinterpret_cast<__nv_bfloat16 *>(a.y)[to] = __float2bfloat16_rn(y);
            } else {
                float *rec = records + (((int64_t)blockIdx.x * 2 + (s0 == 0 ? 1 : 0)) * kKvCols + col) * REC;
                rec[4 + d] = o;
                if (d == 0) {
                    rec[0] = mm;
                    rec[1] = mvv;
                    rec[2] = ll;
                }
            }
        }
        at += s1 - s0;
        off += s1 - s0;
    }
}

// Joins the records of the items that were cut: CTA (part, column) does so where the item at the part's beginning began before it and
// ends in it.
template <int FMT>
__global__ void __launch_bounds__(256) kv_join_kernel(const KvAttn a, const float *records) {
    pdl_prologue();
    const KvPlan plan = kv_plan(a, gridDim.x);
    const int64_t at = plan.chunk * blockIdx.x;
    if (at >= plan.total) return;
    const KvRequest rq = kv_request(a, plan.r);
    const int64_t spi = item_steps(a, rq), cols = item_count(a, rq), item = plan.off / spi, s0 = plan.off - item * spi;
    if (s0 == 0 || spi - s0 > plan.chunk) return;   // begins here, or reaches beyond this part
    const int head = (int)(item / cols), vec0 = (int)(item - (int64_t)head * cols) * kKvCols, vecs = min(kKvCols, rq.rows * a.group - vec0);
    const int col = blockIdx.y;
    if (col >= vecs) return;
    const int64_t first = (at - s0) / plan.chunk;   // the part that the item begins in
    const int rec_floats = kv_record_floats(a.dim), d = threadIdx.x;
    auto record = [&](int64_t p) { return records + ((p * 2 + (p == first ? 1 : 0)) * kKvCols + col) * rec_floats; };
    float mm = -INFINITY, mvv = -INFINITY;
    for (int64_t p = first; p <= blockIdx.x; p++) {
        const float *rec = record(p);
        if (rec[0] == -INFINITY) continue;
        mm = fmaxf(mm, rec[0]);
        mvv = fmaxf(mvv, rec[1]);
        if (rec[0] != rec[0]) mm = mvv = rec[0];
    }
    if (d >= a.dim) return;
    float ll = 0.0f, o = 0.0f;
    for (int64_t p = first; p <= blockIdx.x; p++) {
        const float *rec = record(p);
        if (rec[0] == -INFINITY) continue;
        ll += rec[2] * exp2f(rec[0] - mm);
        o += rec[4 + d] * exp2f(rec[1] - mvv);
    }
    const int v = vec0 + col;
    const int64_t to = (int64_t)(rq.row0 + v / a.group) * a.y_ld + (int64_t)(head * a.group + v % a.group) * a.dim + d;
    const float y = mm == -INFINITY ? 0.0f : o * (exp2f(mvv - mm) * CodePairs<FMT>::unscale) / ll;
    if (a.y_dt == NNQ_F32) reinterpret_cast<float *>(a.y)[to] = y;
    else reinterpret_cast<__nv_bfloat16 *>(a.y)[to] = __float2bfloat16_rn(y);
}

static int kv_parts(nnq_ctx *ctx, int dim) { return (dim <= 128 ? 2 : 1) * ctx->sm_count; }

template <int FMT, int D, int QT>
static nnq_status launch_kv_attn(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    const size_t smem = (size_t)kKvWarps * kKvCols * kv_record_floats(D) * 4;
    nnq_status s = check_cuda(ctx, cudaFuncSetAttribute(kv_attn_kernel<FMT, D, QT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "attention shared memory");
    if (s != NNQ_OK) return s;
    const int parts = kv_parts(ctx, D);
    launch_pdl_smem(kv_attn_kernel<FMT, D, QT>, dim3(parts), dim3(kKvWarps * 32), smem, st, a, records);
    launch_pdl(kv_join_kernel<FMT>, dim3(parts, kKvCols), dim3(256), st, a, records);
    ctx->launches += 2;
    return check_cuda(ctx, cudaGetLastError(), "cache attention launch");
}

template <int FMT, int D>
static nnq_status launch_kv_attn(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    return a.q_dt == NNQ_F32 ? launch_kv_attn<FMT, D, 2>(ctx, a, records, st) : launch_kv_attn<FMT, D, 1>(ctx, a, records, st);
}

template <int FMT>
static nnq_status launch_kv_attn(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    switch (a.dim) {
        case 64: return launch_kv_attn<FMT, 64>(ctx, a, records, st);
        case 128: return launch_kv_attn<FMT, 128>(ctx, a, records, st);
        case 192: return launch_kv_attn<FMT, 192>(ctx, a, records, st);
        default: return launch_kv_attn<FMT, 256>(ctx, a, records, st);
    }
}

static nnq_status check_batch(nnq_ctx *ctx, const nnq_kv_cache *c, const nnq_kv_batch *b, int heads) {
    nnq_status s = check_kv_cache(ctx, c);
    if (s != NNQ_OK) return s;
    if (!b) return fail(ctx, NNQ_ERR_INVALID_ARG, "batch is NULL");
    if (heads < 1 || heads % c->kv_heads) return fail(ctx, NNQ_ERR_SHAPE_MISMATCH, "%d query heads over %d key / value heads", heads, c->kv_heads);
    if (b->requests < 1 || b->rows < 0 || b->table_ld < 1 || b->max_rows < 1) return fail(ctx, NNQ_ERR_INVALID_ARG, "bad sizes of a batch");
    if (b->requests > INT32_MAX / 2 || b->rows > INT32_MAX / heads || b->table_ld > INT32_MAX) return fail(ctx, NNQ_ERR_UNSUPPORTED, "a batch of %lld requests and %lld rows", (long long)b->requests, (long long)b->rows);
    return NNQ_OK;
}

}  // namespace nnq

using namespace nnq;

extern "C" {

nnq_status nnq_kv_attention_workspace(nnq_ctx *ctx, const nnq_kv_cache *c, const nnq_kv_batch *b, int heads, size_t *bytes) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    if (!bytes) return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL result");
    nnq_status s = check_batch(ctx, c, b, heads);
    if (s != NNQ_OK) return s;
    *bytes = std::max((size_t)kv_parts(ctx, c->dim) * 2 * kKvCols * kv_record_floats(c->dim) * 4, kv_attn_tc_workspace(ctx, c->dim));
    return NNQ_OK;
}

nnq_status nnq_kv_attention(nnq_ctx *ctx, const nnq_kv_cache *c, const nnq_kv_batch *b, const void *q_dev, nnq_dtype q_dt, int64_t q_ld, int heads,
                            float scale, int window, void *y_dev, nnq_dtype y_dt, int64_t y_ld, void *workspace, size_t workspace_bytes, void *stream) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    nnq_status s = check_batch(ctx, c, b, heads);
    if (s != NNQ_OK) return s;
    if ((q_dt != NNQ_F32 && q_dt != NNQ_BF16) || (y_dt != NNQ_F32 && y_dt != NNQ_BF16)) return fail(ctx, NNQ_ERR_INVALID_ARG, "unknown dtype");
    if (window < 0) return fail(ctx, NNQ_ERR_INVALID_ARG, "a window of %d", window);
    if (!(scale > 0.0f && scale < 3e38f)) return fail(ctx, NNQ_ERR_VALUE_OUT_OF_RANGE, "the scale of the scores must be positive and finite");
    if (b->rows == 0) return NNQ_OK;
    if (!b->length || !b->row_start || !b->table || !q_dev || !y_dev) return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor");
    const int64_t width = (int64_t)heads * c->dim;
    if (q_ld < width || y_ld < width) return fail(ctx, NNQ_ERR_SHAPE_MISMATCH, "rows of queries and outputs must be %lld wide or further apart", (long long)width);
    if (!rows_aligned(q_dev, q_ld, q_dt) || !rows_aligned(y_dev, y_ld, y_dt)) return fail(ctx, NNQ_ERR_INVALID_ARG, "rows of queries and outputs must start at multiples of 16 bytes");
    size_t need = 0;
    if ((s = nnq_kv_attention_workspace(ctx, c, b, heads, &need)) != NNQ_OK) return s;
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u))
        return fail(ctx, NNQ_ERR_INVALID_ARG, "the workspace must be %zu bytes, 16-byte aligned (got %zu)", need, workspace ? workspace_bytes : (size_t)0);
    if ((s = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice")) != NNQ_OK) return s;
    KvAttn a = {(const uint8_t *)c->k, (const uint8_t *)c->v, c->k_exp, c->v_exp, b->length, b->row_start, b->table, q_dev, y_dev, c->blocks, b->table_ld, b->requests, q_ld, y_ld, b->rows,
                      c->kv_heads, heads / c->kv_heads, c->dim, log2_of(c->block), window, (int)q_dt, (int)y_dt, INT32_MAX, scale, ctx->d_status};
    // Requests of more than kFew query vectors per key / value head go to the tensor-core kernel where there can be any; the rest of the
    // batch, down to single tokens beside a prompt, to this file's.
    if (kv_attn_tc_supported(a) && b->max_rows > kFew / a.group) {
        a.few = b->requests == 1 ? 0 : kFew;   // (a request alone is a prompt)
        if ((s = launch_kv_attn_tc(ctx, a, c->format, (float *)workspace, (cudaStream_t)stream)) != NNQ_OK || a.few == 0) return s;
    }
    return c->format == NNQ_KV_INT8 ? launch_kv_attn<NNQ_KV_INT8>(ctx, a, (float *)workspace, (cudaStream_t)stream)
                                    : launch_kv_attn<NNQ_KV_E4M3>(ctx, a, (float *)workspace, (cudaStream_t)stream);
}

}  // extern "C"
