// Attention over the paged 8-bit cache (kv_cache.cuh) for few query vectors per key / value head: a decode step, draft tokens, and
// every size that the prompt kernel does not take.
//
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  over the positions that a row sees.
//
// What bounds it is the reading of the cache, 2 dim bytes per key and head once for all query heads of the group. The codes go from
// global memory by cp.async into a ring of a warp's own, one step of 16 keys ahead of the one that is worked on (64 KB under way on an
// SM; two ahead, with the records in the ring: 2 requests of 130001 positions 111.0 us, one ahead 106.8), and from there as bytes into the operand registers of mma.sync (m16n8k16, f16):
//   scores   S^T [16 keys x 8 vectors] = K [16 x dim] Q^T: lane (g, t) of a warp reads 16 bytes of keys g and g + 8 at a time; which
//            dimension stands at which place of k is free as long as the queries agree.
//   values   O^T [dim x 8 vectors] += V^T [dim x 16 keys] P^T: lane (g, t) reads 8 neighbouring bytes of the four keys whose
//            weights it holds, and a byte permutation puts two keys of a dimension side by side; the weights are turned by movmatrix.
// Keys as the 16 rows waste none of the tensor core on missing query vectors. Codes are exact in f16; a query vector enters under a
// power of two (one f16 term for bf16 queries, which is exact; two for f32), weights as two f16 terms (22 bits), so that scores, sums
// and outputs are of f32 accuracy. A block's scales stay outside: the key's multiplies the scores, the value's goes into the exponent
// of the weight, w = 2^(s - mv + e_v), which has a reference mv of its own beside the maximum m of the sum (l = sum 2^(s - m)), whatever
// the scales are. It stands 2^11 below the largest s + e_v, so that the largest weight is 2^11 to 2^15, next to the end of f16: the second
// term ends at multiples of 2^-24, which is then 2^-35 of the largest weight and scale. Both references move only when a score passes
// them by 2^4, so most steps have one vote in place of the maxima's exchange. (References at the largest score itself and moves by 2^8
// leave 2^-24: the outputs of 1100 keys 16 / 20 nats under a first one whose value is zero are then off by 9e-3 / 0.13 of the largest in place
// of 4e-6 / 1.3e-4, in the same time.)
// The tensor core cuts off what its f32 sums cannot hold, always towards zero, so chains in it are kept short: 32 dimensions of a
// score, kKvFlush steps of an output, which then join sums in shared memory (2 requests of 130001 positions, f32: all steps in one chain
// 113.5 us and an error of the outputs against 64 bits of 2.3e-6, chains of 16 steps 114.8 us and 0.86e-6, of 8 steps 116.6 us and
// 0.65e-6; torch in f32: 1.24e-6).
//
// Work is dealt in steps of 16 keys: all steps of all (request, head, vectors) items in one row, cut into equal parts, one for each
// CTA, whatever the requests' lengths are. An item counts kKvPad steps more than it has, about what beginning and ending one takes, so
// that many short requests in one part weigh what they cost. An item inside one part is written directly; of an item that is cut every part
// leaves a record (m, mv, l, O), and kv_join_kernel joins them in their order.
// Measured (heads of 128, with the joining): 2 requests of 130001 positions, int8, 8 key / value heads of 5 f32 query heads, 115 us (4.6 TB/s of
// codes); 40 requests of up to 12000, e4m3, 8 heads of 4 bf16 query heads, 90 us (4.0 TB/s); one of 2001 positions 12.5 us, of which the
// two launches, the first loads behind the table and the joining are nearly all. Counters of the first two: issue slots 58 / 64 % used, logic
// pipe 44 / 52 %, tensor pipe 29 / 19 %: the codes' way to the operands stands beside the reading. Heads of 128 with f32 queries spill (128 registers, 192
// bytes of stores: 1 % of the instructions).
#include <algorithm>

#include "kv_attn.cuh"
#include "sync.cuh"

namespace nnq {

constexpr int kKvWarps = 8, kKvCols = 8, kKvStep = 16, kKvStages = 2;
constexpr int kKvMinSteps = kKvWarps;   // of a CTA's part (one request of 2001 positions: 1 / 8 steps 14.3 / 12.5 us)
constexpr int kKvPad = 32;              // (us with 8 / 16 / 32 / 64: 40 ragged requests 107.7 / 90.7 / 85.3 / 97.4; 2 long ones 116.0 / 111.3 with 32 / 64)
constexpr int kKvFlush = 16;
constexpr int kNothing = INT32_MIN;   // in place of a block: no key of the step is seen
constexpr float kKvLog2E = 1.4426950408889634f;
constexpr float kKvSlack = 4.0f, kKvLow = 11.0f;   // a score may pass the references by 2^4; mv is 2^11 lower: weights up to 2^15 in f16

// records: [part][began before, begins here][column]: m, mv, l, unused, then O[dim]; behind them what every part has to join
__host__ __device__ inline int kv_record_floats(int dim) { return 4 + dim; }
struct KvJoin {
    int first;   // part that the item begins in, -1: nothing to join
    int vecs, group_row, head;   // vectors; first vector of the item as (row of q, query head)
    int rest;    // number of the first vector within its row's group
    int unused[3];
};

struct KvPlan {
    int64_t total, chunk;   // steps in all, steps of a part
    int64_t off;            // number within its request of the part's first step
    int r;                  // its request
};

// Steps of an item of the request (the same for all its heads and vectors), and its items of one head.
__device__ __forceinline__ int item_steps(const KvAttn &a, const KvRequest &q) {
    if (q.rows == 0 || kv_many(a, q)) return 0;
    const int lo = row_first(a, max(row_pos(q, 0), 0)), steps = (q.length + kKvStep - 1) / kKvStep - lo / kKvStep;
    return max(steps, 1) + kKvPad;
}
__device__ __forceinline__ int item_count(const KvAttn &a, const KvRequest &q) { return (q.rows * a.group + kKvCols - 1) / kKvCols; }

// Sums the steps of all requests and finds where this CTA's part begins. Up to 32 requests every warp does so for itself, without a
// barrier; more are summed by the whole CTA, twice.
__device__ KvPlan kv_plan(const KvAttn &a, int parts) {
    __shared__ int64_t warp_sums[32], found[2];
    const int nt = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5;
    auto steps_of = [&](int64_t r) -> int64_t {
        if (r >= a.requests) return 0;
        const KvRequest q = kv_request(a, r);
        return (int64_t)item_steps(a, q) * item_count(a, q) * a.kv_heads;
    };
    auto scan = [&](long long x) {
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long b = __shfl_up_sync(0xFFFFFFFFu, x, off);
            if (lane >= off) x += b;
        }
        return x;
    };
    KvPlan p;
    p.r = 0;
    p.off = 0;
    if (a.requests <= 32) {
        const int64_t mine = steps_of(lane), upto = scan(mine);
        p.total = __shfl_sync(0xFFFFFFFFu, (long long)upto, 31);
        p.chunk = max((p.total + parts - 1) / parts, (int64_t)kKvMinSteps);
        const int64_t begin = p.chunk * blockIdx.x;
        const uint32_t m = __ballot_sync(0xFFFFFFFFu, begin >= upto - mine && begin < upto);
        if (m) {
            p.r = __ffs(m) - 1;
            p.off = begin - __shfl_sync(0xFFFFFFFFu, (long long)(upto - mine), p.r);
        }
        return p;
    }
    auto block_scan = [&](int64_t mine, int64_t &before) {
        const int64_t x = scan(mine);
        __syncthreads();
        if (lane == 31) warp_sums[warp] = x;
        __syncthreads();
        int64_t all = 0;
        before = x - mine;
        for (int w = 0; w < nw; w++) {
            if (w < warp) before += warp_sums[w];
            all += warp_sums[w];
        }
        return all;
    };
    p.total = 0;
    int64_t before;
    for (int64_t r0 = 0; r0 < a.requests; r0 += nt) p.total += block_scan(steps_of(r0 + tid), before);
    p.chunk = max((p.total + parts - 1) / parts, (int64_t)kKvMinSteps);
    const int64_t begin = p.chunk * blockIdx.x;
    if (begin >= p.total) return p;
    int64_t done = 0;
    for (int64_t r0 = 0; r0 < a.requests && done <= begin; r0 += nt) {
        const int64_t mine = steps_of(r0 + tid), all = block_scan(mine, before);
        if (begin >= done + before && begin < done + before + mine) {
            found[0] = r0 + tid;
            found[1] = begin - done - before;
        }
        done += all;
    }
    __syncthreads();
    p.r = (int)found[0];
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
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
    return v;
}

// A step in the ring: keys, then values, in pieces of 64 dimensions: 16 rows of 64 bytes, two to a line of 128, whose eight 16-byte
// chunks are exchanged by the line's number so that neither the copies nor the reads of either operand meet in a bank.
__device__ __forceinline__ uint32_t chunk_at(int row, int c) { return (uint32_t)((row >> 1) * 128 + (((((row & 1) << 2) | c) ^ (((row >> 1) & 3) << 1)) << 4)); }

template <int D>
constexpr int kKvRing = kKvWarps * kKvStages * 2 * kKvStep * D;
template <int D>
constexpr int kv_smem_bytes() {
    return kKvRing<D> + kKvWarps * kKvCols * (4 + D) * 4;
}

__device__ __forceinline__ void store_out(const KvAttn &a, int64_t at, float y) {
    if (a.y_dt == NNQ_F32) reinterpret_cast<float *>(a.y)[at] = y;
    else reinterpret_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(y);
}

template <int FMT, int D, int QT>
__global__ void __launch_bounds__(kKvWarps * 32, D <= 128 ? 2 : 1) kv_attn_kernel(const KvAttn a, float *records, KvJoin *joins) {
    extern __shared__ __align__(128) uint8_t kv_smem[];   // the warps' rings, then a record of every warp and column
    typedef CodePairs<FMT> Codes;
    constexpr int REC = 4 + D, STEP = 2 * kKvStep * D;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(kv_smem) + warp * kKvStages * STEP;
    float *sm = reinterpret_cast<float *>(kv_smem + kKvRing<D>);
    pdl_prologue();
    pdl_release();
    const KvPlan plan = kv_plan(a, gridDim.x);
    int64_t at = plan.chunk * blockIdx.x, off = plan.off;
    const int64_t end = min(plan.total, at + plan.chunk);
    int r = plan.r;
    KvJoin join = {-1, 0, 0, 0, 0, {0, 0, 0}};
    KvRequest rq;
    int spi = 0, cols = 0;
    int64_t of_request = -1;
    while (at < end) {
        // ---- the next request with steps left, the item and the part of it that is this CTA's
        if (of_request < 0) {
            rq = kv_request(a, r);
            spi = item_steps(a, rq);
            cols = item_count(a, rq);
            of_request = (int64_t)spi * cols * a.kv_heads;
        }
        if (off >= of_request) {
            off = 0;
            r++;
            of_request = -1;
            continue;
        }
        const int item = (int)(off / spi), v0 = (int)(off - (int64_t)item * spi), v1 = (int)min((int64_t)spi, v0 + end - at);   // steps, the padding first
        const int s0 = max(v0 - kKvPad, 0), s1 = max(v1 - kKvPad, 0);
        const int head = item / cols, vec0 = (item - head * cols) * kKvCols, vecs = min(kKvCols, rq.rows * a.group - vec0);
        const int lo_all = row_first(a, max(row_pos(rq, 0), 0)) / kKvStep * kKvStep;   // the item's step 0 begins here
        // positions of the first and the last vector's row; what every vector sees, and what some vector sees
        const int first_pos = row_pos(rq, vec0 / a.group), last_pos = row_pos(rq, (vec0 + vecs - 1) / a.group);
        const int lo_some = row_first(a, max(first_pos, 0)), lo_every = row_first(a, max(last_pos, 0));
        const int n = s1 > s0 + warp ? (s1 - s0 - warp + kKvWarps - 1) / kKvWarps : 0;   // this warp's steps
        const int32_t *table = a.table + (int64_t)r * a.table_ld;
        const int key_base = lo_all + (s0 + warp) * kKvStep;
        // lane i has the block of the warp's steps j with j mod 32 = i, and its exponent bytes, a batch of 32 at a time and one ahead
        auto block_of = [&](int j) {
            const int key = key_base + j * kKvWarps * kKvStep;
            return j < n && key <= last_pos && key + kKvStep > lo_some ? table[key >> a.shift] : kNothing;
        };
        auto bytes_of = [&](int b, int &ke, int &ve) {
            ke = ve = 127;
            if (b >= 0 && b < a.blocks) {
                ke = a.k_exp[(int64_t)b * a.kv_heads + head];
                ve = a.v_exp[(int64_t)b * a.kv_heads + head];
            } else if (b != kNothing) {
                atomicExch(a.status, kStatusIndex);
            }
        };
        auto fetch = [&](int j, int b) {
            if (b >= 0 && b < a.blocks) {
                const int key = key_base + j * kKvWarps * kKvStep;
                const int64_t from = (((((int64_t)b * a.kv_heads + head) << a.shift) + (key & ((1 << a.shift) - 1))) + (lane >> 2)) * D + (lane & 3) * 16;
                const uint8_t *kp = a.k + from, *vp = a.v + from;
                const uint32_t dst = ring + (uint32_t)(j % kKvStages) * STEP + chunk_at(lane >> 2, lane & 3);
#pragma unroll
                for (int c = 0; c < D / 64; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        copy16(dst + c * 1024 + h * 512, kp + c * 64 + h * 8 * D);
                        copy16(dst + kKvStep * D + c * 1024 + h * 512, vp + c * 64 + h * 8 * D);
                    }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();   // the records of the item before have been read
        int blk = block_of(lane), ke, ve;
        fetch(0, __shfl_sync(0xFFFFFFFFu, blk, 0));

        bytes_of(blk, ke, ve);
        int blk1 = kNothing, ke1 = 127, ve1 = 127;

        // ---- queries: lane (g, t) has vector g's dimensions c * 64 + t * 16 .. + 15 of every c, as the scores' second operand
        uint32_t qh[D / 16][2], ql[QT == 2 ? D / 16 : 1][2];
        float q_un = 1.0f;
        {
            float x[D / 64][16];
            const int v = vec0 + g, row = v / a.group, qhead = head * a.group + v - row * a.group;
            const int64_t from = (int64_t)(rq.row0 + row) * a.q_ld + (int64_t)qhead * D + t * 16;
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < D / 64; c++)
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    float y[8] = {};
                    if (g < vecs) {
                        if constexpr (QT == 2) {
                            const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + from + c * 64 + i);
                            const float4 u = __ldg(p), w = __ldg(p + 1);
                            y[0] = u.x; y[1] = u.y; y[2] = u.z; y[3] = u.w; y[4] = w.x; y[5] = w.y; y[6] = w.z; y[7] = w.w;
                        } else {
                            const uint4 u = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(a.q) + from + c * 64 + i));
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
        int pos[2], low[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            fac[j] = a.scale * kKvLog2E * Codes::unscale * __shfl_sync(0xFFFFFFFFu, q_un, (2 * t + j) * 4);
            pos[j] = row_pos(rq, (vec0 + min(2 * t + j, vecs - 1)) / a.group);
            low[j] = row_first(a, pos[j]);
        }

        float acc[D / 16][4];
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = 0.0f;
        float m[2] = {0.0f, 0.0f}, mv[2] = {0.0f, 0.0f}, l[2] = {0.0f, 0.0f};
        float thr[2] = {-INFINITY, -INFINITY}, thv[2] = {-INFINITY, -INFINITY};   // what makes the references move
        float kept[2] = {-INFINITY, -INFINITY};   // reference of the sums in shared memory (-inf: none yet)
        auto flush = [&]() {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (2 * t + j >= vecs || thr[j] == -INFINITY) continue;
                float *rec = sm + (warp * kKvCols + 2 * t + j) * REC + 4 + 8 * g;
                const float f = kv_ex2(kept[j] - mv[j]);
#pragma unroll
                for (int i = 0; i < D / 16; i += 2) {
                    float4 *p = reinterpret_cast<float4 *>(rec + (i >> 2) * 64 + (i & 2) * 2);
                    float4 o = make_float4(acc[i][j], acc[i][j + 2], acc[i + 1][j], acc[i + 1][j + 2]);
                    if (kept[j] != -INFINITY) {
                        const float4 q = *p;
                        o = make_float4(fmaf(q.x, f, o.x), fmaf(q.y, f, o.y), fmaf(q.z, f, o.z), fmaf(q.w, f, o.w));
                    }
                    *p = o;
                    acc[i][j] = acc[i][j + 2] = acc[i + 1][j] = acc[i + 1][j + 2] = 0.0f;
                }
                kept[j] = mv[j];
            }
        };

        for (int j = 0; j < n; j++) {
            if ((j & 31) == 0) {
                if (j) {
                    blk = blk1;
                    ke = ke1;
                    ve = ve1;
                }
                blk1 = n > j + 32 ? block_of(j + 32 + lane) : kNothing;
            }
            if ((j & 31) == 16 && n > (j | 31)) bytes_of(blk1, ke1, ve1);
            fetch(j + 1, __shfl_sync(0xFFFFFFFFu, (j & 31) < 31 ? blk : blk1, (j + 1) & 31));
            const int b = __shfl_sync(0xFFFFFFFFu, blk, j & 31);
            const float kf = pow2_byte(__shfl_sync(0xFFFFFFFFu, ke, j & 31)), vexp = (float)(__shfl_sync(0xFFFFFFFFu, ve, j & 31) - 127);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            if (b >= 0 && b < a.blocks) {
                const uint32_t k_s = ring + (uint32_t)(j % kKvStages) * STEP, v_s = k_s + kKvStep * D;
                // ---- scores
                float part[D / 32][4];
#pragma unroll
                for (int c = 0; c < D / 64; c++) {
#pragma unroll
                    for (int e = 0; e < 8; e++) part[2 * c + (e >> 2)][e & 3] = 0.0f;
                    const uint4 u0 = lds128(k_s + c * 1024 + chunk_at(g, t)), u1 = lds128(k_s + c * 1024 + 512 + chunk_at(g, t));
                    const uint32_t r0[4] = {u0.x, u0.y, u0.z, u0.w}, r1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t u = Codes::word(r0[i]), w = Codes::word(r1[i]);
                        const uint32_t x[4] = {Codes::low(u), Codes::low(w), Codes::high(u), Codes::high(w)};
                        if constexpr (QT == 2) mma_f16(part[2 * c + (i >> 1)], x, ql[4 * c + i][0], ql[4 * c + i][1]);
                        mma_f16(part[2 * c + (i >> 1)], x, qh[4 * c + i][0], qh[4 * c + i][1]);
                    }
                }
                float sc[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sc[i] = part[0][i] + part[1][i];
#pragma unroll
                    for (int c = 1; c < D / 64; c++) sc[i] += part[2 * c][i] + part[2 * c + 1][i];
                    sc[i] *= fac[i & 1] * kf;
                }
                const int key0 = key_base + j * kKvWarps * kKvStep;
                if (key0 + kKvStep - 1 > first_pos || key0 < lo_every) {   // (the same for the whole warp)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int k = key0 + g + (i >> 1) * 8;
                        if (k > pos[i & 1] || k < low[i & 1]) sc[i] = -INFINITY;
                    }
                }
                // ---- references
                float big[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
                if (__any_sync(0xFFFFFFFFu, big[0] > thr[0] || big[1] > thr[1] || big[0] + vexp > thv[0] || big[1] + vexp > thv[1])) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        big[0] = fmaxf(big[0], __shfl_xor_sync(0xFFFFFFFFu, big[0], o));
                        big[1] = fmaxf(big[1], __shfl_xor_sync(0xFFFFFFFFu, big[1], o));
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (big[i] == -INFINITY) continue;   // nothing seen yet or here
                        const bool none = thr[i] == -INFINITY;   // a first reference: the sums are zero
                        const float mn = none ? big[i] : fmaxf(m[i], big[i]), vn = none ? big[i] + vexp - kKvLow : fmaxf(mv[i], big[i] + vexp - kKvLow);
                        const float f = none ? 1.0f : kv_ex2(mv[i] - vn);
                        l[i] *= none ? 1.0f : kv_ex2(m[i] - mn);
#pragma unroll
                        for (int k = 0; k < D / 16; k++) {
                            acc[k][i] *= f;
                            acc[k][i + 2] *= f;
                        }
                        m[i] = mn;
                        mv[i] = vn;
                        thr[i] = mn + kKvSlack;
                        thv[i] = vn + (kKvLow + kKvSlack);
                    }
                }
                // ---- weights
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    l[i & 1] += kv_ex2(sc[i] - m[i & 1]);
                    w[i] = kv_ex2(sc[i] + (vexp - mv[i & 1]));
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
                for (int c = 0; c < D / 64; c++) {
                    const uint32_t p = v_s + c * 1024 + (g & 1) * 8, even = p + chunk_at(2 * t, g >> 1), odd = p + chunk_at(2 * t + 1, g >> 1);
                    const uint2 y0 = lds64(even), y1 = lds64(odd), y2 = lds64(even + 512), y3 = lds64(odd + 512);
#pragma unroll
                    for (int hw = 0; hw < 2; hw++) {
                        uint32_t x0[4], x1[4];
                        Codes::pairs(hw ? y0.y : y0.x, hw ? y1.y : y1.x, x0[0], x0[1], x1[0], x1[1]);
                        Codes::pairs(hw ? y2.y : y2.x, hw ? y3.y : y3.x, x0[2], x0[3], x1[2], x1[3]);
                        mma_f16(acc[4 * c + 2 * hw], x0, l0, l1);
                        mma_f16(acc[4 * c + 2 * hw + 1], x1, l0, l1);
                        mma_f16(acc[4 * c + 2 * hw], x0, h0, h1);
                        mma_f16(acc[4 * c + 2 * hw + 1], x1, h0, h1);
                    }
                }
            }
            if ((j & (kKvFlush - 1)) == kKvFlush - 1) flush();
            __syncwarp();   // the stage may be written again
        }
        flush();
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the rest of the warps' records (m = -inf: nothing seen)
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[j] += __shfl_xor_sync(0xFFFFFFFFu, l[j], o);
            if (2 * t + j >= vecs || g > 0) continue;
            float *rec = sm + (warp * kKvCols + 2 * t + j) * REC;
            rec[0] = thr[j] > -INFINITY ? m[j] : (l[j] == 0.0f ? -INFINITY : l[j]);   // (scores that are all NaN move no reference)
            rec[1] = mv[j];
            rec[2] = l[j];
        }
        __syncthreads();
        const bool whole = v0 == 0 && v1 == spi;
        for (int u = tid; u < vecs * D; u += kKvWarps * 32) {
            const int col = u / D, d = u - col * D;
            float wm[kKvWarps], mm = -INFINITY, mvv = -INFINITY;
#pragma unroll
            for (int w = 0; w < kKvWarps; w++) {
                const float *rec = sm + (w * kKvCols + col) * REC;
                wm[w] = rec[0];
                mm = fmaxf(mm, wm[w]);
                if (wm[w] != -INFINITY) mvv = fmaxf(mvv, rec[1]);
            }
            float ll = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < kKvWarps; w++) {
                const float *rec = sm + (w * kKvCols + col) * REC;
                if (wm[w] == -INFINITY) continue;
                ll += rec[2] * kv_ex2(wm[w] - mm);
                o += rec[4 + d] * kv_ex2(rec[1] - mvv);
            }
            if (whole) {
                const int v = vec0 + col, row = v / a.group;
                // (2^(mv - m) in two halves: it can lie below the numbers where the output does not. No key seen: 0; NaN: l is)
                const float h = exp2f(0.5f * (mvv - mm)), y = ll == 0.0f ? 0.0f : o * Codes::unscale / ll * h * h;
                store_out(a, (int64_t)(rq.row0 + row) * a.y_ld + (int64_t)(head * a.group + v - row * a.group) * D + d, y);
            } else {
                float *rec = records + (((int64_t)blockIdx.x * 2 + (v0 == 0 ? 1 : 0)) * kKvCols + col) * REC;
                rec[4 + d] = o;
                if (d == 0) {
                    rec[0] = ll == 0.0f ? -INFINITY : mm > -INFINITY ? mm : ll;   // (NaN where all scores are)
                    rec[1] = mvv;
                    rec[2] = ll;
                }
            }
        }
        if (!whole && v1 == spi) {
            join.first = (int)((at - v0) / plan.chunk);
            join.vecs = vecs;
            join.group_row = rq.row0 + vec0 / a.group;
            join.head = head;
            join.rest = vec0 % a.group;
        }
        at += v1 - v0;
        off += v1 - v0;
    }
    if (tid == 0) joins[blockIdx.x] = join;
}

// Joins the records of an item that was cut: CTA (part that the item ends in, vector), the records dealt to eight warps.
template <int FMT>
__global__ void __launch_bounds__(256) kv_join_kernel(const KvAttn a, const float *records, const KvJoin *joins) {
    __shared__ float4 part[8][64];
    __shared__ float2 part_l[8];
    pdl_prologue();
    const KvJoin j = joins[blockIdx.x];
    const int col = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quads = a.dim / 4, last = blockIdx.x;
    if (j.first < 0 || col >= j.vecs) return;
    const int rec_floats = kv_record_floats(a.dim);
    auto record = [&](int p) { return records + ((int64_t)(p * 2 + (p == j.first ? 1 : 0)) * kKvCols + col) * rec_floats; };
    // the references of all records, a lane per record and turn
    float mm = -INFINITY, mv = -INFINITY;
    for (int p = j.first + lane; p <= last; p += 32) {
        const float4 h = *reinterpret_cast<const float4 *>(record(p));
        if (h.x == -INFINITY) continue;
        mm = fmaxf(mm, h.x);
        mv = fmaxf(mv, h.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mm = fmaxf(mm, __shfl_xor_sync(0xFFFFFFFFu, mm, o));
        mv = fmaxf(mv, __shfl_xor_sync(0xFFFFFFFFu, mv, o));
    }
    float4 o[2] = {};
    float l = 0.0f;
#pragma unroll 4
    for (int p = j.first + warp; p <= last; p += 8) {
        const float *rec = record(p);
        const float4 h = *reinterpret_cast<const float4 *>(rec);
        if (h.x == -INFINITY) continue;
        const float f = exp2f(h.y - mv);
        l += h.z * exp2f(h.x - mm);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (lane + 32 * i >= quads) continue;
            const float4 x = reinterpret_cast<const float4 *>(rec + 4)[lane + 32 * i];
            o[i].x += x.x * f;
            o[i].y += x.y * f;
            o[i].z += x.z * f;
            o[i].w += x.w * f;
        }
    }
    part[warp][lane] = o[0];
    part[warp][lane + 32] = o[1];
    if (lane == 0) part_l[warp] = make_float2(l, 0.0f);
    __syncthreads();
    const int q = threadIdx.x;
    if (q >= quads) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        const float4 x = part[w][q];
        s.x += x.x;
        s.y += x.y;
        s.z += x.z;
        s.w += x.w;
        l += part_l[w].x;
    }
    const float h = exp2f(0.5f * (mv - mm)), f = l == 0.0f ? 0.0f : CodePairs<FMT>::unscale / l;
    const int v = j.rest + col, row = v / a.group;
    const int64_t to = (int64_t)(j.group_row + row) * a.y_ld + (int64_t)(j.head * a.group + v - row * a.group) * a.dim + 4 * q;
    const float y[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; i++) store_out(a, to + i, l == 0.0f ? 0.0f : y[i] * f * h * h);
}

static int kv_parts(nnq_ctx *ctx, int dim) { return (dim <= 128 ? 2 : 1) * ctx->sm_count; }
static size_t kv_records_bytes(nnq_ctx *ctx, int dim) { return (size_t)kv_parts(ctx, dim) * 2 * kKvCols * kv_record_floats(dim) * 4; }

template <int FMT, int D, int QT>
static nnq_status launch_kv_attn(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    constexpr int smem = kv_smem_bytes<D>();
    static std::atomic<uint64_t> done;
    nnq_status s = allow_smem(ctx, kv_attn_kernel<FMT, D, QT>, smem, done);
    if (s != NNQ_OK) return s;
    const int parts = kv_parts(ctx, D);
    KvJoin *joins = reinterpret_cast<KvJoin *>(reinterpret_cast<uint8_t *>(records) + kv_records_bytes(ctx, D));
    launch_pdl_smem(kv_attn_kernel<FMT, D, QT>, dim3(parts), dim3(kKvWarps * 32), smem, st, a, records, joins);
    launch_pdl(kv_join_kernel<FMT>, dim3(parts, (unsigned)std::min<int64_t>(kKvCols, (int64_t)a.rows * a.group)), dim3(256), st, a, records, joins);
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

// Can the batch have requests for the tensor-core kernel, whatever their lengths are?
static bool tc_rows(int dim, int group, int64_t max_rows, int few) { return kv_attn_tc_supported(dim) && max_rows > few / group; }

static nnq_status check_batch(nnq_ctx *ctx, const nnq_kv_cache *c, const nnq_kv_batch *b, int heads) {
    nnq_status s = check_kv_cache(ctx, c);
    if (s != NNQ_OK) return s;
    if (!b) return fail(ctx, NNQ_ERR_INVALID_ARG, "batch is NULL");
    if (heads < 1 || heads % c->kv_heads) return fail(ctx, NNQ_ERR_SHAPE_MISMATCH, "%d query heads over %d key / value heads", heads, c->kv_heads);
    if (b->requests < 1 || b->rows < 0 || b->table_ld < 1 || b->max_rows < 1) return fail(ctx, NNQ_ERR_INVALID_ARG, "bad sizes of a batch");
    // (positions are counted in 32 bits, up to a tile beyond the last)
    if (b->table_ld > (INT32_MAX - 1024) / c->block) return fail(ctx, NNQ_ERR_UNSUPPORTED, "tables of %lld blocks of %d tokens", (long long)b->table_ld, c->block);
    // (so are query vectors, up to an item beyond the last)
    if (b->requests > INT32_MAX / 2 || b->rows > (INT32_MAX - 1024) / heads) return fail(ctx, NNQ_ERR_UNSUPPORTED, "a batch of %lld requests and %lld rows", (long long)b->requests, (long long)b->rows);
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
    *bytes = kv_records_bytes(ctx, c->dim) + kv_parts(ctx, c->dim) * sizeof(KvJoin);
    if (tc_rows(c->dim, heads / c->kv_heads, b->max_rows, kKvFew)) *bytes = std::max(*bytes, kv_attn_tc_workspace(ctx, c->dim));
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
                      c->kv_heads, heads / c->kv_heads, c->dim, log2_of(c->block), window, (int)q_dt, (int)y_dt, INT32_MAX, INT32_MAX, scale, ctx->d_status};
    // The batch's requests are dealt between the two kernels on the device (kv_many). The tensor-core kernel is not launched where the
    // rows, the table's width and the window leave it none; a prompt alone goes to it wholly.
    const bool prompt = b->max_rows > kKvAlways / a.group;
    const int few = q_dt == NNQ_BF16 && y_dt == NNQ_BF16 ? kKvFew : kKvFewF32;
    int64_t keys = b->table_ld * c->block;
    if (window > 0) keys = std::min(keys, window + std::min(b->max_rows, b->rows));
    if (tc_rows(a.dim, a.group, b->max_rows, few) && (prompt || keys * a.kv_heads >= (kKvManyKeys + b->requests - 1) / b->requests)) {
        const bool all = prompt && b->requests == 1;
        a.few = all ? 0 : few;
        a.many = all ? 0 : kKvAlways;
        if ((s = launch_kv_attn_tc(ctx, a, c->format, (float *)workspace, (cudaStream_t)stream)) != NNQ_OK || all) return s;
    }
    return c->format == NNQ_KV_INT8 ? launch_kv_attn<NNQ_KV_INT8>(ctx, a, (float *)workspace, (cudaStream_t)stream)
                                    : launch_kv_attn<NNQ_KV_E4M3>(ctx, a, (float *)workspace, (cudaStream_t)stream);
}

}  // extern "C"
