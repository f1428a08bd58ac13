// Attention over the paged 8-bit cache (kv_cache.cuh) for many query vectors per key / value head -- prompts and their portions -- on
// the 5th-generation tensor cores: heads of 64 and 128.
//
// One CTA has up to 256 query vectors of one key / value head (consecutive (row, query head of the group) pairs), 128 for each of two
// softmax groups, and walks over tiles of keys that both share.
//   warps 0-3, 4-7: softmax. Thread r of a group owns query vector r: its scores of 64 keys from tensor memory, maximum and sum; the
//                   weights go back into the columns of the scores as f16, where the second product reads them. Scores have two places,
//                   so that the next tile's are there when a tile is done. The weighted values of all tiles add up in tensor
//                   memory; a reference moves only when a score passes it by 2^8, and then the sums there are scaled.
//   warps 8-15:     codes from the blocks of the table to f16 tiles in shared memory, swizzled as the products read them, keys and values
//                   as they lie (the values are the MN-major operand); the next tile's codes are under way meanwhile.
//   warps 16, 17:   (two more complete their group) a lane of each issues the MMAs of one softmax group: S(t + 1), then O += P(t) V(t). They
//                   run in the order they are issued, so S(t + 1) may overwrite the weights of t - 1, whose product stands in front
//                   of it. (One warp for both groups took 100 clocks an MMA beside the scheduler's other warps and set the pace.)
// What bounds it are waits, not a unit: per 64 keys a softmax group goes through scores -> maxima -> weights -> hand-over, with two of its warps on a
// scheduler. Measured: 2000 rows behind 2100, e4m3, 8 key / value heads of 4 bf16 query heads of 128, 215 us with the joining, 474 TFLOP/s of the
// 102 GFLOP that a causal prompt takes: 7900 warp instructions of an SM per tile of both groups, issue slots 51 % used, tensor pipe 39 %, logic
// pipe 38 %, special functions 28 %, FMA pipe 22 %; of the warps' waits four in ten for loads (of scores from tensor memory, of codes). f32 rows: 346 us, 34 %
// and 32 %, with the records' sums beside them. Slower were 128 keys a tile with both
// MMA warps on each (217 us where this form took 182) and four converter warps in favour of more registers for the softmax (186 beside 182).
// The compiler spills (-Xptxas -v: 404 to 424 bytes of stores, 96 registers; it does not say in which role): 1.7 % of the instructions are loads and
// stores of local memory.
// Codes are exact in f16. A query vector is one f16 term under its power of two where that is exact (T = 1: bf16 queries and outputs), else two (T = 2); a
// weight is always two, 22 bits (with one, 11 bits and 188 us for the prompt above, a bf16 output differed from the rounded exact one by 9e-4 in the
// 2-norm, now by 2e-4).
// The tensor core cuts off what its f32 sums cannot hold, towards zero, so a chain of products in tensor memory ends after kTcChain tiles and its sums
// join others in the item's record in the workspace, in f32 (a second place in tensor memory would need columns that heads of 128 leave
// none of). Mean error of f32 outputs over 3000 / 12001 / 32000 positions, heads of 128, e4m3: in one chain 3.2e-6 / 1.4e-5 / 3.8e-5, of 8 tiles
// 2.0e-6 (3000), of 4 tiles 1.1e-6 / 1.2e-6 / 1.2e-6; 2000 f32 rows behind 2100: 264, 308, 346 us. With bf16 outputs chains of 64 tiles, some 2e-5 of an
// output, which is far below its rounding, and 1.0 of the time of one chain.
// Scales: a block's key exponent multiplies its scores in f32. Its value exponent enters the weight, w = p 2^(m - mv + e_v) with a
// reference mv of its own, 2^7 below the largest score + e_v as m is the largest score: one factor per vector and 16 keys, and weights
// up to 2^15 whatever the scales are, as in kv_attn.cu. References move for 2^8 here, not 2^4, as the sums are scaled in tensor memory
// (prompt of 2000 rows behind 2100, moves for 2^4 / 2^6 / 2^7 / 2^8: 216 / 204 / 194 / 192 us).
//
// Work: the key tiles of all (request, head, 256 vectors) items in one row, cut into equal parts, one per SM: causal rows and
// long contexts load all SMs alike. An item inside a part is written directly, of one that is cut every part leaves a record, and
// kv_tc_join_kernel joins them in order.
#include <algorithm>
#include <type_traits>

#include "kv_attn.cuh"
#include "tcgen05.cuh"

namespace nnq {

constexpr int kTcCols = 256, kTcThreads = 20 * 32, kTcKeys = 64, kTcMinSteps = 8;
constexpr int kTcChain = 4, kTcChainBf16 = 64;   // tiles of a chain, by the outputs' type; powers of two
constexpr int kTcNone = INT32_MIN;   // in place of a block: no such key
constexpr float kTcLog2E = 1.4426950408889634f, kTcSlack = 8.0f, kTcLow = 7.0f;   // weights up to 2^15

struct TcItem {
    int r, head, cb;              // request, key / value head, number of the 256 vectors
    int row0, rows, length;       // of the request
    int vec0, vecs;               // of the item
    int first;                    // first tile of the item
    int steps, s0, s1;            // tiles of the item, and this part's
};

struct TcRequest {
    int row0, rows, length, cbs;   // cbs 0: not this kernel's
};

__device__ __forceinline__ TcRequest tc_request(const KvAttn &a, int64_t r) {
    TcRequest q = {0, 0, 0, 0};
    if (r >= a.requests) return q;
    const KvRequest k = kv_request(a, r);
    q.row0 = k.row0;
    q.rows = k.rows;
    q.length = k.length;
    if (kv_many(a, k)) q.cbs = (k.rows * a.group + kTcCols - 1) / kTcCols;
    return q;
}
template <int KT>
__device__ __forceinline__ void tc_range(const KvAttn &a, const TcRequest &q, int cb, int &first, int &steps) {
    const int base = q.length - q.rows, r0 = base + cb * kTcCols / a.group, r1 = base + (min((cb + 1) * kTcCols, q.rows * a.group) - 1) / a.group;
    const int lo = row_first(a, r0);
    first = r1 < 0 ? 0 : lo / KT;
    steps = r1 < 0 ? 1 : r1 / KT - first + 1;
}
// tiles of one head of a request, by a whole warp
template <int KT>
__device__ __forceinline__ int64_t tc_head_steps(const KvAttn &a, const TcRequest &q) {
    int64_t n = 0;   // (a prompt of some million rows passes 32 bits)
    for (int cb = threadIdx.x & 31; cb < q.cbs; cb += 32) {
        int f, s;
        tc_range<KT>(a, q, cb, f, s);
        n += s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, (long long)n, o);
    return n;
}

struct TcPlan {
    int64_t begin, end, chunk;
};

// Where this CTA's part begins and ends, and the item that it begins in (by all threads; `found` in shared memory).
template <int KT>
__device__ TcPlan tc_plan(const KvAttn &a, int parts, int *found, int64_t *sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    TcPlan p = {0, 0, 1};
    // tiles of 32 requests per warp: a lane has one request's; the warps' sums one behind the other
    auto pass = [&](int64_t r0, int64_t &mine, int64_t &before) {
        const int64_t r = r0 + tid;
        const TcRequest q = tc_request(a, r);
        mine = 0;
        for (uint32_t m = __ballot_sync(0xFFFFFFFFu, q.cbs > 0); m; m &= m - 1) {
            const int src = __ffs(m) - 1;
            const TcRequest o = {__shfl_sync(0xFFFFFFFFu, q.row0, src), __shfl_sync(0xFFFFFFFFu, q.rows, src), __shfl_sync(0xFFFFFFFFu, q.length, src), __shfl_sync(0xFFFFFFFFu, q.cbs, src)};
            const int64_t n = tc_head_steps<KT>(a, o);
            if (lane == src) mine = n * a.kv_heads;
        }
        long long x = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long b = __shfl_up_sync(0xFFFFFFFFu, x, off);
            if (lane >= off) x += b;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int64_t all = 0;
        before = x - mine;
        for (int w = 0; w < nw; w++) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
        return all;
    };
    int64_t total = 0, mine, before;
    for (int64_t r0 = 0; r0 < a.requests; r0 += blockDim.x) total += pass(r0, mine, before);
    p.chunk = max((total + parts - 1) / parts, (int64_t)kTcMinSteps);
    p.begin = min(total, p.chunk * blockIdx.x);
    p.end = min(total, p.begin + p.chunk);
    if (p.begin >= p.end) return p;
    int64_t done = 0;
    for (int64_t r0 = 0; r0 < a.requests && done <= p.begin; r0 += blockDim.x) {
        const int64_t all = pass(r0, mine, before);
        if (p.begin >= done + before && p.begin < done + before + mine) {
            found[0] = (int)(r0 + tid);
            sums[32] = p.begin - done - before;
        }
        done += all;
    }
    __syncthreads();
    if (warp == 0) {   // head and vectors within the request
        const TcRequest q = tc_request(a, found[0]);
        const int64_t per_head = tc_head_steps<KT>(a, q), off = sums[32];
        const int head = (int)(off / per_head);
        const int64_t rest = off - head * per_head;
        int64_t sum = 0;
        for (int c0 = 0; c0 < q.cbs; c0 += 32) {
            int f, s = 0;
            if (c0 + lane < q.cbs) tc_range<KT>(a, q, c0 + lane, f, s);
            int x = s;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int b = __shfl_up_sync(0xFFFFFFFFu, x, o);
                if (lane >= o) x += b;
            }
            if (rest >= sum + x - s && rest < sum + x) {
                found[1] = head;
                found[2] = c0 + lane;
                found[3] = (int)(rest - (sum + x - s));
            }
            sum += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
    }
    __syncthreads();
    return p;
}

// The items of a part, one after the other; every role of the CTA walks through them alike.
template <int KT>
struct TcWalk {
    const KvAttn &a;
    TcRequest q;
    int r, head, cb, s0;
    int64_t left;
    __device__ TcWalk(const KvAttn &a_, const TcPlan &p, const int *found) : a(a_), r(found[0]), head(found[1]), cb(found[2]), s0(found[3]), left(p.end - p.begin) {
        q.cbs = 0;
        if (left > 0) q = tc_request(a, r);
    }
    __device__ bool next(TcItem &it) {
        if (left <= 0) return false;
        while (cb >= q.cbs) {   // (a part ends with the last request's tiles at the latest)
            cb = 0;
            if (q.cbs == 0 || ++head >= a.kv_heads) {
                head = 0;
                if (++r >= a.requests) return false;
                q = tc_request(a, r);
            }
        }
        tc_range<KT>(a, q, cb, it.first, it.steps);
        it.r = r;
        it.head = head;
        it.cb = cb;
        it.row0 = q.row0;
        it.rows = q.rows;
        it.length = q.length;
        it.vec0 = cb * kTcCols;
        it.vecs = min(kTcCols, q.rows * a.group - it.vec0);
        it.s0 = s0;
        it.s1 = (int)min((int64_t)it.steps, s0 + left);
        left -= it.s1 - it.s0;
        s0 = 0;
        cb++;
        return true;
    }
};

__host__ __device__ inline int64_t tc_record_floats(int dim) { return (int64_t)kTcCols * (4 + dim); }   // per vector m, mv, l, unused; then [dim / 4][vector] of four

struct TcJoin {   // what a part has to join: the item that ends in it
    int first;   // part that the item begins in, -1: nothing
    int vecs, row, head, rest;   // vectors; row of the first one, first query head of its group, its number there
    int unused[3];
};

template <int D, int T>
struct TcShared {
    static constexpr int KT = kTcKeys, atoms = D / 64, stages = T == 1 ? 4 : 3;
    static constexpr int q_atom = 128 * 128, k_atom = KT * 128;
    static constexpr int q_bytes = 2 * T * atoms * q_atom, stage = 2 * atoms * k_atom;
    static constexpr int bytes = 1024 + q_bytes + stages * stage;
};

__device__ __forceinline__ void tc_st(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                   "r"(v[14]), "r"(v[15]), "r"(addr) : "memory");
}
// MN-major, 128-byte swizzle: 64 columns by 8 k rows per 1024 bytes, the next 64 columns `next` bytes on
__device__ __forceinline__ uint64_t tc_desc_mn(uint32_t addr, uint32_t next) {
    const uint32_t lo = ((addr >> 4) & 0x3FFFu) | ((next >> 4) << 16), hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
// 64 columns, and the wait for them in the same statement: a register of the load must not be touched in between
__device__ __forceinline__ void tc_ld64(uint32_t addr, uint32_t (&v)[2][32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,"
        "%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[0][4]), "=r"(v[0][5]), "=r"(v[0][6]), "=r"(v[0][7]), "=r"(v[0][8]), "=r"(v[0][9]), "=r"(v[0][10]),
          "=r"(v[0][11]), "=r"(v[0][12]), "=r"(v[0][13]), "=r"(v[0][14]), "=r"(v[0][15]), "=r"(v[0][16]), "=r"(v[0][17]), "=r"(v[0][18]), "=r"(v[0][19]), "=r"(v[0][20]), "=r"(v[0][21]),
          "=r"(v[0][22]), "=r"(v[0][23]), "=r"(v[0][24]), "=r"(v[0][25]), "=r"(v[0][26]), "=r"(v[0][27]), "=r"(v[0][28]), "=r"(v[0][29]), "=r"(v[0][30]), "=r"(v[0][31]), "=r"(v[1][0]),
          "=r"(v[1][1]), "=r"(v[1][2]), "=r"(v[1][3]), "=r"(v[1][4]), "=r"(v[1][5]), "=r"(v[1][6]), "=r"(v[1][7]), "=r"(v[1][8]), "=r"(v[1][9]), "=r"(v[1][10]), "=r"(v[1][11]),
          "=r"(v[1][12]), "=r"(v[1][13]), "=r"(v[1][14]), "=r"(v[1][15]), "=r"(v[1][16]), "=r"(v[1][17]), "=r"(v[1][18]), "=r"(v[1][19]), "=r"(v[1][20]), "=r"(v[1][21]), "=r"(v[1][22]),
          "=r"(v[1][23]), "=r"(v[1][24]), "=r"(v[1][25]), "=r"(v[1][26]), "=r"(v[1][27]), "=r"(v[1][28]), "=r"(v[1][29]), "=r"(v[1][30]), "=r"(v[1][31])
        : "r"(addr)
        : "memory");
}
// A role's registers, of the 640 threads x 96 = 61440 that the block is launched with: 256 x 152 + 256 x 64 + 128 x 48 = 61440.
template <int N>
__device__ __forceinline__ void tc_registers() {
    if constexpr (N > 96) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void group_sync(int w) { asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory"); }

template <int FMT, int D, int T>
__global__ void __launch_bounds__(kTcThreads, 1) kv_attn_tc_kernel(const KvAttn a, float *records, TcJoin *joins) {
    typedef TcShared<D, T> Sh;
    typedef CodePairs<FMT> Codes;
    constexpr int KT = Sh::KT, ATOMS = Sh::atoms, SUBS = KT / 16, STAGES = Sh::stages;
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    uint8_t *smem = tc_smem_raw + (-smem_u32(tc_smem_raw) & 1023u);
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 16];   // full, empty; of two groups q_full, and two places each of s_full, p_full, o_done; drain
    __shared__ __align__(16) int2 sub_info[STAGES][SUBS];                  // exponent bytes of keys and values of every 16 keys; x < 0: unseen
    __shared__ uint32_t tmem_s;
    __shared__ int found[4];
    __shared__ int64_t sums[33];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t full = smem_u32(bars), empty = full + 8 * STAGES, qf = empty + 8 * STAGES, sf = qf + 16, pf = sf + 32, of = pf + 32, drain = of + 32;
    pdl_prologue();
    pdl_release();
    const TcPlan plan = tc_plan<KT>(a, gridDim.x, found, sums);
    if (plan.begin >= plan.end) {
        if (tid == 0) joins[blockIdx.x].first = -1;
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(full + 8 * i, 8);
            mbar_init(empty + 8 * i, 2);
        }
        for (int w = 0; w < 2; w++) {
            mbar_init(qf + 8 * w, 1);
            mbar_init(sf + 16 * w, 1);
            mbar_init(sf + 16 * w + 8, 1);
            mbar_init(pf + 16 * w, 4);
            mbar_init(pf + 16 * w + 8, 4);
            mbar_init(of + 16 * w, 1);
            mbar_init(of + 16 * w + 8, 1);
        }
        mbar_init(drain, 1);
        mbar_init(drain + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_s, 0);   // of group w: O at 256 w, S and P at 256 w + 128 and 64 on
    uint8_t *stages = smem + Sh::q_bytes;
    const int chain = a.y_dt == NNQ_F32 ? kTcChain : kTcChainBf16;
    bool ok = true;
    TcWalk<KT> walk(a, plan, found);
    TcItem it;
    int n = 0;   // tiles so far

    if (warp < 8) {
        // ---------------- softmax ----------------
        tc_registers<152>();
        const int w = warp >> 2, me = tid & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, o_t = tmem + 256 * w + lane_base;
        uint8_t *q_s = smem + w * T * ATOMS * Sh::q_atom;
        int nw = 0;   // this group's tiles
        while (ok && walk.next(it)) {
            if (w * 128 >= it.vecs) {   // nothing for the second group
                n += it.s1 - it.s0;
                continue;
            }
            const int vec = it.vec0 + min(w * 128 + me, it.vecs - 1), row = vec / a.group, qhead = it.head * a.group + vec - row * a.group;
            uint32_t big = 0;
            {
                // the thread's query vector, 32 dimensions at a time: first for its largest value, then (from L1) for the terms
                const int64_t at = (int64_t)(it.row0 + row) * a.q_ld + (int64_t)qhead * D;
                auto part = [&](int c, float (&x)[32]) {
                    if (T == 2 && a.q_dt == NNQ_F32) {
                        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(a.q) + at + 32 * c);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float4 f = __ldg(p + i);
                            x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
                        }
                    } else {
                        const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(a.q) + at + 32 * c);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint4 u = __ldg(p + i);
                            const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                x[8 * i + 2 * e] = __uint_as_float(v[e] << 16);
                                x[8 * i + 2 * e + 1] = __uint_as_float(v[e] & 0xFFFF0000u);
                            }
                        }
                    }
                };
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    float x[32];
                    part(c, x);
#pragma unroll
                    for (int i = 0; i < 32; i++) big = max(big, __float_as_uint(x[i]) & 0x7FFFFFFFu);
                }
                const float sc = kv_top_scale(big);
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    float x[32];
                    part(c, x);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) kv_split(x[8 * i + 2 * e] * sc, x[8 * i + 2 * e + 1] * sc, hi[e], lo[e]);
                        uint8_t *dst = q_s + (c >> 1) * Sh::q_atom + swz(me, (c & 1) * 4 + i);
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if (T == 2) *reinterpret_cast<uint4 *>(dst + ATOMS * Sh::q_atom) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
            }
            fence_async_smem();
            group_sync(w);
            if (me == 0) mbar_arrive(qf + 8 * w);
            const int pos = it.length - it.rows + row;
            const int low = row_first(a, pos);
            const float fac = a.scale * kTcLog2E * Codes::unscale * kv_top_unscale(big);
            float m = 0.0f, mv = 0.0f, l = 0.0f, thr = -INFINITY, thv = -INFINITY;
            // the weights of the group's tile number `t` are in tensor memory
            auto hand_over = [&](int t) {
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (elect_one()) mbar_arrive(pf + 8 * (2 * w + (t & 1)));
            };
            // Products add up in tensor memory for `chain` tiles at most, then join the sums in the item's record, of which a thread has one vector as well.
            float4 *rec = reinterpret_cast<float4 *>(records + ((int64_t)blockIdx.x * 2 + (it.s0 == 0 ? 1 : 0)) * tc_record_floats(D)) + w * 128 + me;
            float kept = -INFINITY;   // reference of the record's sums (-inf: they are zero)
            auto join_sums = [&](int c, uint32_t (&x)[32]) {   // 32 dimensions
                const float f = exp2f(kept - mv);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float4 q = rec[kTcCols * (1 + 8 * c + i)];
                    x[4 * i] = __float_as_uint(fmaf(q.x, f, __uint_as_float(x[4 * i])));
                    x[4 * i + 1] = __float_as_uint(fmaf(q.y, f, __uint_as_float(x[4 * i + 1])));
                    x[4 * i + 2] = __float_as_uint(fmaf(q.z, f, __uint_as_float(x[4 * i + 2])));
                    x[4 * i + 3] = __float_as_uint(fmaf(q.w, f, __uint_as_float(x[4 * i + 3])));
                }
            };
            auto keep_sums = [&](int c, const uint32_t (&x)[32]) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    rec[kTcCols * (1 + 8 * c + i)] = make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]), __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3]));
            };
            // the weights of the chain's last tile are handed over here, and the tile behind it begins as an item's first one does
            auto drain_sums = [&](bool again) {
                hand_over(nw - 1);
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(of + 8 * (2 * w + ((nw - 1) & 1)), ((nw - 1) >> 1) & 1));
                if (!ok) return;
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(o_t + 32 * c, x);
                    if (again) join_sums(c, x);
                    keep_sums(c, x);
                }
                kept = thr > -INFINITY ? mv : -INFINITY;
            };
            // A tile of keys, starting at key0; CLEAR: every vector of the warp sees all of it.
            // (`first` of a chain: no weights to hand over, no sums to scale)
            auto tile = [&](auto clear, const int2 *sub, int key0, bool first) {
                const uint32_t s_t = o_t + 128 + 64 * (nw & 1);
                constexpr bool CLEAR = decltype(clear)::value;
                uint32_t seen[KT / 32];   // a bit per key
                if constexpr (!CLEAR) {
#pragma unroll
                    for (int c = 0; c < KT / 32; c++) {
                        const int hi = pos - key0 - 32 * c, lo = low - key0 - 32 * c;   // visible keys of the 32: lo .. hi
                        seen[c] = (hi >= 31 ? 0xFFFFFFFFu : hi < 0 ? 0u : (2u << hi) - 1u) & (lo <= 0 ? 0xFFFFFFFFu : lo > 31 ? 0u : 0xFFFFFFFFu << lo);
                        if (sub[2 * c].x < 0) seen[c] &= 0xFFFF0000u;
                        if (sub[2 * c + 1].x < 0) seen[c] &= 0xFFFFu;
                    }
                }
                // ---- maxima: of the scores, and of scores + value exponents
                float mt = -INFINITY, vt = -INFINITY;
                uint32_t x[2][32];
                float lf[SUBS], fk[SUBS];   // of 16 keys: value exponent (then the weights' factor), the scores' factor
                tc_ld64(s_t, x);
                if (!first) hand_over(nw - 1);   // (the weights' way to tensor memory has passed during the load)
                {
#pragma unroll
                    for (int b = 0; b < SUBS; b++) {
                        const int2 info = sub[b];
                        fk[b] = fac * pow2_byte(max(info.x, 0));
                        lf[b] = (float)(info.y - 127);
                        float t[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            t[i] = __uint_as_float(x[b >> 1][16 * (b & 1) + i]);
                            if (!CLEAR) t[i] = seen[b >> 1] >> (16 * (b & 1) + i) & 1u ? t[i] : -INFINITY;
                        }
                        float top = max3(max3(max3(t[0], t[1], t[2]), max3(t[3], t[4], t[5]), max3(t[6], t[7], t[8])), max3(t[9], t[10], t[11]), max3(t[12], t[13], fmaxf(t[14], t[15])));
                        if (CLEAR || top > -INFINITY) top *= fk[b];   // (the factor can be zero)
                        mt = fmaxf(mt, top);
                        vt = fmaxf(vt, top + lf[b]);
                    }
                }
                // ---- references
                const bool moves = mt > thr || vt > thv;
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    float f = 1.0f;
                    if (moves) {
                        const bool none = thr == -INFINITY;   // a first reference: the sums are zero
                        const float mn = none ? mt : fmaxf(m, mt), vn = none ? vt - kTcLow : fmaxf(mv, vt - kTcLow);
                        if (!none) {
                            l *= exp2f(m - mn);
                            f = exp2f(mv - vn);
                        }
                        m = mn;
                        mv = vn;
                        thr = mn + kTcSlack;
                        thv = vn + (kTcLow + kTcSlack);
                    }
                    if (!first && __any_sync(0xFFFFFFFFu, f != 1.0f)) {
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(of + 8 * (2 * w + ((nw - 1) & 1)), ((nw - 1) >> 1) & 1));
                        if (!ok) return;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32], y[16];
                            tmem_ld32(o_t + 32 * c, o);
#pragma unroll
                            for (int h = 0; h < 2; h++) {
#pragma unroll
                                for (int i = 0; i < 16; i++) y[i] = __float_as_uint(__uint_as_float(o[16 * h + i]) * f);
                                tc_st(o_t + 32 * c + 16 * h, y);
                            }
                        }
                    }
                }
                // ---- weights: w = 2^(s - m + lf); the sum takes 2^-lf of the 16 together (below 2^-56 a weight is zero in f16 either way)
                {
#pragma unroll
                    for (int b = 0; b < SUBS; b++) lf[b] = fmaxf(lf[b] + (m - mv), -64.0f);
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t hw[16], lw[16];
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const float2 f2 = make_float2(fk[2 * c + b], fk[2 * c + b]), nm = make_float2(lf[2 * c + b] - m, lf[2 * c + b] - m);
                            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const int k = 16 * b + i;
                                float2 y = __ffma2_rn(make_float2(__uint_as_float(x[c][k]), __uint_as_float(x[c][k + 1])), f2, nm);
                                if (!CLEAR) {
                                    y.x = seen[c] >> k & 1u ? y.x : -INFINITY;
                                    y.y = seen[c] >> (k + 1) & 1u ? y.y : -INFINITY;
                                }
                                const float2 v = make_float2(kv_ex2(y.x), kv_ex2(y.y));
                                sum = __fadd2_rn(sum, v);
                                kv_split(v.x, v.y, hw[k / 2], lw[k / 2]);
                            }
                            l = fmaf(sum.x + sum.y, kv_ex2(-lf[2 * c + b]), l);
                        }
                        tc_st(s_t + 16 * c, hw);
                        tc_st(s_t + 32 + 16 * c, lw);
                    }
                }
            };
            // (o_done has two places as well: a warp can be done with a tile before the product of the one before is, and a parity tells two
            // phases apart; the scores of a tile are there only when the product of two tiles before is done)
            for (int s = it.s0; s < it.s1 && ok; s++, n++, nw++) {
                const int st = n % STAGES, key0 = (it.first + s) * KT;
                // (the scores first: behind them the tile's barrier is in the phase asked for, whatever tiles this group has skipped)
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(sf + 8 * (2 * w + (nw & 1)), (nw >> 1) & 1) && mbar_wait_fast(full + 8 * st, (n / STAGES) & 1));
                if (!ok) break;
                tc_fence_after();
                const bool first = ((s - it.s0) & (chain - 1)) == 0;
                if (first && s > it.s0) {
                    drain_sums(s - it.s0 > chain);
                    if (!ok) break;
                }
                const int2 *sub = sub_info[st];
                const int4 i0 = *reinterpret_cast<const int4 *>(sub), i1 = *reinterpret_cast<const int4 *>(sub + 2);
                if (__all_sync(0xFFFFFFFFu, pos - key0 >= KT - 1 && low <= key0 && (i0.x | i0.z | i1.x | i1.z) >= 0)) tile(std::true_type(), sub, key0, first);
                else tile(std::false_type(), sub, key0, first);
            }
            if (!ok) break;
            hand_over(nw - 1);
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(of + 8 * (2 * w + ((nw - 1) & 1)), ((nw - 1) >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const bool whole = it.s0 == 0 && it.s1 == it.steps, mine = w * 128 + me < it.vecs, none = !(thr > -INFINITY) && l == 0.0f, drained = it.s1 - it.s0 > chain;
            if (whole) {
                const float h = exp2f(0.5f * (mv - m)), inv = none ? 0.0f : Codes::unscale / l;   // (in two halves as in kv_attn.cu)
                const int64_t to = (int64_t)(it.row0 + row) * a.y_ld + (int64_t)qhead * D;
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(o_t + 32 * c, x);
                    if (!mine) continue;
                    if (drained) join_sums(c, x);
                    float y[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) y[i] = none ? 0.0f : __uint_as_float(x[i]) * inv * h * h;
                    if (a.y_dt == NNQ_F32) {
                        float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.y) + to + 32 * c);
#pragma unroll
                        for (int i = 0; i < 8; i++) p[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    } else {
                        uint4 *p = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(a.y) + to + 32 * c);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            p[i] = make_uint4(pack_bf16(y[8 * i], y[8 * i + 1]), pack_bf16(y[8 * i + 2], y[8 * i + 3]), pack_bf16(y[8 * i + 4], y[8 * i + 5]), pack_bf16(y[8 * i + 6], y[8 * i + 7]));
                    }
                }
            } else {
                if (mine) rec[0] = make_float4(none ? -INFINITY : thr > -INFINITY ? m : l, mv, l, 0.0f);   // (l: scores that are all NaN)
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(o_t + 32 * c, x);
                    if (!mine) continue;
                    if (drained) join_sums(c, x);
                    keep_sums(c, x);
                }
            }
            tc_fence_before();
        }
    } else if (warp < 16) {
        // ---------------- codes to f16 tiles ----------------
        tc_registers<64>();
        // Thread pt has 16 dimensions of every 64 of key pt / 4: four lanes read 64 bytes of a key, eight store to different banks.
        const int pt = tid - 256, key_of = pt >> 2, c4 = pt & 3;
        const uint32_t at_lo = swz(key_of, 2 * c4), at_hi = swz(key_of, 2 * c4 + 1);
        while (ok && walk.next(it)) {
            const int32_t *table = a.table + (int64_t)it.r * a.table_ld;
            uint4 k[ATOMS], v[ATOMS];
            int2 info = make_int2(-1, 127);
            int blk, info_blk;   // of the next tile: this thread's key's, and (threads 0 .. SUBS - 1) that of 16 keys
            // keys in front of what the first row sees and behind the last row are not looked for (their blocks may have been given back), by 16
            const int base = it.length - it.rows, lo = row_first(a, base + it.vec0 / a.group) & ~15, hi = base + (it.vec0 + it.vecs - 1) / a.group;
            auto blocks = [&](int s) {
                const int key0 = (it.first + s) * KT, key = key0 + key_of, key16 = key0 + 16 * pt;
                blk = s < it.s1 && key >= lo && key <= hi ? table[key >> a.shift] : kTcNone;
                info_blk = pt < SUBS && s < it.s1 && key16 >= lo && key16 <= hi ? table[key16 >> a.shift] : kTcNone;
            };
            auto load = [&](int s) {
                const bool there = blk >= 0 && blk < a.blocks;
                if (!there && blk != kTcNone) atomicExch(a.status, kStatusIndex);
                const int64_t at = ((((int64_t)blk * a.kv_heads + it.head) << a.shift) + (((it.first + s) * KT + key_of) & ((1 << a.shift) - 1))) * D + c4 * 16;
#pragma unroll
                for (int i = 0; i < ATOMS; i++) {
                    k[i] = there ? __ldg(reinterpret_cast<const uint4 *>(a.k + at + 64 * i)) : make_uint4(0, 0, 0, 0);
                    v[i] = there ? __ldg(reinterpret_cast<const uint4 *>(a.v + at + 64 * i)) : make_uint4(0, 0, 0, 0);
                }
                const int64_t bh = (int64_t)info_blk * a.kv_heads + it.head;
                info = info_blk >= 0 && info_blk < a.blocks ? make_int2(a.k_exp[bh], a.v_exp[bh]) : make_int2(-1, 127);
            };
            auto store = [&](uint8_t *dst, const uint4 &x) {
                uint4 lo, hi;
                Codes::four(x.x, lo.x, lo.y);
                Codes::four(x.y, lo.z, lo.w);
                Codes::four(x.z, hi.x, hi.y);
                Codes::four(x.w, hi.z, hi.w);
                *reinterpret_cast<uint4 *>(dst + at_lo) = lo;
                *reinterpret_cast<uint4 *>(dst + at_hi) = hi;
            };
            blocks(it.s0);
            load(it.s0);
            blocks(it.s0 + 1);
            for (int s = it.s0; s < it.s1; s++, n++) {
                const int st = n % STAGES;
                if (n >= STAGES) ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty + 8 * st, (n / STAGES - 1) & 1));
                if (!ok) break;
                uint8_t *k_s = stages + st * Sh::stage, *v_s = k_s + ATOMS * Sh::k_atom;
#pragma unroll
                for (int i = 0; i < ATOMS; i++) {
                    store(k_s + i * Sh::k_atom, k[i]);
                    store(v_s + i * Sh::k_atom, v[i]);
                }
                if (pt < SUBS) sub_info[st][pt] = info;
                if (s + 1 < it.s1) load(s + 1);
                fence_async_smem();
                __syncwarp();
                if (elect_one()) mbar_arrive(full + 8 * st);
                blocks(s + 2);
            }
        }
    } else {
        tc_registers<48>();
        if (warp < 18) {
            // ---------------- MMA issuers (a warp waits together, one lane issues) ----------------
            const int w = warp - 16;
            const uint32_t id_s = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((128u >> 4) << 24);                 // both operands f16
            const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);     // B is MN-major
            const uint32_t qa = smem_u32(smem + w * T * ATOMS * Sh::q_atom), o_t = tmem + 256 * w;
            int nw = 0, items = 0;
            TcJoin join = {-1, 0, 0, 0, 0, {0, 0, 0}};
            auto wait = [&](uint32_t bar, int count) {
                ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_fast(bar, count & 1));
                return ok;
            };
            while (ok && walk.next(it)) {
                const int steps = it.s1 - it.s0;
                if (it.s0 > 0 && it.s1 == it.steps) join = {(int)((plan.begin - it.s0) / plan.chunk), it.vecs, it.row0 + it.vec0 / a.group, it.head * a.group, it.vec0 % a.group, {0, 0, 0}};
                if (w * 128 >= it.vecs) {   // nothing for the second group: its word for the stages alone
                    for (int s = 0; s < steps && ok; s++, n++)
                        if (wait(full + 8 * (n % STAGES), n / STAGES) && lane == 0) mbar_arrive(empty + 8 * (n % STAGES));
                    continue;
                }
                wait(qf + 8 * w, items++);
                for (int s = -1; s < steps && ok; s++) {
                    if (s + 1 < steps) {   // the next tile's scores
                        const int st = (n + s + 1) % STAGES, place = (nw + 1 + s) & 1;
                        if (!wait(full + 8 * st, (n + s + 1) / STAGES)) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t ka = smem_u32(stages + st * Sh::stage);
    #pragma unroll
                            for (int x = T - 1; x >= 0; x--)   // the small products first, so that their sums are rounded at their size
    #pragma unroll
                                for (int i = 0; i < ATOMS; i++) {
                                    const uint64_t dq = smem_desc(qa + (x * ATOMS + i) * Sh::q_atom), dk = smem_desc(ka + i * Sh::k_atom);
    #pragma unroll
                                    for (int k = 0; k < 4; k++) umma_bf16(o_t + 128 + 64 * place, dq + 2 * k, dk + 2 * k, id_s, x < T - 1 || (i | k) != 0);
                                }
                            umma_commit(sf + 8 * (2 * w + place));
                        }
                        __syncwarp();
                    }
                    if (s < 0) continue;
                    const int st = (n + s) % STAGES, place = (nw + s) & 1;
                    if (!wait(pf + 8 * (2 * w + place), (nw + s) >> 1)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t va = smem_u32(stages + st * Sh::stage) + ATOMS * Sh::k_atom, pa = o_t + 128 + 64 * place;
                        const uint64_t dv = tc_desc_mn(va, Sh::k_atom);
    #pragma unroll
                        for (int x = 1; x >= 0; x--)
    #pragma unroll
                            for (int k = 0; k < KT / 16; k++) umma_ts(o_t, pa + 32 * x + 8 * k, dv + (2048 >> 4) * k, id_o, (s & (chain - 1)) != 0 || x == 0 || k != 0);
                        umma_commit(of + 8 * (2 * w + place));
                        umma_commit(empty + 8 * st);
                    }
                    __syncwarp();
                }
                n += steps;
                nw += steps;
            }
            if (w == 0 && lane == 0) joins[blockIdx.x] = join;
            // MMAs that were issued may still read shared memory and write tensor memory
            if (elect_one()) umma_commit(drain + 8 * w);
            __syncwarp();
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(drain + 8 * w, 0)) && ok;
        }
    }
    if (!ok && lane == 0) atomicExch(a.status, 1);
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the records of the items that were cut: CTA (part that the item ends in, some dimensions). A thread has a vector.
__global__ void __launch_bounds__(kTcCols) kv_tc_join_kernel(const KvAttn a, const float *records, const TcJoin *joins, float unscale) {
    pdl_prologue();
    const TcJoin j = joins[blockIdx.x];
    const int first = j.first, last = blockIdx.x, v = threadIdx.x;
    if (first < 0 || v >= j.vecs) return;
    const int64_t rec_floats = tc_record_floats(a.dim);
    auto record = [&](int p) { return reinterpret_cast<const float4 *>(records + ((int64_t)p * 2 + (p == first ? 1 : 0)) * rec_floats); };
    float mm = -INFINITY, mv = -INFINITY;
    for (int p = first; p <= last; p++) {
        const float4 h = record(p)[v];
        if (h.x == -INFINITY) continue;
        mm = fmaxf(mm, h.x);
        mv = fmaxf(mv, h.y);
    }
    constexpr int Q = 4;   // quadruples of dimensions at a time
    const int vec = j.rest + v, row = vec / a.group, quads = a.dim / 4, q0 = blockIdx.y * Q;
    float4 o[Q];
#pragma unroll
    for (int q = 0; q < Q; q++) o[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    for (int p = first; p <= last; p++) {
        const float4 h = record(p)[v];
        if (h.x == -INFINITY) continue;
        l += h.z * exp2f(h.x - mm);
        const float f = exp2f(h.y - mv);
        float4 x[Q];
#pragma unroll
        for (int q = 0; q < Q; q++) x[q] = record(p)[kTcCols * (1 + min(q0 + q, quads - 1)) + v];
#pragma unroll
        for (int q = 0; q < Q; q++) {
            o[q].x += x[q].x * f;
            o[q].y += x[q].y * f;
            o[q].z += x[q].z * f;
            o[q].w += x[q].w * f;
        }
    }
    const int64_t to = (int64_t)(j.row + row) * a.y_ld + (int64_t)(j.head + vec - row * a.group) * a.dim;
    const float inv = l == 0.0f ? 0.0f : unscale / l, h = l == 0.0f ? 0.0f : exp2f(0.5f * (mv - mm));   // (l is NaN where only NaN scores came)
#pragma unroll
    for (int q = 0; q < Q; q++) {
        if (q0 + q >= quads) break;
        const float4 y = make_float4(o[q].x * inv * h * h, o[q].y * inv * h * h, o[q].z * inv * h * h, o[q].w * inv * h * h);
        if (a.y_dt == NNQ_F32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.y) + to + 4 * (q0 + q)) = y;
        else *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.y) + to + 4 * (q0 + q)) = make_uint2(pack_bf16(y.x, y.y), pack_bf16(y.z, y.w));
    }
}

bool kv_attn_tc_supported(int dim) { return dim == 64 || dim == 128; }
static size_t tc_records_bytes(nnq_ctx *ctx, int dim) { return (size_t)ctx->sm_count * 2 * tc_record_floats(dim) * 4; }
size_t kv_attn_tc_workspace(nnq_ctx *ctx, int dim) { return tc_records_bytes(ctx, dim) + ctx->sm_count * sizeof(TcJoin); }

template <int FMT, int D, int T>
static nnq_status launch_tc(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    constexpr int smem = TcShared<D, T>::bytes;
    static std::atomic<uint64_t> done;
    nnq_status s = allow_smem(ctx, kv_attn_tc_kernel<FMT, D, T>, smem, done);
    if (s != NNQ_OK) return s;
    TcJoin *joins = reinterpret_cast<TcJoin *>(reinterpret_cast<uint8_t *>(records) + tc_records_bytes(ctx, D));
    launch_pdl_smem(kv_attn_tc_kernel<FMT, D, T>, dim3(ctx->sm_count), dim3(kTcThreads), smem, st, a, records, joins);
    launch_pdl(kv_tc_join_kernel, dim3(ctx->sm_count, D / 16), dim3(kTcCols), st, a, records, joins, CodePairs<FMT>::unscale);
    ctx->launches += 2;
    return check_cuda(ctx, cudaGetLastError(), "cache attention launch");
}

nnq_status launch_kv_attn_tc(nnq_ctx *ctx, const KvAttn &a, int fmt, float *records, cudaStream_t st) {
    const bool one = a.q_dt == NNQ_BF16 && a.y_dt == NNQ_BF16;
    if (fmt == NNQ_KV_INT8) {
        if (a.dim == 64) return one ? launch_tc<NNQ_KV_INT8, 64, 1>(ctx, a, records, st) : launch_tc<NNQ_KV_INT8, 64, 2>(ctx, a, records, st);
        return one ? launch_tc<NNQ_KV_INT8, 128, 1>(ctx, a, records, st) : launch_tc<NNQ_KV_INT8, 128, 2>(ctx, a, records, st);
    }
    if (a.dim == 64) return one ? launch_tc<NNQ_KV_E4M3, 64, 1>(ctx, a, records, st) : launch_tc<NNQ_KV_E4M3, 64, 2>(ctx, a, records, st);
    return one ? launch_tc<NNQ_KV_E4M3, 128, 1>(ctx, a, records, st) : launch_tc<NNQ_KV_E4M3, 128, 2>(ctx, a, records, st);
}

}  // namespace nnq
