// Attention over the paged 8-bit cache (kv_cache.cuh) for many query vectors per key / value head -- prompts and their portions -- on
// the 5th-generation tensor cores: heads of 64 and 128.
//
// One CTA has up to 256 query vectors of one key / value head (consecutive (row, query head of the group) pairs), 128 for each of two
// softmax groups, and walks over tiles of keys that both share.
//   warps 0-3, 4-7: softmax. Thread r of a group owns query vector r: its scores from tensor memory, maximum and sum; the weights go back
//                   into the columns of the scores as f16, where the second product reads them. The weighted values of all tiles
//                   add up in tensor memory; a reference moves only when a score passes it by 2^8, and then the sums there are scaled.
//   warps 8-11:     codes from the blocks of the table to f16 tiles in shared memory, swizzled as the products read them, keys and values
//                   as they lie (the values are the MN-major operand); the next tile's codes are under way meanwhile.
//   warp 12:        one lane issues the MMAs: S(t + 1) of a group right behind its O += P(t) V(t). MMAs run in the order they are issued,
//                   so the scores may overwrite the weights in front of them.
// While one group is at its softmax, the other's products run. Codes are exact in f16. T = 1 (bf16 queries and outputs): a query vector is
// exact under its power of two, a weight is one f16 number, off by up to 2^-11 of itself where the output's own rounding is 2^-8 of it. T = 2 (f32
// on either side): both have two terms, 22 bits.
// Scales: a block's key exponent multiplies its scores in f32. Its value exponent enters the weight, w = p 2^(m - mv + e_v) with a
// reference mv of its own, the largest score + e_v as m is that of the scores: one factor per vector and 16 keys, and weights
// between 0 and 2^8 whatever the scales are.
//
// Work: the key tiles of all (request, head, 256 vectors) items in one row, cut into equal parts, one per SM: causal rows and
// long contexts load all SMs alike. An item inside a part is written directly, of one that is cut every part leaves a record, and
// kv_tc_join_kernel joins them in order.
#include <algorithm>

#include "kv_attn.cuh"
#include "tcgen05.cuh"

namespace nnq {

constexpr int kTcCols = 256, kTcThreads = 13 * 32, kTcStages = 2, kTcMinSteps = 4;
constexpr float kTcLog2E = 1.4426950408889634f, kTcSlack = 8.0f;

// keys of a tile: 128, 64 where the queries' second terms take the room
template <int T>
struct TcTile {
    static constexpr int keys = T == 1 ? 128 : 64;
};

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
    if (k.rows * a.group > a.few) q.cbs = (k.rows * a.group + kTcCols - 1) / kTcCols;
    return q;
}
template <int KT>
__device__ __forceinline__ void tc_range(const KvAttn &a, const TcRequest &q, int cb, int &first, int &steps) {
    const int base = q.length - q.rows, r0 = base + cb * kTcCols / a.group, r1 = base + (min((cb + 1) * kTcCols, q.rows * a.group) - 1) / a.group;
    const int lo = a.window > 0 ? max(r0 - a.window + 1, 0) : 0;
    first = r1 < 0 ? 0 : lo / KT;
    steps = r1 < 0 ? 1 : r1 / KT - first + 1;
}
// tiles of one head of a request, by a whole warp
template <int KT>
__device__ __forceinline__ int tc_head_steps(const KvAttn &a, const TcRequest &q) {
    int n = 0;
    for (int cb = threadIdx.x & 31; cb < q.cbs; cb += 32) {
        int f, s;
        tc_range<KT>(a, q, cb, f, s);
        n += s;
    }
    return __reduce_add_sync(0xFFFFFFFFu, n);
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
            const int n = tc_head_steps<KT>(a, o);
            if (lane == src) mine = (int64_t)n * a.kv_heads;
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
        const int per_head = tc_head_steps<KT>(a, q);
        const int64_t off = sums[32];
        const int head = (int)(off / per_head);
        int rest = (int)(off - (int64_t)head * per_head), sum = 0;
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
                found[3] = rest - (sum + x - s);
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

template <int D, int T>
struct TcShared {
    static constexpr int KT = TcTile<T>::keys, atoms = D / 64;
    static constexpr int q_atom = 128 * 128, k_atom = KT * 128;
    static constexpr int q_bytes = 2 * T * atoms * q_atom, stage = 2 * atoms * k_atom;
    static constexpr int bytes = 1024 + q_bytes + kTcStages * stage;
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
__device__ __forceinline__ void group_sync(int w) { asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory"); }

template <int FMT, int D, int T>
__global__ void __launch_bounds__(kTcThreads, 1) kv_attn_tc_kernel(const KvAttn a, float *records) {
    typedef TcShared<D, T> Sh;
    typedef CodePairs<FMT> Codes;
    constexpr int KT = Sh::KT, ATOMS = Sh::atoms, SUBS = KT / 16;
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    uint8_t *smem = tc_smem_raw + (-smem_u32(tc_smem_raw) & 1023u);
    __shared__ __align__(8) uint64_t bars[2 * kTcStages + 9];   // full, empty; q_full, s_full, p_full, o_done of two groups; drain
    __shared__ int2 sub_info[kTcStages][SUBS];                  // exponent bytes of keys and values of every 16 keys; x < 0: unseen
    __shared__ float q_un[2][128];
    __shared__ uint32_t tmem_s;
    __shared__ int found[4];
    __shared__ int64_t sums[33];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t full = smem_u32(bars), empty = full + 8 * kTcStages, qf = empty + 8 * kTcStages, sf = qf + 16, pf = sf + 16, of = pf + 16, drain = of + 16;
    pdl_prologue();
    const TcPlan plan = tc_plan<KT>(a, gridDim.x, found, sums);
    if (plan.begin >= plan.end) return;
    if (tid == 0) {
        for (int i = 0; i < kTcStages; i++) {
            mbar_init(full + 8 * i, 4);
            mbar_init(empty + 8 * i, 1);
        }
        for (int w = 0; w < 2; w++) {
            mbar_init(qf + 8 * w, 1);
            mbar_init(sf + 8 * w, 1);
            mbar_init(pf + 8 * w, 4);
            mbar_init(of + 8 * w, 1);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_s, 0);   // of group w: O at 256 w, S and P at 256 w + 128
    uint8_t *stages = smem + Sh::q_bytes;
    bool ok = true;
    TcWalk<KT> walk(a, plan, found);
    TcItem it;
    int n = 0;   // tiles so far

    if (warp < 8) {
        // ---------------- softmax ----------------
        const int w = warp >> 2, me = tid & 127;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, o_t = tmem + 256 * w + lane_base, s_t = o_t + 128;
        uint8_t *q_s = smem + w * T * ATOMS * Sh::q_atom;
        int nw = 0;   // this group's tiles
        while (ok && walk.next(it)) {
            if (w * 128 >= it.vecs) {   // nothing for the second group
                n += it.s1 - it.s0;
                continue;
            }
            {
                // the group's query vectors, a warp per vector and turn, a lane has D / 32 dimensions; the loads of a turn before its stores
                constexpr int E = D / 32, QN = 8;
                for (int v0 = warp & 3; v0 < 128; v0 += 4 * QN) {
                    float x[QN][E];
#pragma unroll
                    for (int i = 0; i < QN; i++) {
                        const int v = w * 128 + v0 + 4 * i, vec = it.vec0 + v, row = vec / a.group;
#pragma unroll
                        for (int e = 0; e < E; e++) x[i][e] = 0.0f;
                        if (v >= it.vecs) continue;
                        const int64_t at = (int64_t)(it.row0 + row) * a.q_ld + (int64_t)(it.head * a.group + vec - row * a.group) * D + lane * E;
                        if (a.q_dt == NNQ_F32) {
#pragma unroll
                            for (int e = 0; e < E; e += 2) {
                                const float2 f = __ldg(reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(a.q) + at + e));
                                x[i][e] = f.x;
                                x[i][e + 1] = f.y;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < E; e += 2) {
                                const uint32_t u = __ldg(reinterpret_cast<const uint32_t *>(reinterpret_cast<const __nv_bfloat16 *>(a.q) + at + e));
                                x[i][e] = __uint_as_float(u << 16);
                                x[i][e + 1] = __uint_as_float(u & 0xFFFF0000u);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < QN; i++) {
                        const int v = v0 + 4 * i, d = lane * E;
                        uint32_t big = 0;
#pragma unroll
                        for (int e = 0; e < E; e++) big = max(big, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
                        big = __reduce_max_sync(0xFFFFFFFFu, big);
                        const float sc = kv_top_scale(big);
                        if (lane == 0) q_un[w][v] = kv_top_unscale(big);
                        uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
                        for (int e = 0; e < E / 2; e++) kv_split(x[i][2 * e] * sc, x[i][2 * e + 1] * sc, hi[e], lo[e]);
                        uint8_t *dst = q_s + (d >> 6) * Sh::q_atom + swz(v, (d & 63) >> 3) + 2 * (d & 7);
#pragma unroll
                        for (int e = 0; e < E / 2; e++) {
                            reinterpret_cast<uint32_t *>(dst)[e] = hi[e];
                            if (T == 2) reinterpret_cast<uint32_t *>(dst + ATOMS * Sh::q_atom)[e] = lo[e];
                        }
                    }
                }
            }
            fence_async_smem();
            group_sync(w);
            if (me == 0) mbar_arrive(qf + 8 * w);
            const int vec = it.vec0 + min(w * 128 + me, it.vecs - 1), row = vec / a.group, pos = it.length - it.rows + row;
            const int low = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
            const float fac = a.scale * kTcLog2E * Codes::unscale * q_un[w][me];
            float m = 0.0f, mv = 0.0f, l = 0.0f, thr = -INFINITY, thv = -INFINITY;
            for (int s = it.s0; s < it.s1; s++, n++, nw++) {
                const int st = n % kTcStages, key0 = (it.first + s) * KT;
                // (the scores first: behind them the tile's barrier is in the phase asked for, whatever tiles this group has skipped)
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(sf + 8 * w, nw & 1) && mbar_wait_fast(full + 8 * st, (n / kTcStages) & 1));
                if (!ok) break;
                tc_fence_after();
                const int hi = pos - key0, lo = low - key0;   // visible keys of the tile: lo .. hi
                // (in tiles that all vectors of the warp see whole, of blocks that exist, nothing is masked)
                bool there = true;
#pragma unroll
                for (int b = 0; b < SUBS; b++) there = there && sub_info[st][b].x >= 0;
                const bool clear = __all_sync(0xFFFFFFFFu, hi >= KT - 1 && lo <= 0) && there;
                auto masked = [&](int i, float x) { return clear || (i <= hi && i >= lo && sub_info[st][i >> 4].x >= 0) ? x : -INFINITY; };
                // ---- maxima: of the scores, and of scores + value exponents
                float mt = -INFINITY, vt = -INFINITY;
                uint32_t sc[T == 2 ? 64 : 32];
#pragma unroll
                for (int c = 0; c < KT / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(s_t + 32 * c, x);
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const int2 info = sub_info[st][2 * c + b];
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            t0 = fmaxf(t0, masked(32 * c + 16 * b + i, __uint_as_float(x[16 * b + i])));
                            t1 = fmaxf(t1, masked(32 * c + 16 * b + i + 1, __uint_as_float(x[16 * b + i + 1])));
                        }
                        float t = fmaxf(t0, t1);
                        if (t > -INFINITY) t *= fac * pow2_byte(info.x);   // (the factor can be zero)
                        mt = fmaxf(mt, t);
                        vt = fmaxf(vt, t + (float)(info.y - 127));
                    }
                    if (T == 2) {
#pragma unroll
                        for (int i = 0; i < 32; i++) sc[32 * (c & 1) + i] = x[i];
                    }
                }
                // ---- references
                const bool moves = mt > thr || vt > thv;
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    float f = 1.0f;
                    if (moves) {
                        const bool none = thr == -INFINITY;   // a first reference: the sums are zero
                        const float mn = none ? mt : fmaxf(m, mt), vn = none ? vt : fmaxf(mv, vt);
                        if (!none) {
                            l *= exp2f(m - mn);
                            f = exp2f(mv - vn);
                        }
                        m = mn;
                        mv = vn;
                        thr = mn + kTcSlack;
                        thv = vn + kTcSlack;
                    }
                    if (s > it.s0 && __any_sync(0xFFFFFFFFu, f != 1.0f)) {
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(of + 8 * w, (nw - 1) & 1));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t x[32], y[16];
                            tmem_ld32(o_t + 32 * c, x);
#pragma unroll
                            for (int h = 0; h < 2; h++) {
#pragma unroll
                                for (int i = 0; i < 16; i++) y[i] = __float_as_uint(__uint_as_float(x[16 * h + i]) * f);
                                tc_st(o_t + 32 * c + 16 * h, y);
                            }
                        }
                    }
                }
                // ---- weights
                float2 sum = make_float2(0.0f, 0.0f);
                const float2 nm = make_float2(-m, -m);
#pragma unroll
                for (int c = 0; c < KT / 32; c++) {
                    uint32_t x[32], h[16], lw[16];
                    if (T == 2) {
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] = sc[32 * (c & 1) + i];
                    } else {
                        tmem_ld32(s_t + 32 * c, x);
                    }
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const int2 info = sub_info[st][2 * c + b];
                        const float fk = fac * pow2_byte(max(info.x, 0)), fv = kv_ex2(m - mv + (float)(info.y - 127));
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const int k = 32 * c + 16 * b + i;
                            const float2 y = __ffma2_rn(make_float2(__uint_as_float(x[16 * b + i]), __uint_as_float(x[16 * b + i + 1])), make_float2(fk, fk), nm);
                            const float2 p = make_float2(kv_ex2(masked(k, y.x)), kv_ex2(masked(k + 1, y.y)));
                            sum = __fadd2_rn(sum, p);
                            const float2 v = __fmul2_rn(p, make_float2(fv, fv));
                            if (T == 2) kv_split(v.x, v.y, h[8 * b + i / 2], lw[8 * b + i / 2]);
                            else h[8 * b + i / 2] = half_bits(__floats2half2_rn(v.x, v.y));
                        }
                    }
                    tc_st(s_t + 16 * c, h);
                    if (T == 2) tc_st(s_t + 32 + 16 * c, lw);
                }
                l += sum.x + sum.y;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (elect_one()) mbar_arrive(pf + 8 * w);
            }
            if (!ok) break;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(of + 8 * w, (nw - 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const bool whole = it.s0 == 0 && it.s1 == it.steps, mine = w * 128 + me < it.vecs, none = !(thr > -INFINITY) && l == 0.0f;
            if (whole) {
                const float inv = none ? 0.0f : exp2f(mv - m) * Codes::unscale / l;
                const int64_t to = (int64_t)(it.row0 + row) * a.y_ld + (int64_t)(it.head * a.group + vec - row * a.group) * D;
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(o_t + 32 * c, x);
                    if (!mine) continue;
                    float y[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) y[i] = none ? 0.0f : __uint_as_float(x[i]) * inv;
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
                float4 *rec = reinterpret_cast<float4 *>(records + ((int64_t)blockIdx.x * 2 + (it.s0 == 0 ? 1 : 0)) * tc_record_floats(D));
                const int v = w * 128 + me;
                if (mine) rec[v] = make_float4(none ? -INFINITY : thr > -INFINITY ? m : l, mv, l, 0.0f);   // (l: scores that are all NaN)
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(o_t + 32 * c, x);
                    if (!mine) continue;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        rec[kTcCols * (1 + 8 * c + i) + v] = make_float4(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1]), __uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3]));
                }
            }
            tc_fence_before();
        }
    } else if (warp < 12) {
        // ---------------- codes to f16 tiles ----------------
        constexpr int CH = D / 16, PER = KT * CH / 128;   // 16-byte chunks of a row, chunks of a thread
        const int pt = tid - 256;
        while (ok && walk.next(it)) {
            const int32_t *table = a.table + (int64_t)it.r * a.table_ld;
            uint4 k[PER], v[PER];
            int2 info = make_int2(-1, 0);
            auto block_at = [&](int key) -> int {
                if (key >= it.length) return -1;
                const int b = table[key >> a.shift];
                if (b >= 0 && b < a.blocks) return b;
                atomicExch(a.status, kStatusIndex);
                return -1;
            };
            auto load = [&](int s) {
                const int key0 = (it.first + s) * KT;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int u = pt + 128 * i, key = key0 + u / CH, c = u % CH, b = block_at(key);
                    k[i] = v[i] = make_uint4(0, 0, 0, 0);
                    if (b >= 0) {
                        const int64_t at = ((((int64_t)b * a.kv_heads + it.head) << a.shift) + (key & ((1 << a.shift) - 1))) * D + c * 16;
                        k[i] = __ldg(reinterpret_cast<const uint4 *>(a.k + at));
                        v[i] = __ldg(reinterpret_cast<const uint4 *>(a.v + at));
                    }
                }
                if (pt < SUBS) {
                    const int b = block_at(key0 + 16 * pt);
                    const int64_t bh = (int64_t)b * a.kv_heads + it.head;
                    info = b >= 0 ? make_int2(a.k_exp[bh], a.v_exp[bh]) : make_int2(-1, 127);
                }
            };
            load(it.s0);
            for (int s = it.s0; s < it.s1; s++, n++) {
                const int st = n % kTcStages;
                if (n >= kTcStages) ok = __all_sync(0xFFFFFFFFu, mbar_wait_fast(empty + 8 * st, (n / kTcStages - 1) & 1));
                if (!ok) break;
                uint8_t *k_s = stages + st * Sh::stage, *v_s = k_s + ATOMS * Sh::k_atom;
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int u = pt + 128 * i, key = u / CH, c = u % CH, flip = (c >> 2) & 1;   // (neighbours of two pieces store their halves in turn: no bank twice)
                    const uint32_t kw[4] = {Codes::word(k[i].x), Codes::word(k[i].y), Codes::word(k[i].z), Codes::word(k[i].w)};
                    const uint32_t vw[4] = {Codes::word(v[i].x), Codes::word(v[i].y), Codes::word(v[i].z), Codes::word(v[i].w)};
                    const int at = (c >> 2) * Sh::k_atom, c8 = (c & 3) * 2;
                    const uint4 k0 = make_uint4(Codes::low(kw[0]), Codes::high(kw[0]), Codes::low(kw[1]), Codes::high(kw[1])), k1 = make_uint4(Codes::low(kw[2]), Codes::high(kw[2]), Codes::low(kw[3]), Codes::high(kw[3]));
                    const uint4 v0 = make_uint4(Codes::low(vw[0]), Codes::high(vw[0]), Codes::low(vw[1]), Codes::high(vw[1])), v1 = make_uint4(Codes::low(vw[2]), Codes::high(vw[2]), Codes::low(vw[3]), Codes::high(vw[3]));
                    *reinterpret_cast<uint4 *>(k_s + at + swz(key, c8 + flip)) = flip ? k1 : k0;
                    *reinterpret_cast<uint4 *>(k_s + at + swz(key, c8 + 1 - flip)) = flip ? k0 : k1;
                    *reinterpret_cast<uint4 *>(v_s + at + swz(key, c8 + flip)) = flip ? v1 : v0;
                    *reinterpret_cast<uint4 *>(v_s + at + swz(key, c8 + 1 - flip)) = flip ? v0 : v1;
                }
                if (pt < SUBS) sub_info[st][pt] = info;
                fence_async_smem();
                __syncwarp();
                if (elect_one()) mbar_arrive(full + 8 * st);
                if (s + 1 < it.s1) load(s + 1);
            }
        }
    } else {
        // ---------------- MMA issuer (the warp waits together, one lane issues) ----------------
        const uint32_t id_s = (1u << 4) | ((uint32_t)(KT >> 3) << 17) | ((128u >> 4) << 24);                 // both operands f16
        const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);     // B is MN-major
        int nw[2] = {0, 0}, items[2] = {0, 0};
        auto wait = [&](uint32_t bar, int count) {
            ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_fast(bar, count & 1));
            return ok;
        };
        auto scores = [&](int w, int st) {
            if (elect_one()) {
                const uint32_t qa = smem_u32(smem + w * T * ATOMS * Sh::q_atom), ka = smem_u32(stages + st * Sh::stage);
#pragma unroll
                for (int x = T - 1; x >= 0; x--)   // the small products first, so that their sums are rounded at their size
#pragma unroll
                    for (int at = 0; at < ATOMS; at++) {
                        const uint64_t dq = smem_desc(qa + (x * ATOMS + at) * Sh::q_atom), dk = smem_desc(ka + at * Sh::k_atom);
#pragma unroll
                        for (int k = 0; k < 4; k++) umma_bf16(tmem + 256 * w + 128, dq + 2 * k, dk + 2 * k, id_s, x < T - 1 || (at | k) != 0);
                    }
                umma_commit(sf + 8 * w);
            }
            __syncwarp();
        };
        while (ok && walk.next(it)) {
            const int groups = it.vecs > 128 ? 2 : 1, steps = it.s1 - it.s0;
            for (int w = 0; w < groups; w++) wait(qf + 8 * w, items[w]++);
            if (!wait(full + 8 * (n % kTcStages), n / kTcStages)) break;
            tc_fence_after();
            for (int w = 0; w < groups; w++) scores(w, n % kTcStages);
            for (int s = 0; s < steps && ok; s++, n++) {
                const int st = n % kTcStages, st1 = (n + 1) % kTcStages;
                for (int w = 0; w < groups; w++) {
                    if (!wait(pf + 8 * w, nw[w]++)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t va = smem_u32(stages + st * Sh::stage + ATOMS * Sh::k_atom), pa = tmem + 256 * w + 128;
                        const uint64_t dv = tc_desc_mn(va, Sh::k_atom);
#pragma unroll
                        for (int x = T - 1; x >= 0; x--)
#pragma unroll
                            for (int k = 0; k < KT / 16; k++) umma_ts(tmem + 256 * w, pa + 32 * x + 8 * k, dv + (2048 >> 4) * k, id_o, s > 0 || x < T - 1 || k != 0);
                        umma_commit(of + 8 * w);
                        if (w == groups - 1) umma_commit(empty + 8 * st);
                    }
                    __syncwarp();
                    if (s + 1 < steps) {
                        if (w == 0 && !wait(full + 8 * st1, (n + 1) / kTcStages)) break;
                        tc_fence_after();
                        scores(w, st1);
                    }
                }
            }
        }
        // MMAs that were issued may still read shared memory and write tensor memory
        if (elect_one()) umma_commit(drain);
        __syncwarp();
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(drain, 0)) && ok;
    }
    if (!ok && lane == 0) atomicExch(a.status, 1);
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the records of the items that were cut: CTA (part, some dimensions) where the item at the part's beginning began before it
// and ends in it. A thread has a vector.
template <int KT>
__global__ void __launch_bounds__(kTcCols) kv_tc_join_kernel(const KvAttn a, const float *records, float unscale) {
    __shared__ int found[4];
    __shared__ int64_t sums[33];
    pdl_prologue();
    const TcPlan plan = tc_plan<KT>(a, gridDim.x, found, sums);
    TcItem it;
    TcWalk<KT> walk(a, plan, found);
    if (!walk.next(it) || it.s0 == 0 || it.s1 < it.steps) return;
    const int first = (int)((plan.begin - it.s0) / plan.chunk), v = threadIdx.x;   // the part that the item begins in
    if (v >= it.vecs) return;
    const int64_t rec_floats = tc_record_floats(a.dim);
    auto record = [&](int p) { return reinterpret_cast<const float4 *>(records + ((int64_t)p * 2 + (p == first ? 1 : 0)) * rec_floats); };
    float mm = -INFINITY, mv = -INFINITY;
    for (int p = first; p <= (int)blockIdx.x; p++) {
        const float4 h = record(p)[v];
        if (h.x == -INFINITY) continue;
        mm = fmaxf(mm, h.x);
        mv = fmaxf(mv, h.y);
    }
    float l = 0.0f;
    for (int p = first; p <= (int)blockIdx.x; p++) {
        const float4 h = record(p)[v];
        if (h.x == -INFINITY) continue;
        l += h.z * exp2f(h.x - mm);
    }
    const int vec = it.vec0 + v, row = vec / a.group, quads = a.dim / 4, per = (quads + gridDim.y - 1) / gridDim.y;
    const int64_t to = (int64_t)(it.row0 + row) * a.y_ld + (int64_t)(it.head * a.group + vec - row * a.group) * a.dim;
    const float inv = mm == -INFINITY && l == 0.0f ? 0.0f : exp2f(mv - mm) * unscale / l;   // (l is NaN where only NaN scores came)
    for (int q = blockIdx.y * per; q < min(quads, (int)(blockIdx.y + 1) * per); q++) {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = first; p <= (int)blockIdx.x; p++) {
            const float4 h = record(p)[v];
            if (h.x == -INFINITY) continue;
            const float f = exp2f(h.y - mv);
            const float4 x = record(p)[kTcCols * (1 + q) + v];
            o.x += x.x * f;
            o.y += x.y * f;
            o.z += x.z * f;
            o.w += x.w * f;
        }
        o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (a.y_dt == NNQ_F32) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.y) + to + 4 * q) = o;
        else *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.y) + to + 4 * q) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
    }
}

bool kv_attn_tc_supported(const KvAttn &a) { return a.dim == 64 || a.dim == 128; }
size_t kv_attn_tc_workspace(nnq_ctx *ctx, int dim) { return (size_t)ctx->sm_count * 2 * tc_record_floats(dim) * 4; }

template <int FMT, int D, int T>
static nnq_status launch_tc(nnq_ctx *ctx, const KvAttn &a, float *records, cudaStream_t st) {
    constexpr int smem = TcShared<D, T>::bytes;
    nnq_status s = check_cuda(ctx, cudaFuncSetAttribute(kv_attn_tc_kernel<FMT, D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "attention shared memory");
    if (s != NNQ_OK) return s;
    launch_pdl_smem(kv_attn_tc_kernel<FMT, D, T>, dim3(ctx->sm_count), dim3(kTcThreads), smem, st, a, records);
    launch_pdl(kv_tc_join_kernel<TcTile<T>::keys>, dim3(ctx->sm_count, 8), dim3(kTcCols), st, a, records, CodePairs<FMT>::unscale);
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
