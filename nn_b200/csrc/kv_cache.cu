// Block tables and slot maps of a batch of requests, and what writes and reads the codes of the paged 8-bit cache (kv_cache.cuh).
// The reference keeps one sequence's keys and values in f32 and doubles the buffer as it grows
// (crates/nn-core/src/layers/generation/kv_cache.rs:132).
#include <algorithm>

#include "kv_cache.cuh"
#include "tcgen05.cuh"

namespace nnq {

// ---- tables ---------------------------------------------------------------------------------------------------------------------

// One launch of one cluster: every CTA sums the counts of all requests, in portions of kTabChunk that lie in shared memory, and writes
// its share of the tables: entry i of the portion's new blocks, row i of its rows, found by bisection of the sums. The cluster meets
// between the reading of a portion and the writing, so lengths may be written where the old ones lie. Single tokens are bound by latency:
// the requests' loads, the sums, the bisection, one dependent load for a block that was there before (8 of them 2.4 us). Many rows are
// bound by the threads of one cluster, which bisect for every row: 300 requests with some 32000 rows 10.2 us, half of the issue slots of its eight
// SMs used (one CTA of 256 threads: 84 us).
constexpr int kTabChunk = 2048;

struct TableArgs {
    const int32_t *past, *count, *free_list, *skip;
    int32_t *table, *length, *row_start, *slot, *position, *used;
    int64_t requests, n_free, table_ld, rows;
    int shift;
};

// exclusive sums of two numbers over the block's threads; returns the totals
__device__ __forceinline__ longlong2 block_scan2(longlong2 &v, longlong2 *warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    longlong2 x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const long long a = __shfl_up_sync(0xFFFFFFFFu, x.x, off), b = __shfl_up_sync(0xFFFFFFFFu, x.y, off);
        if (lane >= off) {
            x.x += a;
            x.y += b;
        }
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    longlong2 before = make_longlong2(0, 0), all = make_longlong2(0, 0);
    for (int w = 0; w < nw; w++) {
        if (w == warp) before = all;
        all.x += warp_sums[w].x;
        all.y += warp_sums[w].y;
    }
    v = make_longlong2(before.x + x.x - v.x, before.y + x.y - v.y);
    return all;
}

// the last of `n` ascending sums that is not above x (sums[0] <= x)
__device__ __forceinline__ int find_sum(const long long *sums, int n, long long x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(1024) kv_tables_kernel(const TableArgs a) {
    __shared__ long long row0[kTabChunk], new0[kTabChunk];   // first row and first new block of every request of the portion
    __shared__ int held[kTabChunk];
    __shared__ longlong2 warp_sums[32];
    pdl_prologue();
    const int tid = threadIdx.x, nt = blockDim.x;
    const int64_t me = (int64_t)blockIdx.x * nt + tid, all = (int64_t)gridDim.x * nt;
    const int64_t block = (int64_t)1 << a.shift;
    const int64_t skip = a.skip ? max(*a.skip, 0) : 0;
    longlong2 done = make_longlong2(0, 0);   // rows and new blocks of the portions before
    for (int64_t r0 = 0; r0 < a.requests; r0 += kTabChunk) {
        const int n = (int)min((int64_t)kTabChunk, a.requests - r0);
        longlong2 sum = make_longlong2(0, 0);
        for (int i0 = 0; i0 < n; i0 += nt) {
            const int i = i0 + tid;
            longlong2 v = make_longlong2(0, 0);
            int64_t past = 0;
            if (i < n) {
                past = max(a.past[r0 + i], 0);
                v.x = max(a.count[r0 + i], 0);
                v.y = ((past + v.x + block - 1) >> a.shift) - ((past + block - 1) >> a.shift);
            }
            const longlong2 part = block_scan2(v, warp_sums);
            if (i < n) {
                held[i] = (int)past;
                row0[i] = sum.x + v.x;
                new0[i] = sum.y + v.y;
            }
            sum.x += part.x;
            sum.y += part.y;
        }
        __syncthreads();
        if (gridDim.x > 1) cluster_sync();
        auto count_of = [&](int i) { return (i + 1 < n ? row0[i + 1] : sum.x) - row0[i]; };
        for (int64_t i = me; i < n; i += all) {
            a.length[r0 + i] = (int32_t)min((long long)held[i] + count_of((int)i), (long long)INT32_MAX);
            a.row_start[r0 + i] = (int32_t)min(done.x + row0[i], (long long)INT32_MAX);
        }
        // the block a request's new block number j (from its first) gets
        auto fresh = [&](int i, int64_t j) {
            const int64_t at = skip + done.y + new0[i] + j;
            return at < a.n_free ? a.free_list[at] : -1;
        };
        for (int64_t e = me; e < sum.y; e += all) {
            const int i = find_sum(new0, n, e);
            const int64_t col = (((int64_t)held[i] + block - 1) >> a.shift) + e - new0[i];
            if (col < a.table_ld) a.table[(r0 + i) * a.table_ld + col] = fresh(i, e - new0[i]);
        }
        const int64_t last = min((int64_t)sum.x, a.rows - (int64_t)done.x);
        for (int64_t t = me; t < last; t += all) {
            const int i = find_sum(row0, n, t);
            const int64_t pos = held[i] + t - row0[i], col = pos >> a.shift, first = ((int64_t)held[i] + block - 1) >> a.shift;
            int64_t b = -1;
            if (col < a.table_ld) b = col < first ? a.table[(r0 + i) * a.table_ld + col] : fresh(i, col - first);
            const int64_t s = (b << a.shift) + (pos & (block - 1));
            a.slot[done.x + t] = b >= 0 && s <= INT32_MAX ? (int32_t)s : -1;
            a.position[done.x + t] = (int32_t)min(pos, (int64_t)INT32_MAX);
        }
        done.x += sum.x;
        done.y += sum.y;
        __syncthreads();   // the portion's sums have been read
    }
    for (int64_t t = done.x + me; t < a.rows; t += all) a.slot[t] = a.position[t] = -1;
    if (gridDim.x > 1) cluster_sync();   // (every CTA has read *skip)
    if (me == 0) {
        a.row_start[a.requests] = (int32_t)min(done.x, (long long)INT32_MAX);
        if (a.used) *a.used = (int32_t)min(skip + done.y, (long long)INT32_MAX);
    }
}

// ---- append ---------------------------------------------------------------------------------------------------------------------

// Rows whose slots run on inside one block are a run; its first row is the leader. A warp has `tile` rows of one head, keys or values, and
// takes the runs that are led there, wherever they end: the largest absolute value (bits compare like the numbers; non-finite ones are
// left out), the exponent byte, the codes; codes the block held before are rounded again where the exponent grew. The first pieces of
// eight values of a lane stay in registers in between.
// What bounds it is latency: the chain slot -> values -> codes, which a warp goes through alone (a CTA per run, with a barrier in it:
// 12000 rows of 8 heads of 128, bf16, blocks of 32, 43 us). Measured: those 32 us, issue slots 44 % used, most waits for loads; 48 single f32 rows
// with the read behind them 4.4 us. Large runs are slow, as one warp has them whole: 4000 rows of a prompt, 8 heads, in blocks of 16 / 64 / 256 tokens 5.7 /
// 12.7 / 33.6 us (dim 64) and 15.9 / 45.9 / 136 us (dim 256); 48 single tokens that raise the scale of a full block 2.9 / 5 / 14 us and
// 4.6 / 14 / 53 us, else 3 us.
constexpr int kAppWarps = 8;

struct AppendArgs {
    struct Part {
        const void *x;
        int64_t ld;
        uint8_t *codes, *exps;
    } keys, values;
    const int32_t *slot;
    int64_t rows, slots;
    int kv_heads, dim, shift, tile;
    int *status;
};

// eight values of a row as they lie in memory
template <bool F32>
struct Eight {
    uint4 w[F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *p, int64_t at) {
        const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p) + at * (F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (F32 ? 2 : 1); i++) w[i] = __ldg(q + i);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t *u = &w[0].x;
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __uint_as_float((i < 4 ? (&w[0].x)[i] : (&w[1].x)[i - 4]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
            }
        }
    }
};

// Codes of eight values already divided by the scale: finite ones within the range.
template <int FMT>
__device__ __forceinline__ uint2 encode_within(const float (&v)[8]) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if constexpr (FMT == NNQ_KV_INT8) {   // the integer is the low byte of the sum's bits, rounded to the nearest, ties to even
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) b[i] = __float_as_uint(v[4 * h + i] + 12582912.0f);
            w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        } else {
            uint16_t p, q;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p) : "f"(v[4 * h + 1]), "f"(v[4 * h]));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(v[4 * h + 3]), "f"(v[4 * h + 2]));
            w[h] = (uint32_t)p | (uint32_t)q << 16;
        }
    }
    return make_uint2(w[0], w[1]);
}

// A run of `n` rows from row `t` on, by a warp.
template <int FMT, bool F32>
__device__ __forceinline__ void append_run(const AppendArgs &a, const AppendArgs::Part &p, int head, int64_t t, int first, int n) {
    constexpr int KEEP = F32 ? 2 : 4;
    const int lane = threadIdx.x & 31, per = a.dim >> 3, units = n * per, magic = (65535 + per) / per;   // (exact below 8192)
    const int64_t blk = first >> a.shift;
    const int off = first & ((1 << a.shift) - 1);
    const void *x = reinterpret_cast<const uint8_t *>(p.x) + (t * p.ld + (int64_t)head * a.dim) * (F32 ? 4 : 2);
    uint8_t *codes = p.codes + (((blk * a.kv_heads + head) << a.shift) * a.dim), *exp_at = p.exps + blk * a.kv_heads + head;
    const int old = off ? min((int)*exp_at, kExpMax) : 0;
    auto at_of = [&](int u) {
        const int row = u * magic >> 16;   // u / per
        return row * p.ld + (u - row * per) * 8;
    };
    uint32_t top = 0;
    bool bad = false;
    Eight<F32> keep[KEEP];
    auto look = [&](const Eight<F32> &e) {
        float v[8];
        e.values(v);
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        if (most >= 0x7F800000u) {
            bad = true;
            most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
                if (b < 0x7F800000u) most = max(most, b);
            }
        }
        top = max(top, most);
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lane + 32 * i < units) keep[i].load(x, at_of(lane + 32 * i));
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lane + 32 * i < units) look(keep[i]);
#pragma unroll 4
    for (int u = lane + 32 * KEEP; u < units; u += 32) {
        Eight<F32> e;
        e.load(x, at_of(u));
        look(e);
    }
    if (bad) atomicExch(a.status, kStatusValue);
    const int e = max(exponent_byte<FMT>(__reduce_max_sync(0xFFFFFFFFu, top)), old);
    const float inv = pow2_byte(254 - e);
    uint8_t *to = codes + (int64_t)off * a.dim;   // (the rows of a run lie one behind the other in the block)
    auto write = [&](const Eight<F32> &q, int u) {
        float v[8];
        q.values(v);
        constexpr float most = FMT == NNQ_KV_INT8 ? 127.0f : 448.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] *= inv;
            if (bad) v[i] = v[i] == v[i] ? fminf(fmaxf(v[i], -most), most) : 0.0f;   // (some value of this lane's is not finite)
        }
        *reinterpret_cast<uint2 *>(to + (int64_t)u * 8) = encode_within<FMT>(v);
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        if (lane + 32 * i < units) write(keep[i], lane + 32 * i);
#pragma unroll 4
    for (int u = lane + 32 * KEEP; u < units; u += 32) {
        Eight<F32> q;
        q.load(x, at_of(u));
        write(q, u);
    }
    if (off && e > old) {
        const float again = pow2_byte(max(127 + old - e, 0));
        for (int u = lane; u < off * per; u += 32) {
            uint2 *at = reinterpret_cast<uint2 *>(codes) + u;
            const uint2 c = *at;
            const uint32_t in[2] = {c.x, c.y};
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = kv_decode<FMT>(in[i >> 2] >> (8 * (i & 3)) & 0xFFu) * again;   // (again is a half or less)
            *at = encode_within<FMT>(v);
        }
    }
    __syncwarp();   // every lane has read the old byte
    if (lane == 0) *exp_at = (uint8_t)e;
}

template <int FMT, bool F32>
__global__ void __launch_bounds__(kAppWarps * 32, 4) kv_append_kernel(const AppendArgs a) {
    pdl_prologue();
    const int lane = threadIdx.x & 31, heads = 2 * a.kv_heads, block = 1 << a.shift;
    const int64_t id = (int64_t)blockIdx.x * kAppWarps + (threadIdx.x >> 5), tile = id / heads, t0 = tile * a.tile;
    const int which = (int)(id - tile * heads), head = which >> 1;
    if (t0 >= a.rows) return;
    const AppendArgs::Part part = which & 1 ? a.values : a.keys;
    const int64_t t = t0 + lane;
    int s = -1, before = -1;
    if (lane < a.tile && t < a.rows) {
        s = a.slot[t];
        if (t > 0) before = a.slot[t - 1];
    }
    if (s >= a.slots) {
        atomicExch(a.status, kStatusIndex);
        s = -1;
    }
    const bool leads = s >= 0 && (before < 0 || before != s - 1 || (s & (block - 1)) == 0);
    for (uint32_t leaders = __ballot_sync(0xFFFFFFFFu, leads); leaders; leaders &= leaders - 1) {
        const int src = __ffs(leaders) - 1, first = __shfl_sync(0xFFFFFFFFu, s, src), most = block - (first & (block - 1));
        const int64_t from = t0 + src;
        int n = 0;
        for (;;) {   // rows that continue the run
            const int i = n + lane;
            const uint32_t m = __ballot_sync(0xFFFFFFFFu, i < most && from + i < a.rows && a.slot[from + i] == first + i);
            n += m == 0xFFFFFFFFu ? 32 : __ffs(~m) - 1;
            if (m != 0xFFFFFFFFu || n >= most) break;
        }
        append_run<FMT, F32>(a, part, head, from, first, n);
    }
}

// ---- read -----------------------------------------------------------------------------------------------------------------------

struct ReadArgs {
    struct Part {
        const uint8_t *codes, *exps;
        void *y;
    } keys, values;
    const int32_t *slot;
    int64_t rows, slots;
    int kv_heads, dim, shift;
    int *status;
};

// A thread has 16 values of a row: one load, two or four stores. Rows of no slot are zeros. 12000 rows of 8 heads of 128, e4m3, to bf16:
// 16.6 us (4.4 TB/s both ways), bound by the conversions: issue slots 75 % used, logic pipe 65 %. (A warp's stores leave gaps of 16 bytes
// that its next ones fill.)
template <int FMT, bool F32>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadArgs a) {
    pdl_prologue();
    const ReadArgs::Part part = blockIdx.y ? a.values : a.keys;
    const int units = a.kv_heads * (a.dim >> 4);
    const int64_t total = a.rows * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / units;
        const int u = (int)(i - row * units), head = u / (a.dim >> 4), d = (u - head * (a.dim >> 4)) * 16;
        const int s = a.slot[row];
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; k++) v[k] = 0.0f;
        if (s >= a.slots) atomicExch(a.status, kStatusIndex);
        else if (s >= 0) {
            const int64_t bh = (int64_t)(s >> a.shift) * a.kv_heads + head;
            const uint4 c = __ldg(reinterpret_cast<const uint4 *>(part.codes + ((bh << a.shift) + (s & ((1 << a.shift) - 1))) * a.dim + d));
            const float f = pow2_byte(part.exps[bh]);
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = kv_decode<FMT>(w[k >> 2] >> (8 * (k & 3)) & 0xFFu) * f;
        }
        const int64_t at = (row * a.kv_heads + head) * a.dim + d;
        if constexpr (F32) {
            float4 *y = reinterpret_cast<float4 *>(reinterpret_cast<float *>(part.y) + at);
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        } else {
            uint4 *y = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(part.y) + at);
#pragma unroll
            for (int k = 0; k < 2; k++)
                y[k] = make_uint4(pack_bf16(v[8 * k], v[8 * k + 1]), pack_bf16(v[8 * k + 2], v[8 * k + 3]), pack_bf16(v[8 * k + 4], v[8 * k + 5]), pack_bf16(v[8 * k + 6], v[8 * k + 7]));
        }
    }
}

}  // namespace nnq

using namespace nnq;

extern "C" {

nnq_status nnq_kv_tables(nnq_ctx *ctx, const int32_t *past_dev, const int32_t *count_dev, int64_t requests, const int32_t *free_dev, int64_t n_free,
                         const int32_t *skip_dev, int block, int32_t *table_dev, int64_t table_ld, int32_t *length_dev, int32_t *row_start_dev,
                         int32_t *slot_dev, int32_t *position_dev, int64_t rows, int32_t *used_dev, void *stream) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    if (requests < 1 || n_free < 0 || table_ld < 1 || rows < 0) return fail(ctx, NNQ_ERR_INVALID_ARG, "bad sizes of a batch");
    if (requests > INT32_MAX / 2 || rows > INT32_MAX) return fail(ctx, NNQ_ERR_UNSUPPORTED, "a batch of %lld requests and %lld rows", (long long)requests, (long long)rows);
    if (block < 16 || block > 256 || (block & (block - 1))) return fail(ctx, NNQ_ERR_UNSUPPORTED, "blocks must hold 16, 32, 64, 128 or 256 tokens (got %d)", block);
    if (!past_dev || !count_dev || (n_free && !free_dev) || !table_dev || !length_dev || !row_start_dev || (rows && (!slot_dev || !position_dev)))
        return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor in a batch");
    nnq_status s = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice");
    if (s != NNQ_OK) return s;
    const TableArgs a = {past_dev, count_dev, free_dev, skip_dev, table_dev, length_dev, row_start_dev, slot_dev, position_dev, used_dev, requests, n_free, table_ld, rows, log2_of(block)};
    // one CTA of 256 threads for what it does in a pass or four, else a cluster of up to 8 CTAs of 1024, one for 2048 rows (us, small / large:
    // 8 requests of a row 2.4 / 4.9, 300 requests of some 32000 rows 84 / 10.2)
    const bool small = requests <= 256 && rows <= 1024;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(small ? 256 : 1024);
    cfg.gridDim = dim3(small ? 1 : (unsigned)std::min<int64_t>(8, (std::max(rows, requests) + 2047) / 2048));
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {cfg.gridDim.x, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    s = check_cuda(ctx, cudaLaunchKernelEx(&cfg, kv_tables_kernel, a), "block tables launch");
    if (s == NNQ_OK) ctx->launches++;
    return s;
}

nnq_status nnq_kv_append(nnq_ctx *ctx, const nnq_kv_cache *c, const void *k_dev, int64_t k_ld, const void *v_dev, int64_t v_ld, nnq_dtype dt,
                         const int32_t *slot_dev, int64_t rows, void *stream) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    nnq_status s = check_kv_cache(ctx, c);
    if (s != NNQ_OK) return s;
    if (dt != NNQ_F32 && dt != NNQ_BF16) return fail(ctx, NNQ_ERR_INVALID_ARG, "unknown dtype %d", (int)dt);
    if (rows < 0 || rows > INT32_MAX) return fail(ctx, NNQ_ERR_INVALID_ARG, "%lld rows", (long long)rows);
    if (rows == 0) return NNQ_OK;
    if (!k_dev || !v_dev || !slot_dev) return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor");
    const int64_t width = (int64_t)c->kv_heads * c->dim;
    if (k_ld < width || v_ld < width) return fail(ctx, NNQ_ERR_SHAPE_MISMATCH, "rows of keys and values must be %lld wide or further apart", (long long)width);
    if (!rows_aligned(k_dev, k_ld, dt) || !rows_aligned(v_dev, v_ld, dt)) return fail(ctx, NNQ_ERR_INVALID_ARG, "rows of keys and values must start at multiples of 16 bytes");
    if ((s = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice")) != NNQ_OK) return s;
    const AppendArgs a = {{k_dev, k_ld, (uint8_t *)c->k, c->k_exp}, {v_dev, v_ld, (uint8_t *)c->v, c->v_exp}, slot_dev, rows, c->blocks * c->block, c->kv_heads, c->dim,
                          log2_of(c->block), rows > 1024 ? 16 : 1, ctx->d_status};   // (few rows are single tokens more often than not: a warp each.
                          // us with the read behind, 1 / 16 rows: 48 single tokens 4.4 / 17.6, three prompts of some 4000 rows 79 / 48; 4 / 8 rows 54 / 50)
    const int64_t warps = (rows + a.tile - 1) / a.tile * 2 * c->kv_heads;
    if (warps / kAppWarps >= INT32_MAX) return fail(ctx, NNQ_ERR_UNSUPPORTED, "%lld rows of %d heads", (long long)rows, c->kv_heads);
    const dim3 grid((unsigned)((warps + kAppWarps - 1) / kAppWarps)), block(kAppWarps * 32);
    auto kernel = c->format == NNQ_KV_INT8 ? (dt == NNQ_F32 ? kv_append_kernel<NNQ_KV_INT8, true> : kv_append_kernel<NNQ_KV_INT8, false>)
                                           : (dt == NNQ_F32 ? kv_append_kernel<NNQ_KV_E4M3, true> : kv_append_kernel<NNQ_KV_E4M3, false>);
    launch_pdl(kernel, grid, block, (cudaStream_t)stream, a);
    ctx->launches++;
    return check_cuda(ctx, cudaGetLastError(), "cache append launch");
}

nnq_status nnq_kv_read(nnq_ctx *ctx, const nnq_kv_cache *c, const int32_t *slot_dev, int64_t rows, void *k_dev, void *v_dev, nnq_dtype dt, void *stream) {
    if (!ctx) return NNQ_ERR_INVALID_ARG;
    nnq_status s = check_kv_cache(ctx, c);
    if (s != NNQ_OK) return s;
    if (dt != NNQ_F32 && dt != NNQ_BF16) return fail(ctx, NNQ_ERR_INVALID_ARG, "unknown dtype %d", (int)dt);
    if (rows < 0 || rows > INT32_MAX) return fail(ctx, NNQ_ERR_INVALID_ARG, "%lld rows", (long long)rows);
    if (rows == 0) return NNQ_OK;
    if (!k_dev || !v_dev || !slot_dev) return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor");
    if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15u) return fail(ctx, NNQ_ERR_INVALID_ARG, "outputs must be 16-byte aligned");
    if ((s = check_cuda(ctx, cudaSetDevice(ctx->device), "cudaSetDevice")) != NNQ_OK) return s;
    const ReadArgs a = {{(const uint8_t *)c->k, c->k_exp, k_dev}, {(const uint8_t *)c->v, c->v_exp, v_dev}, slot_dev, rows, c->blocks * c->block, c->kv_heads, c->dim,
                        log2_of(c->block), ctx->d_status};
    const int64_t units = rows * c->kv_heads * (c->dim >> 4);
    const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, (int64_t)8 * ctx->sm_count), 2);
    auto kernel = c->format == NNQ_KV_INT8 ? (dt == NNQ_F32 ? kv_read_kernel<NNQ_KV_INT8, true> : kv_read_kernel<NNQ_KV_INT8, false>)
                                           : (dt == NNQ_F32 ? kv_read_kernel<NNQ_KV_E4M3, true> : kv_read_kernel<NNQ_KV_E4M3, false>);
    launch_pdl(kernel, grid, dim3(256), (cudaStream_t)stream, a);
    ctx->launches++;
    return check_cuda(ctx, cudaGetLastError(), "cache read launch");
}

}  // extern "C"
