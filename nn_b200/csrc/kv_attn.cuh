// Attention over the paged 8-bit cache: what its kernels share (layout of the cache: kv_cache.cuh).
#pragma once
#include "kv_cache.cuh"

namespace nnq {

struct KvAttn {
    const uint8_t *k, *v, *k_exp, *v_exp;
    const int32_t *length, *row_start, *table;
    const void *q;
    void *y;
    int64_t blocks, table_ld, requests, q_ld, y_ld, rows;
    int kv_heads, group, dim, shift, window;   // window 0: every earlier position
    int q_dt, y_dt;
    int few, many;   // see kv_many; both 0: all requests go to kv_attn_tc_kernel, both INT32_MAX: none goes
    float scale;
    int *status;
};

// One request of the batch as the kernels take it: numbers outside their range are brought inside (the results of such a request are
// undefined, its reads and writes are not).
struct KvRequest {
    int row0, rows;   // its rows of q and y
    int length;       // positions held, the rows' own included
};
__device__ __forceinline__ KvRequest kv_request(const KvAttn &a, int64_t r) {
    KvRequest q;
    const int s0 = (int)min(max((int64_t)a.row_start[r], (int64_t)0), a.rows), s1 = (int)min(max((int64_t)a.row_start[r + 1], (int64_t)s0), a.rows);
    q.row0 = s0;
    q.rows = s1 - s0;
    q.length = (int)min(max((int64_t)a.length[r], (int64_t)0), a.table_ld << a.shift);
    if (q.length < a.length[r] || s0 != a.row_start[r] || s1 != a.row_start[r + 1]) atomicExch(a.status, kStatusIndex);
    return q;
}
// position of row i, and the first position it sees
__device__ __forceinline__ int row_pos(const KvRequest &q, int i) { return q.length - q.rows + i; }
__device__ __forceinline__ int row_first(const KvAttn &a, int pos) { return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0; }

// Which kernel a request goes to. kv_attn_tc_kernel takes 256 query vectors of a key / value head for the price of one, but begins
// slowly and deals a batch in coarser parts; kv_attn_kernel reads the keys again for every 8 vectors. Heads of 128, int8, group 4,
// 8 key / value heads, us of kv_attn_kernel / kv_attn_tc_kernel:
//   bf16, vectors       32             40             56             80            112
//   2 x 500      17.7 / 30.8    18.8 / 30.8    20.5 / 31.2    23.2 / 31.6    24.5 / 33.0
//   2 x 4000     27.6 / 44.5    29.3 / 44.6    36.6 / 45.6    46.7 / 46.7    58.6 / 48.1
//   16 x 500     37.6 / 42.2    43.8 / 41.9    51.2 / 42.3    68.2 / 43.4    86.9 / 44.1
//   2 x 30000    98.1 / 121      117 / 121      159 / 122      219 / 123      300 / 125
//   16 x 4000     118 / 131      140 / 132      188 / 134      262 / 138      356 / 140
//   16 x 30000    686 / 718      853 / 723     1156 / 729     1699 / 738     2363 / 744
//   f32
//   2 x 4000     32.1 / 53.2    33.4 / 53.8    41.1 / 54.6    51.6 / 56.1    64.3 / 58.1
//   16 x 500     42.1 / 48.2    49.5 / 48.7    58.0 / 49.1    77.4 / 50.6    97.2 / 51.9
//   2 x 30000     109 / 171      129 / 171      175 / 172      243 / 173      329 / 173
//   16 x 4000     131 / 184      156 / 185      208 / 187      291 / 190      393 / 192
//   16 x 30000   748 / 1066     934 / 1068    1278 / 1069    1839 / 1077    2534 / 1080
// So: beyond 64, and beyond 32 (48 where queries or outputs are f32) if the batch has 2^16 keys of all heads and requests (taken for
// as long as this one).
constexpr int kKvFew = 32, kKvFewF32 = 48, kKvAlways = 64;
constexpr int64_t kKvManyKeys = 1 << 16;
__device__ __forceinline__ bool kv_many(const KvAttn &a, const KvRequest &q) {
    const int64_t vecs = (int64_t)q.rows * a.group, keys = q.length - row_first(a, max(row_pos(q, 0), 0));
    return vecs > a.many || (vecs > a.few && (float)keys * (float)a.kv_heads * (float)a.requests >= (float)kKvManyKeys);
}

// Two f16 numbers of two codes that lie in the bytes of a 16-bit half each: int8 exactly, e4m3 times 2^-8 (its bits moved to their
// place in an f16 number, subnormal ones included).
template <int FMT>
struct CodePairs;
template <>
struct CodePairs<NNQ_KV_INT8> {
    static constexpr float unscale = 1.0f;
    // codes + 128 in the low bits of 1024: exact
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w ^ 0x80808080u; }
    static __device__ __forceinline__ uint32_t half(uint32_t biased) {
        const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&biased), __half2half2(__ushort_as_half(0x6480)));   // 1152
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    // bytes 0, 1 (2, 3) of a word
    static __device__ __forceinline__ uint32_t low(uint32_t w) { return half(__byte_perm(w, 0x64646464u, 0x4140)); }
    static __device__ __forceinline__ uint32_t high(uint32_t w) { return half(__byte_perm(w, 0x64646464u, 0x4342)); }
    // the four codes of a word
    static __device__ __forceinline__ void four(uint32_t w, uint32_t &p0, uint32_t &p1) {
        p0 = low(word(w));
        p1 = high(word(w));
    }
    // bytes i of x and y side by side, i = 0 .. 3
    static __device__ __forceinline__ void pairs(uint32_t x, uint32_t y, uint32_t &p0, uint32_t &p1, uint32_t &p2, uint32_t &p3) {
        const uint32_t u = __byte_perm(word(x), word(y), 0x5140), v = __byte_perm(word(x), word(y), 0x7362);
        p0 = low(u);
        p1 = high(u);
        p2 = low(v);
        p3 = high(v);
    }
};
template <>
struct CodePairs<NNQ_KV_E4M3> {
    static constexpr float unscale = 256.0f;
    static __device__ __forceinline__ uint32_t word(uint32_t w) { return w; }
    // 128 (b + (b & 128)) moves the magnitude by seven bits and the sign by eight; multiplications, as the logic pipe has enough to do
    static __device__ __forceinline__ uint32_t half(uint32_t x) {
        uint32_t t, r;
        asm("mul.lo.u32 %0, %1, 128;" : "=r"(t) : "r"(x));
        asm("mad.lo.u32 %0, %1, 128, %2;" : "=r"(r) : "r"(x & 0x00800080u), "r"(t));
        return r;
    }
    static __device__ __forceinline__ uint32_t low(uint32_t w) { return half(__byte_perm(w, 0, 0x4140)); }
    static __device__ __forceinline__ uint32_t high(uint32_t w) { return half(__byte_perm(w, 0, 0x4342)); }
    // (the upper bytes of the f16 numbers of all four codes, and the lower ones, then put together)
    static __device__ __forceinline__ void four(uint32_t w, uint32_t &p0, uint32_t &p1) {
        const uint32_t up = (w & 0x80808080u) | (((w & 0x7F7F7F7Fu) >> 1) & 0x7F7F7F7Fu), down = (w << 7) & 0x80808080u;
        p0 = __byte_perm(down, up, 0x5140);
        p1 = __byte_perm(down, up, 0x7362);
    }
    static __device__ __forceinline__ void pairs(uint32_t x, uint32_t y, uint32_t &p0, uint32_t &p1, uint32_t &p2, uint32_t &p3) {
        const uint32_t a = low(x), b = low(y), c = high(x), d = high(y);
        p0 = __byte_perm(a, b, 0x5410);
        p1 = __byte_perm(a, b, 0x7632);
        p2 = __byte_perm(c, d, 0x5410);
        p3 = __byte_perm(c, d, 0x7632);
    }
};

__device__ __forceinline__ float kv_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The power of two that brings the largest absolute value of a query vector (its bits) to 2^14 .. 2^15, and its inverse. Elements
// from 2^-28 of the largest on keep all of an f16 number's bits. Largest values below 2^-112 are scaled like that one.
__device__ __forceinline__ uint32_t kv_top(uint32_t bits) { return min(max(bits >> 23, 15u), 254u); }
__device__ __forceinline__ float kv_top_scale(uint32_t bits) { return __uint_as_float((268u - kv_top(bits)) << 23); }
__device__ __forceinline__ float kv_top_unscale(uint32_t bits) { return __uint_as_float((kv_top(bits) - 14u) << 23); }

__device__ __forceinline__ uint32_t half_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
// x and y as f16 pairs: the nearest values, and the nearest values of what they leave
__device__ __forceinline__ void kv_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = half_bits(h);
    lo = half_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// kv_attn_tc.cu: requests of more than a.few query vectors per key / value head
bool kv_attn_tc_supported(int dim);
size_t kv_attn_tc_workspace(nnq_ctx *ctx, int dim);
nnq_status launch_kv_attn_tc(nnq_ctx *ctx, const KvAttn &a, int fmt, float *records, cudaStream_t st);

}  // namespace nnq
