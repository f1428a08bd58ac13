// The paged cache of keys and values in 8 bits: layout, codes and checks shared by its kernels.
//
// Codes lie in blocks of `block` tokens (16 .. 256, a power of two): [blocks, kv_heads, block, dim], so that a block's tokens of one
// head are one run of block * dim bytes. A code is an int8, or a sign, four exponent bits (bias 7) and three mantissa bits (e4m3).
// Every block and head has one exponent byte for the keys and one for the values: value = code * 2^(byte - 127). The scale is a power
// of two so that it can grow when later tokens of the block need it: codes under the old one become codes under the new one by a
// shift (int8: rounded once more; e4m3: exact but for its subnormal numbers), and so that scales multiply exactly wherever a kernel
// puts them. Up to one bit of the int8 range is lost by it: the largest value of a block has a code of 64 to 127.
// Every byte is a number: int8 -128 is -128, and the two e4m3 codes that stand for NaN elsewhere are +-480. Blocks that nothing has
// been written to can therefore hold anything without reaching a result through a weight of zero.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "nnq_internal.h"
#include "pdl.cuh"

namespace nnq {

// device status word (nnq_device_status)
constexpr int kStatusValue = 3;   // a key or value that was appended is not finite
constexpr int kStatusIndex = 4;   // a slot, a block of a table or a token outside its range

constexpr int kExpMin = 7, kExpMax = 253;   // exponent bytes that are written: both 2^(e - 127) and its inverse are normal numbers

__device__ __forceinline__ float pow2_byte(int e) { return __uint_as_float((uint32_t)min(e, 254) << 23); }   // 2^(e - 127) (0: zero)

// Least exponent byte under which an absolute value of these bits does not pass the largest code (127 = 1.984375 * 2^6 and
// 448 = 1.75 * 2^8): the value's own exponent less 6 (8), and one more where its mantissa is larger.
template <int FMT>
__device__ __forceinline__ int exponent_byte(uint32_t bits) {
    constexpr int shift = FMT == NNQ_KV_INT8 ? 6 : 8;
    constexpr uint32_t top = FMT == NNQ_KV_INT8 ? 0x7E0000u : 0x600000u;
    return min(max((int)(bits >> 23) - shift + ((bits & 0x7FFFFFu) > top ? 1 : 0), kExpMin), kExpMax);
}

// The value of a code. e4m3: its bits are those of an f16 number 2^8 smaller, subnormal numbers included.
template <int FMT>
__device__ __forceinline__ float kv_decode(uint32_t code) {
    if constexpr (FMT == NNQ_KV_INT8) return (float)(int)(int8_t)code;
    else return __half2float(__ushort_as_half((unsigned short)((code & 0x80u) << 8 | (code & 0x7Fu) << 7))) * 256.0f;
}

// Host side: what is wrong with a cache, or NNQ_OK.
inline nnq_status check_kv_cache(nnq_ctx *ctx, const nnq_kv_cache *c) {
    if (!c) return fail(ctx, NNQ_ERR_INVALID_ARG, "cache is NULL");
    if (c->format != NNQ_KV_INT8 && c->format != NNQ_KV_E4M3) return fail(ctx, NNQ_ERR_INVALID_ARG, "unknown cache format %d", c->format);
    if (c->dim != 64 && c->dim != 128 && c->dim != 192 && c->dim != 256)
        return fail(ctx, NNQ_ERR_UNSUPPORTED, "heads of a cache must be 64, 128, 192 or 256 wide (got %d)", c->dim);
    if (c->block < 16 || c->block > 256 || (c->block & (c->block - 1)))
        return fail(ctx, NNQ_ERR_UNSUPPORTED, "blocks of a cache must hold 16, 32, 64, 128 or 256 tokens (got %d)", c->block);
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->blocks < 1) return fail(ctx, NNQ_ERR_INVALID_ARG, "a cache of %d heads and %lld blocks", c->kv_heads, (long long)c->blocks);
    if (c->blocks > INT32_MAX / c->block) return fail(ctx, NNQ_ERR_UNSUPPORTED, "a cache of %lld blocks of %d tokens: slots are numbered in 31 bits", (long long)c->blocks, c->block);
    if (!c->k || !c->v || !c->k_exp || !c->v_exp) return fail(ctx, NNQ_ERR_INVALID_ARG, "NULL tensor in a cache");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) return fail(ctx, NNQ_ERR_INVALID_ARG, "codes of a cache must be 16-byte aligned");
    return NNQ_OK;
}

// Dynamic shared memory of a kernel beyond the default, asked for once per device (a call of its own takes about 1 us): `done` is a
// static of the caller's, one for each kernel.
template <typename K>
inline nnq_status allow_smem(nnq_ctx *ctx, K kernel, size_t bytes, std::atomic<uint64_t> &done) {
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return NNQ_OK;
    nnq_status s = check_cuda(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "shared memory of a kernel");
    if (s == NNQ_OK && ctx->device < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return s;
}

inline int log2_of(int x) { return 31 - __builtin_clz((unsigned)x); }

// Rows of a tensor that a kernel reads or writes 16 bytes at a time.
inline bool rows_aligned(const void *p, int64_t ld, int dt) { return ((uintptr_t)p & 15u) == 0 && ld * (dt == NNQ_F32 ? 4 : 2) % 16 == 0; }

}  // namespace nnq
