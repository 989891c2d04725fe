// The 8-bit key/value cache of one attention layer: where its parts lie, and what the kernels that write, read and attend
// over it share.
//
// For every sequence and key/value head the tokens come in blocks of 32.  A full block is held as 8-bit codes with one scale
// for its keys and one for its values,
//     scale = max |x| / 127 over the block's 32 x D numbers,  code = round_half_even(127 x / max |x|),  value = code * scale,
// and the block that is being filled is held as it came, in 16 bits (the tail).  So a number is rounded once, with the scale of
// the block it ends up in, and what the cache holds depends on the tokens alone, not on how many came at a time.  (With a scale
// that grows as tokens arrive, codes already written would be rounded again at every growth.)  The tail has two slots, for
// blocks of even and of odd index, which hold the last token's block and the one before it: the length may fall to the beginning of
// that, as it does when drafted tokens are refused.
//
// A full block lies in the order in which attention's matrix instructions take it, so that a warp's 16-byte reads are
// contiguous and nothing has to be transposed there:
//     keys    [token group of 16][token parity][D / 64][(token / 2 % 8) * 4 + (d / 16 % 4)][d % 16]
//     values  [D / 16][(d % 8) * 4 + (token / 4 % 4)][d / 8 % 2][token group of 16][token % 4]
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"
#include "unpack.cuh"

namespace w4a16 {

constexpr int kKvBlock = 32;           // tokens that share a scale
constexpr unsigned kKvBadLength = 1;   // status: a length or count outside the cache
constexpr unsigned kKvGaveUp = 2;      // status: a bounded wait ran out
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLightest = -100.0f;         // values' scales below 2^-100 count as that where weights are compared
constexpr float kShrink = 0x1p-32f;      // BF16: sums of values over tokens are held times this, so that those of its largest are finite
constexpr float kNone = -3.4028235e38f;      // the maximum of nothing: no score is below it but minus infinity

// Offset of a number among a full block's codes.
template <int D>
__host__ __device__ constexpr int kv_key_offset(int token, int d) {
    return ((token / 16 * 2 + token % 2) * (D / 64) + d / 64) * 512 + (token / 2 % 8 * 4 + d / 16 % 4) * 16 + d % 16;
}
template <int D>
__host__ __device__ constexpr int kv_value_offset(int token, int d) {
    return d / 16 * 512 + (d % 8 * 4 + token / 4 % 4) * 16 + d / 8 % 2 * 8 + token / 16 * 4 + token % 4;
}

// Where a cache's parts lie in one piece of memory; returns its bytes.  Sizes have been checked.
inline size_t kv_cache_layout(void* memory, int64_t batch, int64_t kv_heads, int64_t max_len, int64_t head_dim, w4a16_kv8_cache* cache) {
    const size_t pairs = static_cast<size_t>(batch) * kv_heads, blocks = max_len / kKvBlock;
    size_t at = 0;
    auto place = [&](size_t bytes) {
        void* part = reinterpret_cast<void*>(reinterpret_cast<uintptr_t>(memory) + at);
        at += (bytes + 255) / 256 * 256;
        return part;
    };
    cache->status = static_cast<uint32_t*>(place(sizeof(uint32_t)));
    cache->k_tail = place(pairs * 2 * kKvBlock * head_dim * 2);
    cache->v_tail = place(pairs * 2 * kKvBlock * head_dim * 2);
    cache->k_scales = static_cast<float*>(place(pairs * blocks * sizeof(float)));
    cache->v_scales = static_cast<float*>(place(pairs * blocks * sizeof(float)));
    cache->k_codes = place(pairs * blocks * kKvBlock * head_dim);
    cache->v_codes = place(pairs * blocks * kKvBlock * head_dim);
    cache->batch = static_cast<int32_t>(batch);
    cache->kv_heads = static_cast<int32_t>(kv_heads);
    cache->max_len = static_cast<int32_t>(max_len);
    cache->head_dim = static_cast<int32_t>(head_dim);
    return at;
}

namespace {

// The cache as the kernels see it.
struct KvCache {
    uint8_t* k_codes;      // [batch * kv heads][blocks][32 * D]
    uint8_t* v_codes;
    float* k_scales;       // [batch * kv heads][blocks]
    float* v_scales;
    char* k_tail;          // [batch * kv heads][2][32][D], 16-bit
    char* v_tail;
    unsigned* status;
    int batch, kv_heads, max_len, blocks;      // blocks: max_len / 32, those that can become full
};

inline KvCache kv_view(const w4a16_kv8_cache& cache) {
    return KvCache{static_cast<uint8_t*>(cache.k_codes), static_cast<uint8_t*>(cache.v_codes), cache.k_scales, cache.v_scales,
                   static_cast<char*>(cache.k_tail), static_cast<char*>(cache.v_tail), cache.status, cache.batch, cache.kv_heads,
                   cache.max_len, cache.max_len / kKvBlock};
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two numbers of a 32-bit word, and back.
template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t word);
template <>
__device__ __forceinline__ float2 widen2<__half>(uint32_t word) { return __half22float2(*reinterpret_cast<__half2*>(&word)); }
template <>
__device__ __forceinline__ float2 widen2<__nv_bfloat16>(uint32_t word) {
    return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float a, float b);
template <>
__device__ __forceinline__ uint32_t narrow2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A power of two that brings `top`, finite and not negative, to between 2^9 and 2^10 (1 for zero), and its inverse.  Both are normal
// numbers for all that FP32 has down to 2^-109; what is below that comes to less than 2^9, which loses none of its bits.
__device__ __forceinline__ float power_for(float top, float& inverse) {
    const int exponent = top > 0.0f ? min(118, 9 - ilogbf(top)) : 0;
    inverse = __int_as_float((127 - exponent) << 23);
    return __int_as_float((127 + exponent) << 23);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) { return narrow2<__half>(a, b); }

// Four codes of a word as (c0, c2) and (c1, c3).
__device__ __forceinline__ void codes_to_half(uint32_t word, uint32_t& even, uint32_t& odd) {
    even = hsub2_u32(and_xor(word, 0x00ff00ffu, 0x64806480u), 0x64806480u);
    odd = hsub2_u32(and_xor(word >> 8, 0x00ff00ffu, 0x64806480u), 0x64806480u);
}

// row / group, for attention's parameters of either kernel; rows are fewer than 2^24, so that the quotient in FP32 is off by one at most.
template <typename Params>
__device__ __forceinline__ int by_group(const Params& p, int row) {
    int quotient = static_cast<int>(static_cast<float>(row) * p.per_group);
    const int rest = row - quotient * p.group;
    if (rest < 0) --quotient;
    if (rest >= p.group) ++quotient;
    return quotient;
}

// A copy into shared memory that counts its bytes on an mbarrier; addresses and size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

template <typename... Params, typename... Args>
int kv_launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, bool programmatic, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t launch = {};
    launch.gridDim = grid;
    launch.blockDim = block;
    launch.dynamicSmemBytes = smem;
    launch.stream = stream;
    cudaLaunchAttribute attr;
    launch.attrs = &attr;
    if (programmatic) {
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        launch.numAttrs = 1;
    }
    if (cudaLaunchKernelEx(&launch, kernel, static_cast<Params>(args)...) != cudaSuccess) return W4A16_ERR_LAUNCH;
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return W4A16_OK;
}

}  // namespace
}  // namespace w4a16
