// The paged 4-bit cache: layout of a page and what its kernels share.
//
// A page of one KV head is a row of units of 16 tokens; a unit is 2304 bytes:
//     [0, 1024)     K codes: token t, half-word W (0..31) at 64 t + 2 W
//     [1024, 2048)  V codes: token t, half-word W at 1024 + 128 (t / 2) + 4 W + 2 (t % 2)
//     [2048, 2176)  K scales, bf16: token t, group g (0..3) at 2048 + 8 t + 2 g
//     [2176, 2304)  V scales, the same at 2176
// Nibble n of half-word W holds the code of dim 32 n + W plus 8, group n is dims 32 n .. 32 n + 31; value = code * scale.
//
// What the layout is for: a word of two neighbouring half-words (K: two dims of a token; V: the same dim of two tokens) under one mask is
// a pair of numbers that mma.sync takes as fp16 operands after a shift or an addition at most, and all pairs of one mask belong to
// one group, so that the scale is constant over a product.  A warp's 16-byte loads of a unit's rows are contiguous 512 bytes.
//
// code * scale has at most 3 + 8 significant bits and scales lie in [2^-17, 9344]: every value is exactly an fp16 number.
#pragma once
#include <cuda_bf16.h>

#include <atomic>

#include "bgtq_common.cuh"

namespace bgtq {

constexpr int kUnitTok = 16;
constexpr int kUnitBytes = 2304;
constexpr int kUnitV = 1024, kUnitKs = 2048, kUnitVs = 2176;
constexpr float kPgScaleMin = 7.62939453125e-6f;       // 2^-17: 2^-24 is the last bit of a scale that is multiplied by a code
constexpr float kPgScaleMax = 9344.0f;                 // 7 * 9344 < 65504
constexpr int kStatusBadPage = 4;                      // a page number outside the pool: its tokens were left out

// Where the pages are.  Strides in bytes.
struct PgPool {
    const uint8_t* pages;
    int64_t page_stride, head_stride;
    int32_t n_pages, units;         // units per page
};

__device__ __forceinline__ float pg_lo(uint32_t w) { return __uint_as_float(w << 16); }              // bf16 pair -> fp32
__device__ __forceinline__ float pg_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

template <typename T> struct PgType;
template <> struct PgType<__half> {
    static constexpr bool kHalf = true;
    static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) { return pack_half2(a, b); }
};
template <> struct PgType<__nv_bfloat16> {
    static constexpr bool kHalf = false;
    static __device__ __forceinline__ float2 up(uint32_t w) { return make_float2(pg_lo(w), pg_hi(w)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        uint32_t d;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
        return d;
    }
};

// A query row of largest magnitude `top` comes to [2^13, 2^14) by 2^e; a row of zeros, or with an infinity, stays.  e: -114 .. 140.
__device__ __forceinline__ int pg_row_exponent(float top) {
    const int ex = (int)(__float_as_uint(top) >> 23) - 127;
    return top > 0.f && ex < 128 ? 13 - ex : 0;
}
// 2^e as a product of two factors
__device__ __forceinline__ void pg_pow2(int e, float& a, float& b) {
    a = __uint_as_float((uint32_t)(127 + e / 2) << 23);
    b = __uint_as_float((uint32_t)(127 + e - e / 2) << 23);
}

// The factor from products to logits is held above zero: hidden ones are minus infinity before it.  (Products are below 2^38: nothing is left of
// them at the smallest normal number either.)
constexpr float kPgFactorMin = 1.17549435e-38f;

// Kernels that this thread's last call of an entry point enqueued.
inline thread_local int32_t pg_launched = 0;
inline bool pg_launch_ok(cudaError_t e) {
    pg_launched += e == cudaSuccess;
    return e == cudaSuccess;
}

// Lets a kernel use this much dynamic shared memory, once per device.
template <typename K>
inline bool pg_allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (bit & done.load(std::memory_order_relaxed)) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

}  // namespace bgtq
