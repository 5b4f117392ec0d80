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

// What differs from plain attention: logits capped and biased by distance, tokens hidden by a window or shown by a prefix.
struct PgScores {
    const float* slopes;             // (n_q) or null
    const int32_t* prefix;           // (n_seq) or null
    float cap, cap_inv;              // of logits to the base of 2, and its reciprocal; 0: none
    int32_t window, max_prefix;      // 0: none; what prefixes are held to
    static constexpr int kNear = 5;
    float near[kNear];               // of the cap, below
};
// What an attention's logits go through beside the scale, each with kernels of its own: in one that asks at run time, the layers that only mask paid 7 % of
// a decode for the others' registers.  Rows may be masked in all but the plain one.
enum PgMode { kPlain, kMasked, kCapped, kBiased, kCappedBiased };
inline PgMode pg_mode(const PgScores& S, bool mod) {
    return !mod ? kPlain : S.slopes ? S.cap > 0.f ? kCappedBiased : kBiased : S.cap > 0.f ? kCapped : kMasked;
}
// A sequence's prefix
__device__ __forceinline__ int pg_prefix(const PgScores& S, int seq, int len) { return S.prefix ? max(0, min(S.prefix[seq], min(S.max_prefix, len))) : 0; }

// A slope to the base of 2: finite where it is positive and finite, so that a row's own token has no bias; none where it is none.  (One instruction: a comparison and
// a choice for both signs cost 64 ragged sequences 85.7 us instead of 85.1.)
__device__ __forceinline__ float pg_slope(float s) {
    float x;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(s * 1.44269504088896340736f), "f"(3.402823466e38f));
    return x;
}

__device__ __forceinline__ float pg_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap * tanh(x / cap), u = x / cap.  Up to 1/2 an odd polynomial of degree 9, fitted to the relative error (1.5e-8; near[]: times the cap); beyond it
// 1 - 2 / (e^2u + 1), whose terms are then of one magnitude, so that both are off by a few roundings of the result itself.
__device__ __forceinline__ float pg_cap_near(float u, float v, const PgScores& S) {      // v = u^2
    float p = S.near[PgScores::kNear - 1];
#pragma unroll
    for (int i = PgScores::kNear - 2; i >= 0; --i) p = fmaf(p, v, S.near[i]);
    return u * p;
}
__device__ __forceinline__ float pg_cap_far(float u, float cap) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(pg_ex2(u * 2.8853900817779268f) + 1.f));
    return cap * fmaf(-2.f, r, 1.f);
}
// The factor from products to u, finite and above zero: products of zero are nothing under it and hidden ones minus infinity, and what it would take beyond has
// long reached the cap, or is nothing beside it.
__device__ __forceinline__ float pg_unit(float factor, const PgScores& S) { return fmaxf(fminf(factor * S.cap_inv, 1.329227995784916e36f), kPgFactorMin); }
__device__ __forceinline__ float pg_cap_any(float u, const PgScores& S) {
    const float f = pg_cap_far(u, S.cap), v = u * u;
    return v <= 0.25f ? pg_cap_near(u, v, S) : f;
}

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
