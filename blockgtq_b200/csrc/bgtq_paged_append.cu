// Writing tokens into the paged 4-bit cache, with the rotary embedding on the way, and reading them back.
//
// append: for every token i with slot s_i >= 0, every KV head:  k' = rope(k, angle of positions[i]), scale_g = bf16(max |x| over
// the group's 32 dims / 7) held in [2^-17, 9344], code = x / scale rounded to the nearest whole number, ties to even, held in
// [-7, 7].  The rotation is four fp32 products and two sums, none of them fused, and its result is quantised without another
// rounding.  A group with a NaN gets a NaN scale; infinities and what lies beyond 65408 saturate.
#include "bgtq_paged_common.cuh"
#include "bgtq_paged_rows.h"

namespace bgtq {
namespace {

constexpr int kApThreads = 256;
// 1.5 * 2^23 + 8: a sum with it has the nearest whole number, ties to even, plus 8 in its lower sixteen bits
constexpr float kRound = 12582920.0f;

struct ApParams {
    uint8_t* pages;
    int64_t page_stride, head_stride;
    int32_t n_pages, units;
    const int64_t* slots;
    const void *k, *v, *q;
    int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;        // elements
    void* q_out;                                       // (n_tok, n_q, 128) contiguous
    const float *cos, *sin;                            // (n_positions, 64) rows, or null: no rotation
    int64_t cs_st;
    const int64_t* positions;
    int64_t pos_st;                                    // from one axis to the next
    uint32_t axis[4];                                  // the pairs' axes, two bits each (where there are several)
    int32_t n_axes, n_positions, n_tok, n_kv, n_q;
    int32_t kv_chunks, q_chunks, per;                  // chunks of 16 / L heads' K (or V) rows, of queries; chunks of a warp's task
    int32_t* status;
};

// L lanes hold a row: lane j its dims 32 g + E j .. + E - 1 of every group g, E = 32 / L, so that a group's largest magnitude is two or three
// exchanges away, both dims of every rotated pair (d, d + 64) lie in one lane, and a lane's codes are 2 E bytes of a K row.
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
template <int E>
struct Row {
    uint32_t w[4][E / 2];
};
template <int E> struct Vec;
template <> struct Vec<4> { using type = uint2; };
template <> struct Vec<8> { using type = uint4; };
template <int E, typename T>
__device__ __forceinline__ Row<E> ap_load(const T* row, int j) {
    Row<E> r;
#pragma unroll
    for (int g = 0; g < 4; ++g) *reinterpret_cast<typename Vec<E>::type*>(r.w[g]) = *reinterpret_cast<const typename Vec<E>::type*>(row + 32 * g + E * j);
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {             // NaN when either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// bf16(a / 7) within the scales' range; the quotient as a division rounds it, by Markstein's correction: the product with the rounded reciprocal, and
// its remainder, both fused, on top (an infinity ends up as the largest scale).
__device__ __forceinline__ float ap_scale(float a) {
    const float c = 1.0f / 7.0f, q0 = __fmul_rn(a, c), q = __fmaf_rn(__fmaf_rn(-7.0f, q0, a), c, q0);
    return __bfloat162float(__float2bfloat16_rn(fmaxf(fminf(q, kPgScaleMax), kPgScaleMin)));
}
// A group's E values -> k = code + 8 + 1.5 * 2^23 each.  x / scale is not divided out: k = round(x * (1 / scale)) is the whole number next to
// the quotient unless that is within 2^-20 of a tie, and the remainder x - code * scale, exact (11 bits of code * scale, and no more than
// scale / 2 left), says so: only then is it decided by it.
template <int E>
__device__ __forceinline__ void ap_codes(const float (&in)[E], float largest, float scale, float (&k)[E]) {
    float x[E], r, far = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = in[e];
    if (largest > 7.45f * scale) {           // (only at the largest scale: beyond it values saturate)
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fminf(fmaxf(x[e], -7.45f * scale), 7.45f * scale);
    }
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
#pragma unroll
    for (int e = 0; e < E; ++e) {
        k[e] = __fmaf_rn(x[e], r, kRound);
        far = fmaxf(far, fabsf(__fmaf_rn(-__fsub_rn(k[e], kRound), scale, x[e])));
    }
    if (2.f * far >= scale) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float left = __fmaf_rn(-__fsub_rn(k[e], kRound), scale, x[e]), twice = 2.f * fabsf(left);
            if (twice > scale || (twice == scale && (__float_as_uint(k[e]) & 1u))) k[e] = __fadd_rn(k[e], copysignf(1.f, left));
        }
    }
}

// A warp's task: two tokens and a run of chunks of 16 / L rows (KV heads' K, then V, then queries); the L lanes o take row o / 2 of a chunk for
// token o % 2.  The tables' rows are read once for all of a task's chunks.
// Bound: memory, 512 bytes in and 144 out per token and KV head, 512 per query row, where there are queries: 65536 tokens of 32 query and 8 KV
// heads 223 us, 6.5 TB/s, and 16384 63.8 us, 5.7 TB/s, with three chunks of a warp on their way to shared memory (in registers there was room
// for one: 289 and 82 us; three CTAs on an SM instead of two, with spills: 267 and 78).  Without queries the quantisation's
// instructions: 16384 tokens 30.7 us, 2.8 TB/s.  32 tokens: 2.9 us, a chain of latencies.
// kAxes: a pair's angle is looked up at its token's position along the pair's axis, four pairs at once where they have one axis (sections of 16, 24 and
// 24, 16384 tokens: 66.7 us beside 63.3 with one axis; each pair by itself 78), and axes that take turns one by one (68.4).
template <typename T, int L, bool kAxes>
__global__ void __launch_bounds__(kApThreads, L == 8 ? 4 : 2) pg_append_kernel(const ApParams P) {
    constexpr int E = 32 / L, kHeads = 16 / L;
    constexpr uint32_t kAhead = L == 4 ? 3 : 0;            // chunks of a warp on their way
    __shared__ __align__(16) uint4 ring[kAhead ? kApThreads / 32 * kAhead * 4 * 32 : 1];
    const int lane = threadIdx.x & 31, o = lane / L, j = lane % L;
    const uint32_t n_chunks = 2 * P.kv_chunks + P.q_chunks, n_tasks = (n_chunks + P.per - 1) / P.per;
    const uint32_t task = blockIdx.x * (kApThreads / 32) + (threadIdx.x >> 5), pair = task / n_tasks;
    const int64_t tok = 2 * (int64_t)pair + (o & 1);
    grid_launch_dependents();
    grid_dependency_wait();
    const bool there = tok < P.n_tok;
    const uint32_t first = (task - pair * n_tasks) * P.per, last = min(n_chunks, first + P.per);
    if (2 * (int64_t)pair >= P.n_tok) return;
    // kind (0 K, 1 V, 2 query) and head of these lanes' row of a chunk; a row past the end is none
    auto place = [&](uint32_t chunk, int& kind, int& head) {
        kind = chunk < (uint32_t)P.kv_chunks ? 0 : chunk < 2u * P.kv_chunks ? 1 : 2;
        head = kHeads * (int)(chunk - kind * (uint32_t)P.kv_chunks) + (o >> 1);
        return there && head < (kind == 2 ? P.n_q : P.n_kv);
    };
    auto row_of = [&](int kind, int head) {
        return kind == 0 ? reinterpret_cast<const T*>(P.k) + tok * P.k_st + head * P.k_sh
               : kind == 1 ? reinterpret_cast<const T*>(P.v) + tok * P.v_st + head * P.v_sh
                           : reinterpret_cast<const T*>(P.q) + tok * P.q_st + head * P.q_sh;
    };
    auto fetch = [&](uint32_t chunk) {
        int kind, head;
        Row<E> r = {};
        if (place(chunk, kind, head)) r = ap_load<E>(row_of(kind, head), j);
        return r;
    };
    // Bulk: the next chunks are on their way to shared memory, each lane's pieces to places of its own.
    const uint32_t mine = kAhead ? smem_u32(ring) + ((threadIdx.x >> 5) * kAhead * 4 * 32 + lane) * 16 : 0u;
    auto request = [&](uint32_t chunk, uint32_t slot) {
        if (chunk < last) {
            int kind, head;
            const bool live = place(chunk, kind, head);
            const T* const src = live ? row_of(kind, head) + E * j : reinterpret_cast<const T*>(P.k);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mine + (slot * 4 + g) * 512), "l"(live ? src + 32 * g : src), "r"(live ? 16 : 0)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Row<E> next;
    if constexpr (kAhead) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) request(first + i, i);
    } else {
        next = fetch(first);
    }
    int64_t slot = there ? P.slots[tok] : -1;
    const int page_tok = P.units * kUnitTok;
    if (slot >= (int64_t)P.n_pages * page_tok) {
        if (P.status) *P.status = kStatusOverflow;
        slot = -1;
    }
    float cs[2][E] = {}, sn[2][E] = {};
    const bool turns = !(first >= (uint32_t)P.kv_chunks && last <= 2u * P.kv_chunks);          // (V alone needs no angle)
    if constexpr (kAxes) {
        if (there) {
            int64_t p[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) p[a] = a < P.n_axes ? P.positions[a * P.pos_st + tok] : 0;
            const auto in = [&](int64_t x) { return x >= 0 && x < P.n_positions; };
            if (!(in(p[0]) && in(p[1]) && in(p[2]) && in(p[3]))) {         // (as below)
                if (P.status && slot >= 0) *P.status = kStatusOverflow;
                slot = -1;
                p[0] = p[1] = p[2] = p[3] = 0;
            }
            if (turns)
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < E; i += 4) {
                        const int d = 32 * g + E * j + i;
                        const uint32_t four = P.axis[d >> 4] >> (2 * (d & 15)) & 255u;         // the axes of pairs d .. d + 3
                        auto row = [&](uint32_t a) { return (a & 2 ? a & 1 ? p[3] : p[2] : a & 1 ? p[1] : p[0]) * P.cs_st + d; };
                        if (four == (four & 3u) * 0x55u) {                     // (all one)
                            const int64_t at = row(four & 3u);
                            *reinterpret_cast<float4*>(&cs[g][i]) = *reinterpret_cast<const float4*>(P.cos + at);
                            *reinterpret_cast<float4*>(&sn[g][i]) = *reinterpret_cast<const float4*>(P.sin + at);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int64_t at = row(four >> (2 * e) & 3u) + e;
                                cs[g][i + e] = P.cos[at];
                                sn[g][i + e] = P.sin[at];
                            }
                        }
                    }
        }
    } else if (P.cos && there) {
        int64_t p = P.positions[tok];
        if (p < 0 || p >= P.n_positions) { // no angle for it: the token is not stored, and the caller learns of it
            if (P.status && slot >= 0) *P.status = kStatusOverflow;
            slot = -1;
            p = 0;
        }
        if (turns)
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < E; i += 4) {
                    *reinterpret_cast<float4*>(&cs[g][i]) = *reinterpret_cast<const float4*>(P.cos + p * P.cs_st + 32 * g + E * j + i);
                    *reinterpret_cast<float4*>(&sn[g][i]) = *reinterpret_cast<const float4*>(P.sin + p * P.cs_st + 32 * g + E * j + i);
                }
    }
    uint8_t* unit = nullptr;
    int t = 0;
    if (slot >= 0) {
        const int64_t page = (uint64_t)slot < 0x100000000ull ? (int64_t)((uint32_t)slot / (uint32_t)page_tok) : slot / page_tok;
        const int in_page = (int)(slot - page * page_tok);
        t = in_page & 15;
        unit = P.pages + page * P.page_stride + (in_page >> 4) * kUnitBytes;
    }
    // the two tokens are neighbours of one pair: their V half-words leave as words
    const int64_t other = __shfl_xor_sync(0xffffffffu, slot, L);
    const bool paired = slot >= 0 && other >= 0 && (slot ^ other) == 1 && ((slot & 1) == (o & 1));
    uint32_t slot_of = 0;
    for (uint32_t chunk = first; chunk < last; ++chunk) {
        Row<E> row;
        if constexpr (kAhead) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
#pragma unroll
            for (int g = 0; g < 4; ++g) *reinterpret_cast<uint4*>(row.w[g]) = lds128(mine + (slot_of * 4 + g) * 512);
        } else {
            row = next;
            if (chunk + 1 < last) next = fetch(chunk + 1);
        }
        int kind, head;
        const bool live = place(chunk, kind, head);
        float x[4][E];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 a = PgType<T>::up(row.w[g][e / 2]);
                x[g][e] = a.x;
                x[g][e + 1] = a.y;
            }
        if constexpr (kAhead) {
            request(chunk + kAhead, slot_of);
            slot_of = slot_of == kAhead - 1 ? 0 : slot_of + 1;
        }
        if (kind != 1 && P.cos) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float a = x[g][e], b = x[g + 2][e];
                    x[g][e] = __fsub_rn(__fmul_rn(a, cs[g][e]), __fmul_rn(b, sn[g][e]));
                    x[g + 2][e] = __fadd_rn(__fmul_rn(b, cs[g][e]), __fmul_rn(a, sn[g][e]));
                }
        }
        if (kind == 2) {
            if (live) {
                T* dst = reinterpret_cast<T*>(P.q_out) + (tok * P.n_q + head) * kHD + E * j;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t w[E / 2];
#pragma unroll
                    for (int e = 0; e < E; e += 2) w[e / 2] = PgType<T>::down(x[g][e], x[g][e + 1]);
                    *reinterpret_cast<typename Vec<E>::type*>(dst + 32 * g) = *reinterpret_cast<typename Vec<E>::type*>(w);
                }
            }
            continue;
        }
        uint32_t half[E] = {};             // half-words E j + e (k's other bits are multiples of 2^16)
        float scale[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float a = 0.f, k[E];
#pragma unroll
            for (int e = 0; e < E; ++e) a = max_nan(a, fabsf(x[g][e]));
#pragma unroll
            for (int d = 1; d < L; d <<= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, d));
            scale[g] = ap_scale(a);
            if (a != a) {
                scale[g] = __uint_as_float(0x7fffffffu);
#pragma unroll
                for (int e = 0; e < E; ++e) k[e] = kRound;
            } else {
                ap_codes<E>(x[g], a, scale[g], k);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) half[e] += __float_as_uint(k[e]) << (4 * g);
        }
        const uint2 s4 = make_uint2(PgType<__nv_bfloat16>::down(scale[0], scale[1]), PgType<__nv_bfloat16>::down(scale[2], scale[3]));
        uint32_t word[E / 2];
#pragma unroll
        for (int e = 0; e < E; e += 2) word[e / 2] = __byte_perm(half[e], half[e + 1], 0x5410);
        uint8_t* const u = unit + head * P.head_stride;
        if (kind == 0) {
            if (live && unit) {
                *reinterpret_cast<typename Vec<E>::type*>(u + 64 * t + 2 * E * j) = *reinterpret_cast<typename Vec<E>::type*>(word);
                if (j == 0) *reinterpret_cast<uint2*>(u + kUnitKs + 8 * t) = s4;
            }
            continue;
        }
        // V, words of two tokens: the even one's lane takes the first E / 2 half-words of both, the odd one's the others
        uint32_t both[E / 2];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
            const uint32_t theirs = __shfl_xor_sync(0xffffffffu, o & 1 ? word[e] : word[e + E / 4], L);
            const uint32_t even = o & 1 ? theirs : word[e], odd = o & 1 ? word[e + E / 4] : theirs;
            both[2 * e] = __byte_perm(even, odd, 0x5410);
            both[2 * e + 1] = __byte_perm(even, odd, 0x7632);
        }
        if (live && unit) {
            uint8_t* const dst = u + kUnitV + 128 * (t >> 1) + 4 * E * j;
            if (paired) {
                *reinterpret_cast<typename Vec<E>::type*>(dst + 2 * E * (o & 1)) = *reinterpret_cast<typename Vec<E>::type*>(both);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) *reinterpret_cast<uint16_t*>(dst + 4 * e + 2 * (t & 1)) = (uint16_t)half[e];
            }
            if (j == 0) *reinterpret_cast<uint2*>(u + kUnitVs + 8 * t) = s4;
        }
    }
}

struct RdParams {
    PgPool pool;
    const int64_t* slots;
    void *k, *v;              // (n_tok, n_kv, 128) contiguous
    int32_t n_tok, n_kv;
    int32_t* status;
};

// Four lanes per row, lane j its dims 32 g + 8 j .. + 7; the values are exact in fp16 and fp32, and rounded once to bf16.
// Bound: memory, 144 bytes in and 512 out per token and KV head: 16384 tokens of 8 KV heads 15.9 us, 5.4 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) pg_read_kernel(const RdParams P) {
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t r = (blockIdx.x * 256 + threadIdx.x) >> 2, rows = 2 * (uint32_t)P.n_kv;
    const int j = threadIdx.x & 3;
    const uint32_t tok = r / rows;
    if (tok >= (uint32_t)P.n_tok) return;
    const int row = (int)(r - tok * rows);
    const bool is_v = row >= P.n_kv;
    const int head = is_v ? row - P.n_kv : row;
    int64_t slot = P.slots[tok];
    const int page_tok = P.pool.units * kUnitTok;
    if (slot >= (int64_t)P.pool.n_pages * page_tok) {
        if (P.status) *P.status = kStatusOverflow;
        slot = -1;
    }
    uint32_t w[4] = {};                    // half-words 8 j .. 8 j + 7
    float scale[4] = {};
    if (slot >= 0) {
        const int64_t page = (uint64_t)slot < 0x100000000ull ? (int64_t)((uint32_t)slot / (uint32_t)page_tok) : slot / page_tok;
        const int in_page = (int)(slot - page * page_tok), t = in_page & 15;
        const uint8_t* u = P.pool.pages + page * P.pool.page_stride + head * P.pool.head_stride + (in_page >> 4) * kUnitBytes;
        if (is_v) {
            const uint4* at = reinterpret_cast<const uint4*>(u + kUnitV + 128 * (t >> 1) + 32 * j);
            const uint4 x = at[0], y = at[1];
            const uint32_t pick = t & 1 ? 0x7632u : 0x5410u;
            w[0] = __byte_perm(x.x, x.y, pick); w[1] = __byte_perm(x.z, x.w, pick);
            w[2] = __byte_perm(y.x, y.y, pick); w[3] = __byte_perm(y.z, y.w, pick);
        } else {
            const uint4 x = *reinterpret_cast<const uint4*>(u + 64 * t + 16 * j);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
        }
        const uint2 s = *reinterpret_cast<const uint2*>(u + (is_v ? kUnitVs : kUnitKs) + 8 * t);
        scale[0] = pg_lo(s.x); scale[1] = pg_hi(s.x); scale[2] = pg_lo(s.y); scale[3] = pg_hi(s.y);
    }
    T* dst = reinterpret_cast<T*>(is_v ? P.v : P.k) + ((int64_t)tok * P.n_kv + head) * kHD + 8 * j;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = slot < 0 ? 0.f : (float)((int)(w[e >> 1] >> (16 * (e & 1) + 4 * g) & 15u) - 8) * scale[g];
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(dst + 32 * g)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(dst + 32 * g)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            *reinterpret_cast<uint4*>(dst + 32 * g) =
                make_uint4(PgType<T>::down(x[0], x[1]), PgType<T>::down(x[2], x[3]), PgType<T>::down(x[4], x[5]), PgType<T>::down(x[6], x[7]));
        }
    }
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

int check_pool(const void* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, int32_t n_kv) {
    if (!pages || n_pages < 1 || n_kv < 1 || page_tokens < kUnitTok || page_tokens % kUnitTok) return BGTQ_E_BADARG;
    if (n_kv > 65535 || (int64_t)n_pages * page_tokens > INT64_MAX / kUnitBytes) return BGTQ_E_TOOBIG;
    if (!aligned(pages, 16) || page_stride % 16 || head_stride % 16) return BGTQ_E_ALIGN;
    return BGTQ_OK;
}

}  // namespace
}  // namespace bgtq

using namespace bgtq;

extern "C" __attribute__((visibility("default"))) int bgtq_paged_launches(void) { return pg_launched; }

// axis_of (host, 64 entries below n_axes): the axis that each rotated pair's position is taken along; null: there is one.
static int append(uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots, const void* k,
                  int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const void* q, int64_t q_st, int64_t q_sh, void* q_out,
                  const float* rope_cos, const float* rope_sin, int64_t rope_st, const int64_t* positions, int64_t pos_st, const uint8_t* axis_of,
                  int32_t n_axes, int32_t n_positions, int32_t n_tok, int32_t n_kv, int32_t n_q, int32_t flags, int32_t* status, void* stream) {
    pg_launched = 0;
    if (n_tok < 0 || n_q < 0 || (flags & ~BGTQ_PAGED_BF16)) return BGTQ_E_BADARG;
    if (const int e = check_pool(pages, page_stride, head_stride, n_pages, page_tokens, n_kv)) return e;
    uint32_t axis[4] = {};
    if (axis_of) {
        if (n_axes < 1 || n_axes > 4 || !rope_cos) return BGTQ_E_BADARG;
        for (int d = 0; d < kHD / 2; ++d) {
            if (axis_of[d] >= n_axes) return BGTQ_E_BADARG;
            axis[d >> 4] |= (uint32_t)axis_of[d] << (2 * (d & 15));
        }
    }
    if (n_tok == 0) return BGTQ_OK;
    if (!slots || !k || !v || (q == nullptr) != (n_q == 0) || (q && !q_out) || !rope_cos != !rope_sin) return BGTQ_E_BADARG;
    if (rope_cos && (!positions || n_positions < 1)) return BGTQ_E_BADARG;
    if (q && !rope_cos) return BGTQ_E_BADARG;
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(q, 16) || !aligned(q_out, 16) || k_st % 8 || k_sh % 8 || v_st % 8 || v_sh % 8 ||
        q_st % 8 || q_sh % 8 || !aligned(rope_cos, 16) || !aligned(rope_sin, 16) || rope_st % 4)
        return BGTQ_E_ALIGN;
    if (!paged_apart(n_pages, n_kv, page_stride, head_stride, (int64_t)page_tokens / kUnitTok * kUnitBytes)) return BGTQ_E_BADARG;
    // Few rows: as many warps as there are, two rows each and eight lanes to a row (32 tokens of 32 query and 8 KV heads 2.8 us, 3.0 with four).
    // Otherwise four rows and four lanes to a row (4096 tokens 3 us less, measured before the ring), as many chunks one behind the other as leave the SMs
    // one round of resident warps (6 of 12 per warp: 2 us more).
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int64_t pairs = ((int64_t)n_tok + 1) / 2;
    const int L = pairs * (n_kv + (n_q + 1) / 2 + 1) <= 8ll * sms ? 8 : 4, heads = 16 / L;
    ApParams P{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok, slots, k, v, q, k_st, k_sh, v_st, v_sh, q_st, q_sh, q_out,
               rope_cos, rope_sin, rope_st, positions, pos_st, {axis[0], axis[1], axis[2], axis[3]}, n_axes, n_positions, n_tok, n_kv, n_q,
               (n_kv + heads - 1) / heads, (n_q + heads - 1) / heads, 1, status};
    const int64_t chunks = 2 * P.kv_chunks + P.q_chunks;
    const int64_t parts = 16ll * sms / pairs;              // of a pair's chunks
    P.per = (int32_t)((chunks + (parts < 1 ? 1 : parts) - 1) / (parts < 1 ? 1 : parts));
    const int64_t tasks = pairs * ((chunks + P.per - 1) / P.per), blocks = (tasks + kApThreads / 32 - 1) / (kApThreads / 32);
    if (tasks + kApThreads / 32 > INT32_MAX) return BGTQ_E_TOOBIG;
    const bool bf16 = flags & BGTQ_PAGED_BF16;
    const auto kernel = axis_of ? L == 8 ? bf16 ? pg_append_kernel<__nv_bfloat16, 8, true> : pg_append_kernel<__half, 8, true>
                                         : bf16 ? pg_append_kernel<__nv_bfloat16, 4, true> : pg_append_kernel<__half, 4, true>
                        : L == 8 ? bf16 ? pg_append_kernel<__nv_bfloat16, 8, false> : pg_append_kernel<__half, 8, false>
                                 : bf16 ? pg_append_kernel<__nv_bfloat16, 4, false> : pg_append_kernel<__half, 4, false>;
    return pg_launch_ok(launch_kernel(kernel, dim3((unsigned)blocks), dim3(kApThreads), 0, (cudaStream_t)stream, true, P)) ? BGTQ_OK : BGTQ_E_LAUNCH;
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_append(
    uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots, const void* k,
    int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const void* q, int64_t q_st, int64_t q_sh, void* q_out,
    const float* rope_cos, const float* rope_sin, int64_t rope_st, const int64_t* positions, int32_t n_positions, int32_t n_tok,
    int32_t n_kv, int32_t n_q, int32_t flags, int32_t* status, void* stream) {
    return append(pages, page_stride, head_stride, n_pages, page_tokens, slots, k, k_st, k_sh, v, v_st, v_sh, q, q_st, q_sh, q_out, rope_cos, rope_sin,
                  rope_st, positions, 0, nullptr, 1, n_positions, n_tok, n_kv, n_q, flags, status, stream);
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_append_axes(
    uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots, const void* k,
    int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const void* q, int64_t q_st, int64_t q_sh, void* q_out,
    const float* rope_cos, const float* rope_sin, int64_t rope_st, const int64_t* positions, int64_t pos_st, const uint8_t* axis_of, int32_t n_axes,
    int32_t n_positions, int32_t n_tok, int32_t n_kv, int32_t n_q, int32_t flags, int32_t* status, void* stream) {
    if (!axis_of) return BGTQ_E_BADARG;
    return append(pages, page_stride, head_stride, n_pages, page_tokens, slots, k, k_st, k_sh, v, v_st, v_sh, q, q_st, q_sh, q_out, rope_cos, rope_sin,
                  rope_st, positions, pos_st, axis_of, n_axes, n_positions, n_tok, n_kv, n_q, flags, status, stream);
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_read(
    const uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots,
    int32_t n_tok, int32_t n_kv, void* k, void* v, int32_t flags, int32_t* status, void* stream) {
    pg_launched = 0;
    if (n_tok < 0 || (flags & ~(BGTQ_PAGED_BF16 | BGTQ_PAGED_F32)) || flags == (BGTQ_PAGED_BF16 | BGTQ_PAGED_F32)) return BGTQ_E_BADARG;
    if (const int e = check_pool(pages, page_stride, head_stride, n_pages, page_tokens, n_kv)) return e;
    if (n_tok == 0) return BGTQ_OK;
    if (!slots || !k || !v) return BGTQ_E_BADARG;
    if (!aligned(k, 16) || !aligned(v, 16)) return BGTQ_E_ALIGN;
    RdParams P{{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok}, slots, k, v, n_tok, n_kv, status};
    const int64_t blocks = ((int64_t)n_tok * 2 * n_kv * 4 + 255) / 256;
    if (blocks * 256 > 1ll << 32) return BGTQ_E_TOOBIG;          // (threads are counted in 32 bits)
    const auto kernel = (flags & BGTQ_PAGED_F32) ? pg_read_kernel<float> : (flags & BGTQ_PAGED_BF16) ? pg_read_kernel<__nv_bfloat16> : pg_read_kernel<__half>;
    return pg_launch_ok(launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, true, P)) ? BGTQ_OK : BGTQ_E_LAUNCH;
}
