// Writing tokens into the paged 4-bit cache, with the rotary embedding on the way, and reading them back.
//
// append: for every token i with slot s_i >= 0, every KV head:  k' = rope(k, angle of positions[i]), scale_g = bf16(max |x| over
// the group's 32 dims / 7) held in [2^-17, 9344], code = x / scale rounded to the nearest whole number, ties to even, held in
// [-7, 7].  The rotation is four fp32 products and two sums, none of them fused, and its result is quantised without another
// rounding.  A group with a NaN gets a NaN scale; infinities and what lies beyond 65408 saturate.
#include "bgtq_paged_common.cuh"

namespace bgtq {
namespace {

constexpr int kApThreads = 256;

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
    int32_t n_positions, n_tok, n_kv, n_q;
    int32_t* status;
};

// Eight lanes hold a row: lane j its dims 32 g + 4 j .. + 3 of every group g, so that a group's largest magnitude is three
// exchanges away and both dims of every rotated pair (d, d + 64) lie in one lane.
template <typename T>
__device__ __forceinline__ void ap_load(const T* row, int j, float (&x)[4][4]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 32 * g + 4 * j);
        const float2 a = PgType<T>::up(w.x), b = PgType<T>::up(w.y);
        x[g][0] = a.x; x[g][1] = a.y; x[g][2] = b.x; x[g][3] = b.y;
    }
}

__device__ __forceinline__ void ap_rotate(float (&x)[4][4], const float4 (&c)[2], const float4 (&s)[2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const float cc[4] = {c[g].x, c[g].y, c[g].z, c[g].w}, ss[4] = {s[g].x, s[g].y, s[g].z, s[g].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = x[g][e], b = x[g + 2][e];
            x[g][e] = __fsub_rn(__fmul_rn(a, cc[e]), __fmul_rn(b, ss[e]));
            x[g + 2][e] = __fadd_rn(__fmul_rn(b, cc[e]), __fmul_rn(a, ss[e]));
        }
    }
}

// A warp takes two tokens and two rows of each: octet o = lane / 8 is row 2 * chunk + o / 2 of token 2 * pair + o % 2, rows
// counted over the K heads, the V heads and the query heads.
template <typename T>
__global__ void __launch_bounds__(kApThreads) pg_append_kernel(const ApParams P) {
    const int lane = threadIdx.x & 31, o = lane >> 3, j = lane & 7;
    const int n_rows = 2 * P.n_kv + P.n_q, n_chunks = (n_rows + 1) >> 1;
    const int64_t task = (int64_t)blockIdx.x * (kApThreads / 32) + (threadIdx.x >> 5);
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t pair = task / n_chunks;
    const int row = 2 * (int)(task - pair * n_chunks) + (o >> 1);
    const int64_t tok = 2 * pair + (o & 1);
    const bool there = tok < P.n_tok && row < n_rows;
    const bool is_k = row < P.n_kv, is_q = row >= 2 * P.n_kv;
    const int head = is_k ? row : is_q ? row - 2 * P.n_kv : row - P.n_kv;
    float x[4][4] = {};
    int64_t slot = -1;
    if (there) {
        const T* src = is_k ? reinterpret_cast<const T*>(P.k) + tok * P.k_st + head * P.k_sh
                     : is_q ? reinterpret_cast<const T*>(P.q) + tok * P.q_st + head * P.q_sh
                            : reinterpret_cast<const T*>(P.v) + tok * P.v_st + head * P.v_sh;
        slot = P.slots[tok];
        ap_load(src, j, x);
        if (P.cos && (is_k || is_q)) {
            int64_t p = P.positions[tok];
            if (p < 0 || p >= P.n_positions) {         // no angle for it: the row is not written, and the caller learns of it
                if (P.status && (slot >= 0)) *P.status = kStatusOverflow;
                p = 0;
                if (is_k) slot = -1;
            }
            float4 c[2], s[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                c[g] = *reinterpret_cast<const float4*>(P.cos + p * P.cs_st + 32 * g + 4 * j);
                s[g] = *reinterpret_cast<const float4*>(P.sin + p * P.cs_st + 32 * g + 4 * j);
            }
            ap_rotate(x, c, s);
        }
        if (is_q) {
            T* dst = reinterpret_cast<T*>(P.q_out) + (tok * P.n_q + head) * kHD;
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2*>(dst + 32 * g + 4 * j) = make_uint2(PgType<T>::down(x[g][0], x[g][1]), PgType<T>::down(x[g][2], x[g][3]));
        }
    }
    if (is_q) slot = -1;
    const int page_tok = P.units * kUnitTok;
    if (slot >= (int64_t)P.n_pages * page_tok) {
        if (P.status) *P.status = kStatusOverflow;
        slot = -1;
    }
    uint32_t word[4] = {0x8888u, 0x8888u, 0x8888u, 0x8888u};         // half-words 4 j .. 4 j + 3
    float scale[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float a = 0.f;
        bool nan = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a = fmaxf(a, fabsf(x[g][e]));
            nan |= x[g][e] != x[g][e];
        }
        if (nan) a = __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            const float b = __shfl_xor_sync(0xffffffffu, a, d);
            a = (a != a || b != b) ? __uint_as_float(0x7fffffffu) : fmaxf(a, b);
        }
        const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(a, 7.0f)));
        scale[g] = s != s ? s : fminf(fmaxf(s, kPgScaleMin), kPgScaleMax);
        if (s == s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float c = fminf(fmaxf(rintf(__fdiv_rn(x[g][e], scale[g])), -7.f), 7.f);
                word[e] = (word[e] & ~(0xfu << (4 * g))) | (uint32_t)((int)c + 8) << (4 * g);
            }
        }
    }
    if (slot < 0) return;
    const int64_t page = slot / page_tok;
    const int in_page = (int)(slot - page * page_tok), t = in_page & 15;
    uint8_t* u = P.pages + page * P.page_stride + head * P.head_stride + (in_page >> 4) * kUnitBytes;
    const uint32_t s01 = PgType<__nv_bfloat16>::down(scale[0], scale[1]), s23 = PgType<__nv_bfloat16>::down(scale[2], scale[3]);
    if (is_k) {
        *reinterpret_cast<uint2*>(u + 64 * t + 8 * j) = make_uint2(word[0] | word[1] << 16, word[2] | word[3] << 16);
        if (j == 0) *reinterpret_cast<uint2*>(u + kUnitKs + 8 * t) = make_uint2(s01, s23);
    } else {
        uint8_t* dst = u + kUnitV + 128 * (t >> 1) + 2 * (t & 1) + 16 * j;
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint16_t*>(dst + 4 * e) = (uint16_t)word[e];
        if (j == 0) *reinterpret_cast<uint2*>(u + kUnitVs + 8 * t) = make_uint2(s01, s23);
    }
}

struct RdParams {
    PgPool pool;
    const int64_t* slots;
    void *k, *v;              // (n_tok, n_kv, 128) contiguous
    int32_t n_tok, n_kv;
    int32_t* status;
};

// Eight lanes per row as above; the values are exact in fp16 and fp32, and rounded once to bf16.
template <typename T>
__global__ void __launch_bounds__(256) pg_read_kernel(const RdParams P) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 3;
    const int j = threadIdx.x & 7;
    const int64_t tok = r / (2 * P.n_kv);
    if (tok >= P.n_tok) return;
    const int row = (int)(r - tok * 2 * P.n_kv), head = row >> 1;
    const bool is_v = row & 1;
    int64_t slot = P.slots[tok];
    const int page_tok = P.pool.units * kUnitTok;
    if (slot >= (int64_t)P.pool.n_pages * page_tok) {
        if (P.status) *P.status = kStatusOverflow;
        slot = -1;
    }
    uint32_t w[4] = {0x8888u, 0x8888u, 0x8888u, 0x8888u};
    float scale[4] = {0.f, 0.f, 0.f, 0.f};
    if (slot >= 0) {
        const int64_t page = slot / page_tok;
        const int in_page = (int)(slot - page * page_tok), t = in_page & 15;
        const uint8_t* u = P.pool.pages + page * P.pool.page_stride + head * P.pool.head_stride + (in_page >> 4) * kUnitBytes;
        if (is_v) {
            const uint4 x = *reinterpret_cast<const uint4*>(u + kUnitV + 128 * (t >> 1) + 16 * j);
            const uint32_t sh = 16u * (t & 1);
            w[0] = x.x >> sh; w[1] = x.y >> sh; w[2] = x.z >> sh; w[3] = x.w >> sh;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(u + 64 * t + 8 * j);
            w[0] = x.x; w[1] = x.x >> 16; w[2] = x.y; w[3] = x.y >> 16;
        }
        const uint2 s = *reinterpret_cast<const uint2*>(u + (is_v ? kUnitVs : kUnitKs) + 8 * t);
        scale[0] = pg_lo(s.x); scale[1] = pg_hi(s.x); scale[2] = pg_lo(s.y); scale[3] = pg_hi(s.y);
    }
    T* dst = reinterpret_cast<T*>(is_v ? P.v : P.k) + (tok * P.n_kv + head) * kHD + 4 * j;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)((int)(w[e] >> (4 * g) & 15u) - 8) * scale[g];
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(dst + 32 * g) = make_float4(x[0], x[1], x[2], x[3]);
        else
            *reinterpret_cast<uint2*>(dst + 32 * g) = make_uint2(PgType<T>::down(x[0], x[1]), PgType<T>::down(x[2], x[3]));
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

extern "C" __attribute__((visibility("default"))) int bgtq_paged_append(
    uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots, const void* k,
    int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const void* q, int64_t q_st, int64_t q_sh, void* q_out,
    const float* rope_cos, const float* rope_sin, int64_t rope_st, const int64_t* positions, int32_t n_positions, int32_t n_tok,
    int32_t n_kv, int32_t n_q, int32_t flags, int32_t* status, void* stream) {
    if (n_tok < 0 || n_q < 0 || (flags & ~BGTQ_PAGED_BF16)) return BGTQ_E_BADARG;
    if (const int e = check_pool(pages, page_stride, head_stride, n_pages, page_tokens, n_kv)) return e;
    if (n_tok == 0) return BGTQ_OK;
    if (!slots || !k || !v || (q == nullptr) != (n_q == 0) || (q && !q_out) || !rope_cos != !rope_sin) return BGTQ_E_BADARG;
    if (rope_cos && (!positions || n_positions < 1)) return BGTQ_E_BADARG;
    if (q && !rope_cos) return BGTQ_E_BADARG;
    if (!aligned(k, 8) || !aligned(v, 8) || !aligned(q, 8) || !aligned(q_out, 8) || k_st % 4 || k_sh % 4 || v_st % 4 || v_sh % 4 ||
        q_st % 4 || q_sh % 4 || !aligned(rope_cos, 16) || !aligned(rope_sin, 16) || rope_st % 4)
        return BGTQ_E_ALIGN;
    ApParams P{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok, slots, k, v, q, k_st, k_sh, v_st, v_sh, q_st, q_sh, q_out,
               rope_cos, rope_sin, rope_st, positions, n_positions, n_tok, n_kv, n_q, status};
    const int64_t tasks = (int64_t)((n_tok + 1) / 2) * ((2 * n_kv + n_q + 1) / 2), blocks = (tasks + kApThreads / 32 - 1) / (kApThreads / 32);
    if (blocks > INT32_MAX) return BGTQ_E_TOOBIG;
    const auto kernel = (flags & BGTQ_PAGED_BF16) ? pg_append_kernel<__nv_bfloat16> : pg_append_kernel<__half>;
    return launch_kernel(kernel, dim3((unsigned)blocks), dim3(kApThreads), 0, (cudaStream_t)stream, true, P) == cudaSuccess ? BGTQ_OK
                                                                                                                            : BGTQ_E_LAUNCH;
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_read(
    const uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages, int32_t page_tokens, const int64_t* slots,
    int32_t n_tok, int32_t n_kv, void* k, void* v, int32_t flags, int32_t* status, void* stream) {
    if (n_tok < 0 || (flags & ~(BGTQ_PAGED_BF16 | BGTQ_PAGED_F32)) || flags == (BGTQ_PAGED_BF16 | BGTQ_PAGED_F32)) return BGTQ_E_BADARG;
    if (const int e = check_pool(pages, page_stride, head_stride, n_pages, page_tokens, n_kv)) return e;
    if (n_tok == 0) return BGTQ_OK;
    if (!slots || !k || !v) return BGTQ_E_BADARG;
    if (!aligned(k, 16) || !aligned(v, 16)) return BGTQ_E_ALIGN;
    RdParams P{{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok}, slots, k, v, n_tok, n_kv, status};
    const int64_t blocks = ((int64_t)n_tok * 2 * n_kv * 8 + 255) / 256;
    if (blocks > INT32_MAX) return BGTQ_E_TOOBIG;
    const auto kernel = (flags & BGTQ_PAGED_F32) ? pg_read_kernel<float> : (flags & BGTQ_PAGED_BF16) ? pg_read_kernel<__nv_bfloat16> : pg_read_kernel<__half>;
    return launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, true, P) == cudaSuccess ? BGTQ_OK : BGTQ_E_LAUNCH;
}
