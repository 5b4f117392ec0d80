// Attention of few query rows per (sequence, KV head) over the paged 4-bit cache, on mma.sync, straight from the packed codes.
//
//     S[t, col] = sum_g ks[t, g] * (sum_{d in g} q[col, d] (u[t, d] - 8)),   P = 2^(S f - M),
//     O[d, col] = sum_t P[t, col] vs[t, g(d)] (u[t, d] - 8),   out = O / sum_t P
//
// A column is one query row: a query head of the KV head's group in a decode step, (position, head) pairs of a chunk.  K's codes
// go to the tensor cores as they lie, as subnormal fp16 numbers u * 2^-20, and the eights are the accumulators' start; V's become
// u - 8 first (1024 + u or 1024 + 16 u by a mask, then one exact fp16 operation), because sums over tokens that carry the eights would lose
// them again to the accumulators' rounding.  Subnormal operands are aligned by their exponent field, not by their leading bit: u * 2^-24
// (one shift less per two pairs) cost S ten bits, u * 2^-20 costs six of twenty-four.  The K scales multiply the groups' sums, the
// V scales the weights.  Nothing is rounded but P * vs (fp16, as the product's operand; sums, maxima, scales and accumulators are fp32).
// Queries are brought to [2^13, 2^14) by a power of two each, so that bf16 queries of any magnitude are exact in fp16 too.
//
// P * vs <= 2^14 holds for every magnitude of V: a column's reference M is the running maximum of S f + log2(max_g vs), minus 6, and moves
// (O rescaled) only when a value exceeds it by 2^14.
//
// Work: the 32-token batches of all (sequence, block of columns, KV head) triples form one list, cut evenly over the CTAs; a CTA's
// eight warps take batches in turn, each with a ring of bulk copies of its own.  At a triple's end the warps' states are merged in shared
// memory; triples cut between CTAs are merged by a second launch.
#include "bgtq_paged_common.cuh"

namespace bgtq {
namespace {

constexpr int kPdWarps = 8, kPdThreads = 32 * kPdWarps;
constexpr int kBatchTok = 32;
constexpr int kBatchBytes = kBatchTok / kUnitTok * kUnitBytes;
constexpr int kPdStages = 3;
constexpr int kMinBatches = kPdWarps;             // a CTA's least share: one batch per warp
constexpr float kLift = 6.f, kReach = 14.f;       // log2 of P * vs at a reference's setting, and where it moves
constexpr int kOutRow = 132;                      // floats between columns of a warp's state in shared memory

struct PdParams {
    PgPool pool;
    const void* q;
    int64_t q_st, q_sh;              // elements
    const int32_t* table;
    int64_t tb_st;
    const int32_t* lens;
    const int32_t* cu_q;             // null: one query row per sequence
    int32_t table_cols, n_seq, n_tok, n_q, n_kv, gqa, causal, n_cta;
    float scale_log2;
    void* out;
    int64_t o_st, o_sh;
    float* lse;                      // (n_tok, n_q) or null
    float* part_o;                   // (2 n_cta, columns, 128)
    float2* part_ml;                 // (2 n_cta, columns): reference, denominator
    int32_t* status;
};

struct SeqInfo {
    int len, q0, n;                  // cached tokens, first query row, query rows
};

__device__ __forceinline__ SeqInfo pd_seq(const PdParams& P, int i) {
    SeqInfo s;
    const int64_t cap = (int64_t)P.table_cols * P.pool.units * kUnitTok;
    s.len = max(0, (int)min((int64_t)P.lens[i], cap));
    if (P.cu_q) {
        s.q0 = min(max(P.cu_q[i], 0), P.n_tok);
        s.n = max(0, min(P.cu_q[i + 1], P.n_tok) - s.q0);
    } else {
        s.q0 = i;
        s.n = 1;
    }
    return s;
}
template <int NT>
__device__ __forceinline__ uint32_t pd_work(const PdParams& P, const SeqInfo& s) {
    return (uint32_t)((s.len + kBatchTok - 1) / kBatchTok) * (uint32_t)P.n_kv * (uint32_t)((s.n * P.gqa + 8 * NT - 1) / (8 * NT));
}

struct ScanSmem {
    uint32_t warp_sum[32];
    uint32_t total, start;
    int32_t seq;
};

// Exclusive prefix of w over the block's threads; S.total = the sum.
__device__ __forceinline__ uint32_t block_scan(ScanSmem& S, uint32_t w) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) S.warp_sum[warp] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
        const uint32_t y = S.warp_sum[i];
        if (i < warp) before += y;
        all += y;
    }
    __syncthreads();
    S.total = all;
    return before + x - w;
}

// Total of the list and, for the position that `at` makes of it, the sequence that it lies in and where that one starts.
template <int NT, typename At>
__device__ __forceinline__ void pd_find(const PdParams& P, ScanSmem& S, uint32_t& total, int& seq, uint32_t& start, At at) {
    const int tid = threadIdx.x, step = blockDim.x;
    if (tid == 0) S.seq = -1;
    uint32_t w = 0, before = 0, sum = 0;
    for (int base = 0; base < P.n_seq; base += step) {
        const int i = base + tid;
        w = i < P.n_seq ? pd_work<NT>(P, pd_seq(P, i)) : 0u;
        before = sum + block_scan(S, w);
        __syncthreads();
        sum += S.total;
        __syncthreads();
    }
    total = sum;
    const uint32_t want = at(total);
    if (P.n_seq <= step) {
        if (w && before <= want && want - before < w) {
            S.seq = tid;
            S.start = before;
        }
    } else {
        sum = 0;
        for (int base = 0; base < P.n_seq; base += step) {
            const int i = base + tid;
            w = i < P.n_seq ? pd_work<NT>(P, pd_seq(P, i)) : 0u;
            before = sum + block_scan(S, w);
            if (w && before <= want && want - before < w) {
                S.seq = i;
                S.start = before;
            }
            __syncthreads();
            sum += S.total;
            __syncthreads();
        }
    }
    __syncthreads();
    seq = S.seq;
    start = S.start;
}

__device__ __forceinline__ uint32_t pd_share(uint32_t total, int n_cta) {
    return max((uint32_t)kMinBatches, (total + n_cta - 1) / n_cta);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
// D = A B + C with the column sums' start in C (rows alike)
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], float c0, float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1));
}
// The pair of codes of group G in a word as fp16: u * 2^-20
template <int G>
__device__ __forceinline__ uint32_t k_codes(uint32_t w) {
    return (G == 0 ? w << 4 : G == 1 ? w : G == 2 ? w >> 4 : w >> 8) & 0x00f000f0u;
}
// u - 8
template <int G>
__device__ __forceinline__ uint32_t v_codes(uint32_t w) {
    const uint32_t x = G >= 2 ? w >> 8 : w;
    uint32_t d;
    if (G & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"((x & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));   // / 16 - 72
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((x & 0x000f000fu) | 0x64006400u), "r"(0x64086408u));                             // - 1032
    return d;
}

template <int NT>
struct PdSmem {
    __align__(128) uint8_t ring[kPdWarps][kPdStages][kBatchBytes];       // at a triple's end: the warps' states
    __align__(8) uint64_t full[kPdWarps][kPdStages];
    float2 ml[kPdWarps][8 * NT];
    ScanSmem scan;
};

// One column block's queries as the products' operands, the accumulators' starts, and the factor from sums to logits.
template <int NT>
struct Query {
    uint32_t b[NT][4][4];            // [group][k-step half: words 0, 1 | 2, 3]
    float c[NT][4][2];               // -8 * sum of the group's operand, columns 2 c and 2 c + 1
    float f[NT][2];
};

template <int NT, typename T>
__device__ __forceinline__ void pd_query(const PdParams& P, Query<NT>& Q, const SeqInfo& s, int cb, int h, int r, int c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = (cb * NT + nt) * 8 + r, pos = row / P.gqa, hq = h * P.gqa + row - pos * P.gqa;
        const bool there = pos < s.n;
        const T* src = reinterpret_cast<const T*>(P.q) + (int64_t)(s.q0 + (there ? pos : 0)) * P.q_st + (there ? hq : 0) * P.q_sh + 8 * c;
        float x[4][8], top = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (there) w = *reinterpret_cast<const uint4*>(src + 32 * g);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 v = PgType<T>::up(ww[e]);
                x[g][2 * e] = v.x;
                x[g][2 * e + 1] = v.y;
                top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e with top * 2^e in [2^13, 2^14); a row of zeros, or with an infinity, stays as it is
        const int ex = (int)(__float_as_uint(top) >> 23) - 127;
        const int e = top > 0.f && ex < 128 ? 13 - ex : 0;
        const float up0 = __uint_as_float((uint32_t)(127 + e / 2) << 23), up1 = __uint_as_float((uint32_t)(127 + e - e / 2) << 23);
        const int fe = 20 - e;                                                         // (-120 .. 134, in two steps)
        const float fac = P.scale_log2 * __uint_as_float((uint32_t)(127 + fe / 2) << 23) * __uint_as_float((uint32_t)(127 + fe - fe / 2) << 23);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = pack_half2(x[g][2 * i] * up0 * up1, x[g][2 * i + 1] * up0 * up1);
                Q.b[nt][g][i] = w;
                const float2 v = PgType<__half>::up(w);
                sum += v.x + v.y;
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= -8.f * 9.5367431640625e-7f;                                      // 2^-20
            Q.c[nt][g][0] = __shfl_sync(0xffffffffu, sum, 8 * c);                   // (lane 4 * column holds column's)
            Q.c[nt][g][1] = __shfl_sync(0xffffffffu, sum, 8 * c + 4);
        }
        Q.f[nt][0] = __shfl_sync(0xffffffffu, fac, 8 * c);
        Q.f[nt][1] = __shfl_sync(0xffffffffu, fac, 8 * c + 4);
    }
}

template <int NT>
struct State {
    float o[NT][2][4][4];            // [i][n]: rows 32 n + 4 r + 2 i (+ 1), columns 2 c (+ 1)
    float m[NT][2], l[NT][2];
};

template <int N> struct Int { static constexpr int value = N; };
template <typename F> __device__ __forceinline__ void each_group(F f) { f(Int<0>{}); f(Int<1>{}); f(Int<2>{}); f(Int<3>{}); }

// 16 tokens at shared address u.  kEdge: some of them (tokens from `left` on of the sequence, from lim[] on of a column) are hidden.
template <int NT, bool kEdge>
__device__ __forceinline__ void pd_unit(uint32_t u, const Query<NT>& Q, State<NT>& st, int r, int c, int t0, int len, const int (&lim)[NT][2]) {
    float s[NT][4];
    {
        const uint32_t kb = u + r * 64 + c * 16;
        const uint4 x = lds128(kb), y = lds128(kb + 512);
        const uint2 ka = lds64(u + kUnitKs + r * 8), kc = lds64(u + kUnitKs + 64 + r * 8);
        const float sa[4] = {pg_lo(ka.x), pg_hi(ka.x), pg_lo(ka.y), pg_hi(ka.y)};
        const float sc[4] = {pg_lo(kc.x), pg_hi(kc.x), pg_lo(kc.y), pg_hi(kc.y)};
        each_group([&](auto gi) {
            constexpr int g = decltype(gi)::value;
            const uint32_t a0[4] = {k_codes<g>(x.x), k_codes<g>(y.x), k_codes<g>(x.y), k_codes<g>(y.y)};
            const uint32_t a1[4] = {k_codes<g>(x.z), k_codes<g>(y.z), k_codes<g>(x.w), k_codes<g>(y.w)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float acc[4];
                const uint32_t b0[2] = {Q.b[nt][g][0], Q.b[nt][g][1]}, b1[2] = {Q.b[nt][g][2], Q.b[nt][g][3]};
                mma_from(acc, a0, b0, Q.c[nt][g][0], Q.c[nt][g][1]);
                mma_16816(acc, a1, b1);
                if (g == 0) {
                    s[nt][0] = acc[0] * sa[g]; s[nt][1] = acc[1] * sa[g];
                    s[nt][2] = acc[2] * sc[g]; s[nt][3] = acc[3] * sc[g];
                } else {
                    s[nt][0] = fmaf(acc[0], sa[g], s[nt][0]); s[nt][1] = fmaf(acc[1], sa[g], s[nt][1]);
                    s[nt][2] = fmaf(acc[2], sc[g], s[nt][2]); s[nt][3] = fmaf(acc[3], sc[g], s[nt][3]);
                }
            }
        });
    }
    uint2 va = lds64(u + kUnitVs + r * 8), vc = lds64(u + kUnitVs + 64 + r * 8);
    if (kEdge) {
        if (t0 + r >= len) va = make_uint2(0, 0);               // what lies behind the sequence may be anything
        if (t0 + 8 + r >= len) vc = make_uint2(0, 0);
    }
    const float ha[4] = {pg_lo(va.x), pg_hi(va.x), pg_lo(va.y), pg_hi(va.y)};
    const float hc[4] = {pg_lo(vc.x), pg_hi(vc.x), pg_lo(vc.y), pg_hi(vc.y)};
    const float la = lg2(fmaxf(fmaxf(fmaxf(ha[0], ha[1]), fmaxf(ha[2], ha[3])), kPgScaleMin));
    const float lc = lg2(fmaxf(fmaxf(fmaxf(hc[0], hc[1]), fmaxf(hc[2], hc[3])), kPgScaleMin));
    float top[NT][2];
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (kEdge) {
                if (t0 + r >= lim[nt][e]) s[nt][e] = -INFINITY;
                if (t0 + 8 + r >= lim[nt][e]) s[nt][2 + e] = -INFINITY;
            }
            top[nt][e] = fmaxf(fmaf(s[nt][e], Q.f[nt][e], la), fmaf(s[nt][2 + e], Q.f[nt][e], lc));
            move |= top[nt][e] > st.m[nt][e] + kReach;
        }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = top[nt][e];
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                const float m = fmaxf(st.m[nt][e], t - kLift);
                const float alpha = m == -INFINITY ? 1.f : ex2(st.m[nt][e] - m);
                st.m[nt][e] = m;
                st.l[nt][e] *= alpha;
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        st.o[nt][i][n][e] *= alpha;
                        st.o[nt][i][n][2 + e] *= alpha;
                    }
            }
    }
    float p[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float z = kEdge && st.m[nt][e] == -INFINITY ? 0.f : st.m[nt][e];
            p[nt][e] = ex2(fmaf(s[nt][e], Q.f[nt][e], -z));
            p[nt][2 + e] = ex2(fmaf(s[nt][2 + e], Q.f[nt][e], -z));
            st.l[nt][e] += p[nt][e] + p[nt][2 + e];
        }
    const uint32_t vb = u + kUnitV + c * 128 + r * 16;
    const uint4 x = lds128(vb), y = lds128(vb + 512);
    each_group([&](auto gi) {
        constexpr int g = decltype(gi)::value;
        const uint32_t a0[4] = {v_codes<g>(x.x), v_codes<g>(x.y), v_codes<g>(y.x), v_codes<g>(y.y)};
        const uint32_t a1[4] = {v_codes<g>(x.z), v_codes<g>(x.w), v_codes<g>(y.z), v_codes<g>(y.w)};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[4] = {p[nt][0] * ha[g], p[nt][1] * ha[g], p[nt][2] * hc[g], p[nt][3] * hc[g]};
            if (kEdge) {                                        // (a hidden token's scale may be no number)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = s[nt][e] == -INFINITY ? 0.f : w[e];
            }
            const uint32_t b[2] = {movmatrix_trans(pack_half2(w[0], w[1])), movmatrix_trans(pack_half2(w[2], w[3]))};
            mma_16816(st.o[nt][0][g], a0, b);
            mma_16816(st.o[nt][1][g], a1, b);
        }
    });
}

// Writes a column's row: four dims per lane.
template <typename T>
__device__ __forceinline__ void pd_write(const PdParams& P, const SeqInfo& s, int cb, int cols, int col, int h, int lane, float4 o, float m, float l) {
    const int row = cb * cols + col, pos = row / P.gqa;
    if (pos >= s.n) return;
    const int hq = h * P.gqa + row - pos * P.gqa;
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;         // (a NaN stays one)
    T* dst = reinterpret_cast<T*>(P.out) + (int64_t)(s.q0 + pos) * P.o_st + hq * P.o_sh + 4 * lane;
    *reinterpret_cast<uint2*>(dst) = make_uint2(PgType<T>::down(o.x * inv, o.y * inv), PgType<T>::down(o.z * inv, o.w * inv));
    if (P.lse && lane == 0) P.lse[(int64_t)(s.q0 + pos) * P.n_q + hq] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

template <int NT, typename T>
__global__ void __launch_bounds__(kPdThreads, NT == 1 ? 2 : 1) pg_attend_kernel(const PdParams P) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PdSmem<NT>& S = *reinterpret_cast<PdSmem<NT>*>(smem_raw);
    constexpr int kCols = 8 * NT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    if (tid < kPdWarps * kPdStages) mbar_init(&S.full[0][0] + tid, 1);
    if (tid == 0) mbar_fence_init();
    grid_launch_dependents();
    grid_dependency_wait();
    uint32_t total, seq_start, share = 0;
    int seq;
    pd_find<NT>(P, S.scan, total, seq, seq_start, [&](uint32_t t) {
        share = pd_share(t, P.n_cta);
        return (uint32_t)blockIdx.x * share;
    });
    const uint64_t begin = (uint64_t)blockIdx.x * share;
    if (begin >= total || seq < 0) return;
    uint32_t pos = (uint32_t)begin;
    const uint32_t end = (uint32_t)min((uint64_t)total, begin + share);
    uint32_t issued = 0, taken = 0;        // this warp's copies so far
    bool ok = true;
    const uint32_t ring0 = smem_u32(S.ring[warp][0]);
    const uint64_t policy = l2_evict_first_policy();

    SeqInfo s = pd_seq(P, seq);
    while (pos < end) {
        const uint32_t nb = (uint32_t)((s.len + kBatchTok - 1) / kBatchTok);
        if (nb == 0) break;              // (row ranges that do not follow one another: the list is not one then)
        const uint32_t triple = (pos - seq_start) / nb, first = (pos - seq_start) - triple * nb;
        const uint32_t count = min(nb - first, end - pos);
        const int cb = (int)(triple / P.n_kv), h = (int)(triple - (uint32_t)cb * P.n_kv);
        // columns' limits
        int lim[NT][2], lim_min = INT_MAX, lim_max = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = cb * kCols + 8 * nt + 2 * c + e, qp = row / P.gqa;
                lim[nt][e] = qp >= s.n ? 0 : P.causal ? max(0, min(s.len, s.len - s.n + 1 + qp)) : s.len;
            }
        {
            const int row1 = min(cb * kCols + kCols, s.n * P.gqa) - 1;
            lim_max = P.causal ? max(0, s.len - s.n + 1 + row1 / P.gqa) : s.len;
            lim_min = row1 + 1 < cb * kCols + kCols ? 0 : P.causal ? max(0, s.len - s.n + 1 + cb * kCols / P.gqa) : s.len;
        }
        const int n_batch = min((int)count, max(0, (lim_max + kBatchTok - 1) / kBatchTok - (int)first));
        const int n_my = (n_batch - warp + kPdWarps - 1) / kPdWarps;      // batches first + warp, + 8, ...
        const int n_units = (s.len + kUnitTok - 1) / kUnitTok;
        int page_of = -1;                                                 // lane i: page of unit i % 2 of batch 16 * block + i / 2
        auto load_pages = [&](int k0) {
            const int k = k0 + (lane >> 1), unit = 2 * ((int)first + warp + kPdWarps * k) + (lane & 1);
            page_of = -1;
            if (k < n_my && unit < n_units) {
                page_of = P.table[(int64_t)seq * P.tb_st + unit / P.pool.units];
                if (page_of < 0 || page_of >= P.pool.n_pages) {
                    page_of = -1;
                    if (P.status) *P.status = kStatusBadPage;
                }
            }
        };
        uint32_t have[kPdStages] = {};                                    // which of a stage's two units are there
        auto issue = [&](int k) {
            if ((k & 15) == 0) load_pages(k);
            const int page = __shfl_sync(0xffffffffu, page_of, 2 * (k & 15) + (lane & 1));
            const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & 3u;
            const int stage = issued % kPdStages;
            uint64_t* bar = &S.full[warp][stage];
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)__popc(there) * kUnitBytes);
            __syncwarp();
            if (lane < 2 && page >= 0) {
                const int unit = 2 * ((int)first + warp + kPdWarps * k) + lane;
                bulk_g2s_hint(S.ring[warp][stage] + lane * kUnitBytes,
                              P.pool.pages + (int64_t)page * P.pool.page_stride + (int64_t)h * P.pool.head_stride + (unit % P.pool.units) * kUnitBytes,
                              kUnitBytes, bar, policy);
            }
#pragma unroll
            for (int i = 0; i < kPdStages; ++i)
                if (i == stage) have[i] = there;
            ++issued;
        };
        if (ok)
            for (int k = 0; k < min(n_my, kPdStages); ++k) issue(k);
        Query<NT> Q;
        pd_query<NT, T>(P, Q, s, cb, h, r, c);
        State<NT> st = {};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) st.m[nt][0] = st.m[nt][1] = -INFINITY;
        for (int k = 0; k < n_my && ok; ++k) {
            const int stage = taken % kPdStages;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&S.full[warp][stage], (taken / kPdStages) & 1u))) {
                ok = false;
                break;
            }
            ++taken;
            uint32_t there = 0;
#pragma unroll
            for (int i = 0; i < kPdStages; ++i)
                if (i == stage) there = have[i];
            const int t0 = ((int)first + warp + kPdWarps * k) * kBatchTok;
            const uint32_t at = ring0 + stage * kBatchBytes;
            if (there == 3u && t0 + kBatchTok <= lim_min) {
                pd_unit<NT, false>(at, Q, st, r, c, t0, s.len, lim);
                pd_unit<NT, false>(at + kUnitBytes, Q, st, r, c, t0 + kUnitTok, s.len, lim);
            } else {
#pragma unroll 1
                for (int i = 0; i < 2; ++i)
                    if (there >> i & 1u) pd_unit<NT, true>(at + i * kUnitBytes, Q, st, r, c, t0 + i * kUnitTok, s.len, lim);
            }
            __syncwarp();
            if (k + kPdStages < n_my) issue(k + kPdStages);
        }
        if (!ok)             // copies in flight land before the ring is used again
            for (; taken < issued; ++taken) mbar_wait_bounded(&S.full[warp][taken % kPdStages], (taken / kPdStages) & 1u);
        // ---- the warps' states into shared memory (each into its own ring), merged by column ----
        float* const mine = reinterpret_cast<float*>(S.ring[warp][0]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = st.l[nt][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                const int col = 8 * nt + 2 * c + e;
                if (r == 0) S.ml[warp][col] = make_float2(st.m[nt][e], l);
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    *reinterpret_cast<float4*>(mine + col * kOutRow + 32 * n + 4 * r) =
                        make_float4(st.o[nt][0][n][e], st.o[nt][0][n][2 + e], st.o[nt][1][n][e], st.o[nt][1][n][2 + e]);
            }
        __syncthreads();
        const bool whole = first == 0 && count == nb;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = 8 * nt + warp;
            float m = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kPdWarps; ++w) m = fmaxf(m, S.ml[w][col].x);
            const float z = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < kPdWarps; ++w) {
                const float2 ml = S.ml[w][col];
                const float f = ex2(ml.x - z);
                const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(S.ring[w][0]) + col * kOutRow + 4 * lane);
                l = fmaf(f, ml.y, l);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
            if (whole) {
                pd_write<T>(P, s, cb, kCols, col, h, lane, o, m, l);
            } else {
                const size_t slot = (size_t)(2 * blockIdx.x + (pos == (uint32_t)begin ? 0 : 1)) * kCols + col;
                *reinterpret_cast<float4*>(P.part_o + slot * kHD + 4 * lane) = o;
                if (lane == 0) P.part_ml[slot] = make_float2(m, l);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the ring: generic accesses, then bulk copies
        __syncthreads();
        pos += count;
        while (pos < end && pos - seq_start >= pd_work<NT>(P, s)) {
            if (seq + 1 >= P.n_seq) {
                pos = end;
                break;
            }
            seq_start += pd_work<NT>(P, s);
            s = pd_seq(P, ++seq);
        }
    }
    if (!ok && lane == 0 && P.status) *P.status = kStatusWaitTimeout;
}

// Block i: the triple that the end of CTA i's share cuts, if that is its first cut; and the rows of every n_cta-th sequence that has none
// of its tokens cached.
template <int NT, typename T>
__global__ void __launch_bounds__(512) pg_merge_kernel(const PdParams P) {
    __shared__ ScanSmem scan;
    __shared__ float4 sum_o[16][32];
    __shared__ float sum_l[16];
    constexpr int kCols = 8 * NT, kPer = 16 / 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_launch_dependents();
    grid_dependency_wait();
    for (int i = blockIdx.x; i < P.n_seq; i += gridDim.x) {
        const SeqInfo s = pd_seq(P, i);
        if (s.len > 0) continue;
        for (int row = warp; row < s.n * P.n_q; row += 16) {
            const int pos = row / P.n_q, hq = row - pos * P.n_q;
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(P.out) + (int64_t)(s.q0 + pos) * P.o_st + hq * P.o_sh + 4 * lane) = make_uint2(0, 0);
            if (P.lse && lane == 0) P.lse[(int64_t)(s.q0 + pos) * P.n_q + hq] = -INFINITY;
        }
    }
    uint32_t total, seq_start, share = 0;
    int seq;
    pd_find<NT>(P, scan, total, seq, seq_start, [&](uint32_t t) {
        share = pd_share(t, P.n_cta);
        return ((uint32_t)blockIdx.x + 1) * share;
    });
    const uint64_t cut = ((uint64_t)blockIdx.x + 1) * share;
    if (cut >= total || seq < 0) return;
    const SeqInfo s = pd_seq(P, seq);
    const uint32_t nb = (uint32_t)((s.len + kBatchTok - 1) / kBatchTok);
    const uint32_t triple = ((uint32_t)cut - seq_start) / nb, a = seq_start + triple * nb, b = a + nb;
    if (a == (uint32_t)cut || a + share < (uint32_t)cut) return;              // not cut here, or not for the first time
    const int cb = (int)(triple / P.n_kv), h = (int)(triple - (uint32_t)cb * P.n_kv);
    const int j0 = blockIdx.x, j1 = min(P.n_cta - 1, (int)((b - 1) / share));                   // CTAs that hold a part of it
    auto slot_of = [&](int j) { return (size_t)(2 * j + (j == j0 && a != (uint32_t)j0 * share ? 1 : 0)) * kCols; };
    const int part = warp & (kPer - 1);
    for (int nt = 0; nt < NT; ++nt) {
        const int col = 8 * nt + (warp / kPer);
        float m = -INFINITY;
        for (int j = j0 + lane; j <= j1; j += 32) m = fmaxf(m, P.part_ml[slot_of(j) + col].x);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float z = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int j = j0 + part; j <= j1; j += kPer) {
            const float2 ml = P.part_ml[slot_of(j) + col];
            const float4 v = *reinterpret_cast<const float4*>(P.part_o + (slot_of(j) + col) * kHD + 4 * lane);
            const float f = ex2(ml.x - z);
            l = fmaf(f, ml.y, l);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
        sum_o[warp][lane] = o;
        if (lane == 0) sum_l[warp] = l;
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int i = 1; i < kPer; ++i) {
                const float4 v = sum_o[warp + i][lane];
                o.x += v.x; o.y += v.y; o.z += v.z; o.w += v.w;
                l += sum_l[warp + i];
            }
            pd_write<T>(P, s, cb, kCols, col, h, lane, o, m, l);
        }
        __syncthreads();
    }
}

template <int NT, typename T>
int pd_launch(const PdParams& P, cudaStream_t stream) {
    const int smem = (int)sizeof(PdSmem<NT>);
    if (cudaFuncSetAttribute(pg_attend_kernel<NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return BGTQ_E_LAUNCH;
    if (launch_kernel(pg_attend_kernel<NT, T>, dim3(P.n_cta), dim3(kPdThreads), smem, stream, true, P) != cudaSuccess) return BGTQ_E_LAUNCH;
    return launch_kernel(pg_merge_kernel<NT, T>, dim3(P.n_cta), dim3(512), 0, stream, true, P) == cudaSuccess ? BGTQ_OK : BGTQ_E_LAUNCH;
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// CTAs of a launch: as many as are resident at once, no more than there can be shares of sequences of max_tokens.
int pd_grid(int nt, int64_t blocks, int32_t n_kv, int64_t max_tokens) {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const double batches = (double)blocks * n_kv * (double)((max_tokens + kBatchTok - 1) / kBatchTok);
    if (batches > 2.0e9) return (nt == 1 ? 2 : 1) * sms;
    const int64_t most = ((int64_t)batches + kMinBatches - 1) / kMinBatches, resident = (nt == 1 ? 2 : 1) * sms;
    return (int)(most < 1 ? 1 : most < resident ? most : resident);
}

}  // namespace
}  // namespace bgtq

using namespace bgtq;

// Column tiles of a product: eight query rows are the operand's width; more of them share what is read and unpacked.
static int pd_tiles(int32_t n_q, int32_t n_kv, int32_t max_q) { return (int64_t)max_q * (n_q / n_kv) <= 8 ? 1 : 2; }

// Column blocks of all sequences, at most.
static int64_t pd_blocks(int nt, int32_t n_seq, int32_t n_tok, int32_t gqa) {
    return n_tok <= n_seq ? n_seq : (int64_t)n_tok * gqa / (8 * nt) + n_seq;
}

extern "C" __attribute__((visibility("default"))) int64_t bgtq_paged_workspace_bytes(int32_t n_seq, int32_t n_tok, int32_t n_q, int32_t n_kv,
                                                                                      int32_t max_q, int64_t max_tokens) {
    if (n_seq < 0 || n_tok < 0 || n_kv < 1 || n_q < 1 || n_q % n_kv || max_q < 1 || max_tokens < 0) return BGTQ_E_BADARG;
    if (n_q / n_kv > 8) return BGTQ_E_UNSUPPORTED;
    const int nt = pd_tiles(n_q, n_kv, max_q);
    return (int64_t)pd_grid(nt, pd_blocks(nt, n_seq, n_tok, n_q / n_kv), n_kv, max_tokens) * 2 * 8 * nt * (kHD * 4 + 8);
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_attend(
    const void* q, int64_t q_st, int64_t q_sh, const uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages,
    int32_t page_tokens, const int32_t* table, int64_t table_stride, int32_t table_cols, const int32_t* seq_lens, const int32_t* cu_q,
    int32_t n_seq, int32_t n_tok, int32_t n_q, int32_t n_kv, int32_t max_q, int64_t max_tokens, float scale, int32_t flags,
    void* workspace, int64_t workspace_bytes, void* out, int64_t o_st, int64_t o_sh, float* lse, int32_t* status, void* stream) {
    if (n_seq < 0 || n_tok < 0 || n_kv < 1 || n_q < 1 || table_cols < 0 || max_q < 1 || max_tokens < 0 ||
        (flags & ~(BGTQ_PAGED_BF16 | BGTQ_PAGED_CAUSAL)))
        return BGTQ_E_BADARG;
    if (!(scale == scale) || n_q % n_kv) return BGTQ_E_BADARG;
    if (n_q / n_kv > 8) return BGTQ_E_UNSUPPORTED;
    if (!cu_q && (n_tok != n_seq || max_q != 1)) return BGTQ_E_BADARG;
    if (n_seq == 0 || n_tok == 0) return BGTQ_OK;
    if (!pages || n_pages < 1 || page_tokens < kUnitTok || page_tokens % kUnitTok || !q || !out || !seq_lens || (!table && table_cols > 0))
        return BGTQ_E_BADARG;
    const int64_t cap = (int64_t)table_cols * page_tokens;
    if (cap > INT32_MAX - 64) return BGTQ_E_TOOBIG;
    if (!aligned(pages, 16) || page_stride % 16 || head_stride % 16 || !aligned(q, 16) || q_st % 8 || q_sh % 8 || !aligned(out, 8) || o_st % 4 ||
        o_sh % 4 || !aligned(workspace, 16))
        return BGTQ_E_ALIGN;
    const int nt = pd_tiles(n_q, n_kv, max_q);
    const int64_t cols = 8 * nt, blocks = pd_blocks(nt, n_seq, n_tok, n_q / n_kv);
    if ((double)blocks * n_kv * (double)((cap + kBatchTok - 1) / kBatchTok) > 2.0e9) return BGTQ_E_TOOBIG;      // (the list's 32 bits)
    const int n_cta = pd_grid(nt, blocks, n_kv, max_tokens);
    const int64_t need = (int64_t)n_cta * 2 * cols * (kHD * 4 + 8);
    if (!workspace || workspace_bytes < need) return BGTQ_E_BADARG;
    PdParams P{{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok}, q, q_st, q_sh, table, table_stride, seq_lens, cu_q,
               table_cols, n_seq, n_tok, n_q, n_kv, n_q / n_kv, !cu_q || (flags & BGTQ_PAGED_CAUSAL) ? 1 : 0, n_cta,
               scale * 1.44269504088896340736f, out, o_st, o_sh, lse, reinterpret_cast<float*>(workspace),
               reinterpret_cast<float2*>(reinterpret_cast<float*>(workspace) + (int64_t)n_cta * 2 * cols * kHD), status};
    const cudaStream_t st = (cudaStream_t)stream;
    const bool bf16 = flags & BGTQ_PAGED_BF16;
    if (nt == 1) return bf16 ? pd_launch<1, __nv_bfloat16>(P, st) : pd_launch<1, __half>(P, st);
    return bf16 ? pd_launch<2, __nv_bfloat16>(P, st) : pd_launch<2, __half>(P, st);
}
