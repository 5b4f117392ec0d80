// Attention of few query rows per (sequence, KV head) over the paged 4-bit cache, on mma.sync, straight from the packed codes.
//
//     S[t, col] = sum_g ks[t, g] * (sum_{d in g} q[col, d] (u[t, d] - 8)),   P = 2^(S f - M),
//     O[d, col] = sum_t P[t, col] * (vs[t, g(d)] (u[t, d] - 8)),   out = O / sum_t P
//
// A column is one query row: a query head of the KV head's group in a decode step, (position, head) pairs of a chunk.  Codes become
// u - 8 in fp16: a mask makes 1024 + u or 1024 + 16 u of two of them at once, one exact operation the rest.  (As subnormal numbers, u * 2^-24
// without that operation, with the eights in the accumulators' start or in a product of their own: operands are aligned by their exponent
// field, not by their leading bit, which cost ten bits of the sums; and over tokens the eights take theirs of the accumulators.)  The K scales
// multiply the groups' sums; V's operand is code * scale, exactly an fp16 number.  Nothing is rounded but P (fp16, as the product's operand; sums,
// maxima, scales and accumulators are fp32).  Queries are brought to [2^13, 2^14) by a power of two each, so that bf16 queries of any
// magnitude are exact in fp16 too.
//
// P <= 2^15: a column's reference M is 12 below its largest S f, and moves (O rescaled) only when a logit passes the largest by more than 3.  The
// weight of the token that set the reference is then a power of two: where one token has nearly all the weight, as in a sequence of one, its values
// come out as they are.  Weights below 2^-26 of the largest are subnormal in fp16, and cut at 2^-37 of it.  V's scales are not taken into the weights,
// although that saves a product per pair of codes: one token of large V, even one of hardly any weight, then pushes the others' weights out of
// fp16's range (values of 0.01 beside one of 65000, a token of zeros at 2^14 of their weight: their sum off by half).  (Moving at 1: 16 sequences of 2047
// tokens, 4 rows each, 21.1 us instead of 20.0; at 8, rows of one dominating token lie up to 1.5 times as far from 64 bits.)
//
// Work, in one of two forms:
//   split    the 32-token batches of all (sequence, block of columns, KV head) triples form one list, each triple headed by kTripleCost
//            places for what it costs beside them (a CTA with many short ones would come last), and the list is cut evenly over the
//            CTAs.  Triples cut between CTAs are merged by a second launch.  (Shares and triples of whole rounds of eight, as the warps
//            take them: 8 sequences of 32768 tokens x 2 KV heads 27.1 us instead of 26.1, 63 short ones beside one of 30000 tokens 27.8 instead of 25.5.)
//   cluster  a cluster of 1 to 8 CTAs per triple, which merge their shares in distributed shared memory: no list, no second launch.
// What bounds it: with long caches the warps' instructions, 339 for a unit of 16 tokens and one column tile (160 of them make operands, two for
// a pair of codes and a third for V's scales; 46 are the loop's), issued in 62 % of the cycles with no pipe more than half busy, 16 warps on
// an SM by their registers.  One sequence of 131072 tokens x 8 KV heads 41.0 us, 3.7 TB/s; 64 of 4500 85.0 us, 3.9 TB/s (loads alone, nothing
// computed: 27.8 and 57.4).  With short ones a launch and the chain length - page number - page - merging: 500 tokens 6.1 us, 4 sequences of 4099
// 8.5.  (The comparisons of forms and shares here and below were timed with V's scales in the weights, 2 to 8 % faster on either side.)
//
// In a CTA eight warps take batches in turn, each with a ring of bulk copies of its own (the next triple's first ones travel while this
// one's states are merged in shared memory).
#include "bgtq_paged_common.cuh"
#include "bgtq_paged_prefill.h"
#include "bgtq_paged_rows.h"

#include <limits.h>

namespace bgtq {
namespace {

constexpr int kPdWarps = 8, kPdThreads = 32 * kPdWarps;
constexpr int kBatchTok = 32;
constexpr int kBatchBytes = kBatchTok / kUnitTok * kUnitBytes;
// Places for what a triple costs beside its batches, a multiple of kPdWarps.  64 sequences of up to 9100 tokens x 8 KV heads: 110 us without,
// 91.4 with 8, 87.5 with 16, 89.4 with 24; 63 short ones beside one of 30000: 26.6, 27.9, 32.0.
constexpr uint32_t kTripleCost = 16;
constexpr float kLift = 12.f, kReach = 15.f;      // log2 of P at a reference's setting, and where it moves
constexpr int kOutRow = 132;                      // floats between columns of a warp's state in shared memory

struct PdParams {
    PgPool pool;
    const void* q;
    int64_t q_st, q_sh;              // elements
    const int32_t* table;
    int64_t tb_st;
    const int32_t* lens;
    const int32_t* cu_q;             // null: one query row per sequence
    int32_t cap, n_seq, n_tok, n_q, n_kv, gqa, causal;
    int32_t grain;                   // split: a triple's places and a CTA's share are multiples of it (1, or 8 where no triple may be cut)
    int32_t n_cta;                   // split: CTAs;  cluster: column blocks of a sequence that have a cluster of their own
    float scale_log2;
    void* out;
    int64_t o_st, o_sh;
    float* lse;                      // (n_tok, n_q) or null
    float* part_o;                   // (2 n_cta, columns, 128)
    float2* part_ml;                 // (2 n_cta, columns): reference, denominator
    int32_t* status;
};

// How a call is launched.
struct PdForm {
    int nt, n_cta, n_rank, blocks_of_seq;       // n_rank: CTAs of a triple's cluster, 0: the split form
    int64_t triples;
    bool merge;                                 // split: triples may be cut (those of one round never are)
    bool prefill;                               // the tcgen05 form
    bool alone;                                 // cluster: every CTA has an SM for itself
};

struct SeqInfo {
    int len, q0, n;                  // cached tokens, first query row, query rows
};

__device__ __forceinline__ SeqInfo pd_seq(const PdParams& P, int i) {
    SeqInfo s;
    s.len = max(0, min(P.lens[i], P.cap));
    if (P.cu_q) {
        s.q0 = min(max(P.cu_q[i], 0), P.n_tok);
        s.n = max(0, min(P.cu_q[i + 1], P.n_tok) - s.q0);
    } else {
        s.q0 = i;
        s.n = 1;
    }
    return s;
}
__device__ __forceinline__ uint32_t pd_batches(const SeqInfo& s) { return (uint32_t)((s.len + kBatchTok - 1) / kBatchTok); }
__device__ __forceinline__ uint32_t pd_whole(const PdParams& P, uint32_t n) { return (n + P.grain - 1) & ~(uint32_t)(P.grain - 1); }
__device__ __forceinline__ uint32_t pd_places(const PdParams& P, const SeqInfo& s) { return s.len > 0 ? pd_whole(P, pd_batches(s)) + kTripleCost : 0u; }
template <int NT>
__device__ __forceinline__ uint32_t pd_work(const PdParams& P, const SeqInfo& s) {
    return pd_places(P, s) * (uint32_t)P.n_kv * (uint32_t)((s.n * P.gqa + 8 * NT - 1) / (8 * NT));
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

// Total of the list and, for the position that `at` makes of it, the sequence that it lies in (-1: none) and where that one starts.  Up to 128
// sequences are looked over by every warp for itself, without a barrier.
template <int NT, typename At>
__device__ __forceinline__ void pd_find(const PdParams& P, ScanSmem& S, uint32_t& total, int& seq, uint32_t& start, At at) {
    const int tid = threadIdx.x, step = blockDim.x;
    if (P.n_seq <= 128) {
        const int lane = tid & 31;
        uint32_t w[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = 4 * lane + i < P.n_seq ? pd_work<NT>(P, pd_seq(P, 4 * lane + i)) : 0u;
            mine += w[i];
        }
        uint32_t before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += y;
        }
        total = __shfl_sync(0xffffffffu, before, 31);
        before -= mine;
        const uint32_t want = at(total);
        const uint32_t who = __ballot_sync(0xffffffffu, before <= want && want - before < mine);
        uint32_t first = before;
        int found = 4 * lane;
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (found == 4 * lane + i && want - first >= w[i]) {
                first += w[i];
                ++found;
            }
        seq = who ? __shfl_sync(0xffffffffu, found, __ffs(who) - 1) : -1;
        start = __shfl_sync(0xffffffffu, first, who ? __ffs(who) - 1 : 0);
        return;
    }
    if (tid == 0) S.seq = -1;
    uint32_t sum = 0;
    for (int base = 0; base < P.n_seq; base += step) {
        const int i = base + tid;
        block_scan(S, i < P.n_seq ? pd_work<NT>(P, pd_seq(P, i)) : 0u);
        __syncthreads();
        sum += S.total;
        __syncthreads();
    }
    total = sum;
    const uint32_t want = at(total);
    sum = 0;
    for (int base = 0; base < P.n_seq; base += step) {
        const int i = base + tid;
        const uint32_t w = i < P.n_seq ? pd_work<NT>(P, pd_seq(P, i)) : 0u;
        const uint32_t before = sum + block_scan(S, w);
        if (before <= want && want - before < w) {
            S.seq = i;
            S.start = before;
        }
        __syncthreads();
        sum += S.total;
        __syncthreads();
    }
    seq = S.seq;
    start = S.start;
}

// A CTA's share.  Short ones are whole rounds: the warps' chains are what they take (one sequence of 24000 tokens x 8 KV heads, 24 places instead
// of 21: 14.6 us instead of 15.2; of 12000, 16 instead of 11: 13.0 instead of 12.2).
__device__ __forceinline__ uint32_t pd_share(const PdParams& P, uint32_t total) {
    const uint32_t n = (total + P.n_cta - 1) / P.n_cta;
    return n <= 4 * kPdWarps ? (n + kPdWarps - 1) / kPdWarps * kPdWarps : pd_whole(P, n);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (as in bgtq_common.cuh, but not volatile: the compiler may move them among one another)
__device__ __forceinline__ void mma_acc(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma_new(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Two constants that one instruction takes beside a mask or a factor: held in registers (two of them cannot be immediates).
struct Magic {
    uint32_t k1024, m72;            // fp16 pairs
};
__device__ __forceinline__ Magic pd_magic() {
    Magic m;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(m.k1024));
    asm volatile("mov.b32 %0, 0xd480d480;" : "=r"(m.m72));
    return m;
}
// The pair of codes of group G in a word, w8 = w >> 8: u - 8 as fp16
template <int G>
__device__ __forceinline__ uint32_t codes(const Magic& m, uint32_t w, uint32_t w8) {
    uint32_t x, d;
    if (G & 1) {
        asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xEA;" : "=r"(x) : "r"(G >= 2 ? w8 : w), "r"(m.k1024));        // 1024 + 16 u
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0x2c002c00u), "r"(m.m72));               // / 16 - 72
    } else {
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xEA;" : "=r"(x) : "r"(G >= 2 ? w8 : w), "r"(m.k1024));        // 1024 + u
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0xe408e408u));                                // - 1032
    }
    return d;
}

template <int NT, int kStages>
struct PdSmem {
    __align__(128) uint8_t ring[kPdWarps][kStages][kBatchBytes];
    __align__(16) float o[kPdWarps][8 * NT][kOutRow];        // the warps' states at a triple's end
    float2 ml[kPdWarps][8 * NT];
    __align__(8) uint64_t full[kPdWarps][kStages];
    ScanSmem scan;
    // cluster form: [rank][8 NT columns][128] and [rank][8 NT] (reference, denominator) follow
};

// One column block's queries as the products' operands, and the factor from sums to logits (columns 2 c, 2 c + 1).
template <int NT>
struct Query {
    uint32_t b[NT][4][4];            // [group][words 0, 1 | 2, 3]
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
        float up0, up1, down0, down1;
        const int ex = pg_row_exponent(top);
        pg_pow2(ex, up0, up1);
        pg_pow2(-ex, down0, down1);
        float fac = fmaxf(fabsf(P.scale_log2) * down0 * down1, kPgFactorMin);
        if (P.scale_log2 < 0.f) up0 = -up0;  // (factors are positive: hidden logits are minus infinity before they meet one)
        if (P.scale_log2 == 0.f) {
            up0 = 0.f;
            fac = 1.f;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) Q.b[nt][g][i] = pack_half2(x[g][2 * i] * up0 * up1, x[g][2 * i + 1] * up0 * up1);
        Q.f[nt][0] = __shfl_sync(0xffffffffu, fac, 8 * c);
        Q.f[nt][1] = __shfl_sync(0xffffffffu, fac, 8 * c + 4);
    }
}

template <int NT>
struct State {
    float o[NT][2][4][4];            // [i][n]: rows 32 n + 4 r + 2 i (+ 1), columns 2 c (+ 1)
    float m[NT][2], l[NT][2];        // reference, denominator
    float top[NT][2];                // the largest logit that the reference allows
};

template <typename V> __device__ __forceinline__ V at(const uint8_t* p) { return *reinterpret_cast<const V*>(p); }
template <int N> struct Int { static constexpr int value = N; };
template <typename F> __device__ __forceinline__ void each_group(F f) { f(Int<0>{}); f(Int<1>{}); f(Int<2>{}); f(Int<3>{}); }

// A value of V that is no number, in a unit that some columns see only in part: as an operand it would reach all of them.  Its scale becomes zero,
// and the columns that see it become none.  s0, s1: scales of tokens t, t + 1, group c.
template <int NT>
__device__ __forceinline__ void pd_no_number(State<NT>& st, float& s0, float& s1, int t, int c, const int (&lim)[NT][2]) {
    const int first = s0 != s0 ? t : s1 != s1 ? t + 1 : INT_MAX;
    if (s0 != s0) s0 = 0.f;
    if (s1 != s1) s1 = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int first_g = __reduce_min_sync(0xffffffffu, c == g ? first : INT_MAX);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (first_g < lim[nt][e])
#pragma unroll
                    for (int i = 0; i < 2; ++i) st.o[nt][i][g][e] = st.o[nt][i][g][2 + e] = __uint_as_float(0x7fffffffu);
    }
}

// U units of 16 tokens at u in shared memory.  kEdge: some of them (tokens from len on of the sequence, from lim[] on of a column) are hidden.
template <int NT, int U, bool kEdge>
__device__ __forceinline__ void pd_units(const uint8_t* u, const Magic& mg, const Query<NT>& Q, State<NT>& st, int r, int c, int t0, int len, const int (&lim)[NT][2]) {
    float s[U][NT][4];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const uint8_t* const k = u + i * kUnitBytes;
        const uint4 x = at<uint4>(k + r * 64 + c * 16), y = at<uint4>(k + 512 + r * 64 + c * 16);
        const uint2 ka = at<uint2>(k + kUnitKs + r * 8), kc = at<uint2>(k + kUnitKs + 64 + r * 8);
        const float sa[4] = {pg_lo(ka.x), pg_hi(ka.x), pg_lo(ka.y), pg_hi(ka.y)};
        const float sc[4] = {pg_lo(kc.x), pg_hi(kc.x), pg_lo(kc.y), pg_hi(kc.y)};
        const uint4 x8 = make_uint4(x.x >> 8, x.y >> 8, x.z >> 8, x.w >> 8), y8 = make_uint4(y.x >> 8, y.y >> 8, y.z >> 8, y.w >> 8);
        each_group([&](auto gi) {
            constexpr int g = decltype(gi)::value;
            const uint32_t a0[4] = {codes<g>(mg, x.x, x8.x), codes<g>(mg, y.x, y8.x), codes<g>(mg, x.y, x8.y), codes<g>(mg, y.y, y8.y)};
            const uint32_t a1[4] = {codes<g>(mg, x.z, x8.z), codes<g>(mg, y.z, y8.z), codes<g>(mg, x.w, x8.w), codes<g>(mg, y.w, y8.w)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float acc[4];
                float(&d)[4] = s[i][nt];
                const uint32_t b0[2] = {Q.b[nt][g][0], Q.b[nt][g][1]}, b1[2] = {Q.b[nt][g][2], Q.b[nt][g][3]};
                mma_new(acc, a0, b0);
                mma_acc(acc, a1, b1);
                if (g == 0) {
                    d[0] = acc[0] * sa[g]; d[1] = acc[1] * sa[g];
                    d[2] = acc[2] * sc[g]; d[3] = acc[3] * sc[g];
                } else {
                    d[0] = fmaf(acc[0], sa[g], d[0]); d[1] = fmaf(acc[1], sa[g], d[1]);
                    d[2] = fmaf(acc[2], sc[g], d[2]); d[3] = fmaf(acc[3], sc[g], d[3]);
                }
            }
        });
    }
    // V's scales of a unit's tokens 2 r, 2 r + 1, group c, exact in fp16; the lanes get theirs from one another (11 instructions; 24 if each lane converted
    // its eight pairs for itself).  All of it ahead of the weights: between them and the products it is part of the warp's chain, 55.3 us instead of
    // 52.5 (16 sequences of 8192 tokens x 8 KV heads, a CTA each).
    uint32_t vs[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const uint8_t* const v = u + i * kUnitBytes + kUnitVs + 16 * r + 2 * c;
        float s0 = pg_lo(at<uint16_t>(v)), s1 = pg_lo(at<uint16_t>(v + 8));
        if (kEdge) {
            const int t = t0 + 16 * i + 2 * r;
            if (t >= len) s0 = 0.f;                                             // what lies behind the sequence may be anything
            if (t + 1 >= len) s1 = 0.f;
            if (__any_sync(0xffffffffu, s0 != s0 || s1 != s1)) pd_no_number<NT>(st, s0, s1, t, c, lim);
        }
        vs[i] = pack_half2(s0, s1);
    }
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (kEdge) {
                    if (t0 + 16 * i + r >= lim[nt][e]) s[i][nt][e] = -INFINITY;
                    if (t0 + 16 * i + 8 + r >= lim[nt][e]) s[i][nt][2 + e] = -INFINITY;
                }
                top[nt][e] = fmaxf(top[nt][e], fmaxf(s[i][nt][e], s[i][nt][2 + e]));
            }
    bool move = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[nt][e] *= Q.f[nt][e];
            move |= top[nt][e] > st.top[nt][e];
        }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = top[nt][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
                // (where fp32's steps are wider than these distances, they become none)
                const float m = fmaxf(st.m[nt][e], t - (t - kLift) > kReach ? t : t - kLift);
                const float alpha = m == -INFINITY ? 1.f : ex2(st.m[nt][e] - m);
                st.m[nt][e] = m;
                st.top[nt][e] = m + kReach - m > kReach ? m : m + kReach;
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
#pragma unroll
    for (int i = 0; i < U; ++i) {
        uint32_t sv[4][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            sv[g][0] = __shfl_sync(0xffffffffu, vs[i], 4 * c + g);
            sv[g][1] = __shfl_sync(0xffffffffu, vs[i], 4 * c + 16 + g);
        }
        uint32_t b[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float z = kEdge && st.m[nt][e] == -INFINITY ? 0.f : st.m[nt][e];
                // (product and difference rounded apart, as the references were: fused, logits beyond 2^26 differ from theirs by more than a weight's range)
                p[e] = ex2(__fmul_rn(s[i][nt][e], Q.f[nt][e]) - z);
                p[2 + e] = ex2(__fmul_rn(s[i][nt][2 + e], Q.f[nt][e]) - z);
                st.l[nt][e] += p[e] + p[2 + e];
            }
            b[nt][0] = transposed(pack_half2(p[0], p[1]));
            b[nt][1] = transposed(pack_half2(p[2], p[3]));
        }
        const uint8_t* const unit = u + i * kUnitBytes;
        const uint4 x = at<uint4>(unit + kUnitV + c * 128 + r * 16), y = at<uint4>(unit + kUnitV + 512 + c * 128 + r * 16);
        const uint4 x8 = make_uint4(x.x >> 8, x.y >> 8, x.z >> 8, x.w >> 8), y8 = make_uint4(y.x >> 8, y.y >> 8, y.z >> 8, y.w >> 8);
        each_group([&](auto gi) {
            constexpr int g = decltype(gi)::value;
            const uint32_t sx = sv[g][0], sy = sv[g][1];
            const uint32_t a0[4] = {hmul2_u32(codes<g>(mg, x.x, x8.x), sx), hmul2_u32(codes<g>(mg, x.y, x8.y), sx),
                                    hmul2_u32(codes<g>(mg, y.x, y8.x), sy), hmul2_u32(codes<g>(mg, y.y, y8.y), sy)};
            const uint32_t a1[4] = {hmul2_u32(codes<g>(mg, x.z, x8.z), sx), hmul2_u32(codes<g>(mg, x.w, x8.w), sx),
                                    hmul2_u32(codes<g>(mg, y.z, y8.z), sy), hmul2_u32(codes<g>(mg, y.w, y8.w), sy)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma_acc(st.o[nt][0][g], a0, b[nt]);
                mma_acc(st.o[nt][1][g], a1, b[nt]);
            }
        });
    }
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

// A run of batches of one triple.
struct Segment {
    SeqInfo s;
    int seq, cb, h, first, n;        // first batch, batches
    bool whole;                      // all of the triple's
};
// A warp's copies of its batches of a segment: first + warp, + 8, ...
struct Copies {
    const uint8_t* from;             // lane i: unit i % 2 of batch 16 * block + i / 2, null: not there
    int issued, n;
    uint32_t have;                   // two bits per stage: which of its units are there
    bool all;                        // the sixteen batches that `from` is about lack none
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

// kStages 2: two CTAs on an SM hide each other's latencies.  4: one CTA on an SM, alone with them.
template <int NT, typename T, bool kCluster, int kStages>
__global__ void __launch_bounds__(kPdThreads, NT == 1 ? 2 : 1) pg_attend_kernel(const PdParams P) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    using Smem = PdSmem<NT, kStages>;
    Smem& S = *reinterpret_cast<Smem*>(smem_raw);
    constexpr int kCols = 8 * NT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    if (lane < kStages) {                // each warp waits on its own
        mbar_init(&S.full[warp][lane], 1);
        mbar_fence_init();
    }
    __syncwarp();
    uint32_t rank = 0, n_rank = 1;
    if (kCluster) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n_rank));
        if (n_rank > 1) cluster_arrive();            // a CTA's shared memory may be written once that CTA runs
    }
    grid_dependency_wait();
    grid_launch_dependents();              // (behind the wait: what the merging launch reads ahead of its own is complete)

    Segment g;
    uint32_t pos = 0, end = 0, begin = 0, seq_start = 0;
    // split: the segment that starts at pos
    auto at_pos = [&]() {
        const uint32_t nb = pd_batches(g.s), np = pd_places(P, g.s), triple = (pos - seq_start) / np, at = (pos - seq_start) - triple * np;
        const uint32_t count = min(np - at, end - pos), to = at + count - min(at + count, kTripleCost);
        g.cb = (int)(triple / P.n_kv);
        g.h = (int)(triple - (uint32_t)g.cb * P.n_kv);
        g.first = (int)(at - min(at, kTripleCost));
        g.n = (int)min(to, nb) - g.first;
        g.whole = g.first == 0 && to >= nb;
        return count;
    };
    // cluster: this CTA's share of the triple
    auto share_of = [&]() {
        const uint32_t nb = pd_batches(g.s), per = (nb + kPdWarps - 1) / kPdWarps, a = per * rank / n_rank * kPdWarps, b = per * (rank + 1) / n_rank * kPdWarps;
        g.first = (int)a;
        g.n = (int)(min(b, nb) - min(a, nb));
        g.whole = true;
    };
    uint32_t count = 0;
    if (kCluster) {
        const uint32_t t = blockIdx.x / n_rank, per_seq = (uint32_t)P.n_kv * P.n_cta;
        g.seq = (int)(t / per_seq);
        const uint32_t in_seq = t - (uint32_t)g.seq * per_seq;
        g.cb = (int)(in_seq / P.n_kv);
        g.h = (int)(in_seq - (uint32_t)g.cb * P.n_kv);
        g.s = pd_seq(P, g.seq);
        if (g.cb * kCols >= g.s.n * P.gqa) {         // (the whole cluster)
            if (n_rank > 1) cluster_wait();
            return;
        }
        share_of();
    } else {
        // rows of sequences that have none of their tokens cached
        for (int i = blockIdx.x; i < P.n_seq; i += P.n_cta) {
            const SeqInfo s = pd_seq(P, i);
            if (s.len > 0) continue;
            for (int row = warp; row < s.n * P.n_q; row += kPdWarps) {
                const int qp = row / P.n_q, hq = row - qp * P.n_q;
                *reinterpret_cast<uint2*>(reinterpret_cast<T*>(P.out) + (int64_t)(s.q0 + qp) * P.o_st + hq * P.o_sh + 4 * lane) = make_uint2(0, 0);
                if (P.lse && lane == 0) P.lse[(int64_t)(s.q0 + qp) * P.n_q + hq] = -INFINITY;
            }
        }
        uint32_t total, share = 0;
        pd_find<NT>(P, S.scan, total, g.seq, seq_start, [&](uint32_t t) {
            share = pd_share(P, t);
            return (uint32_t)blockIdx.x * share;
        });
        if ((uint64_t)blockIdx.x * share >= total || g.seq < 0) return;
        begin = pos = blockIdx.x * share;
        end = (uint32_t)min((uint64_t)total, (uint64_t)begin + share);
        g.s = pd_seq(P, g.seq);
        if (g.s.len == 0) return;                    // (row ranges that do not follow one another: the list is not one then)
        count = at_pos();
        if (g.n <= 0) return;
    }

    uint32_t phases = 0;                   // of this warp's stages
    bool ok = true;
    const Magic mg = pd_magic();
    const uint64_t policy = l2_evict_first_policy();
    auto issue = [&](const Segment& sg, Copies& w, int stage) {
        const int k = w.issued++;
        if ((k & 15) == 0) {
            const int kk = k + (lane >> 1), unit = 2 * (sg.first + warp + kPdWarps * kk) + (lane & 1);
            w.from = nullptr;
            if (kk < w.n && unit < (sg.s.len + kUnitTok - 1) / kUnitTok) {
                const int col = unit / P.pool.units, page = P.table[(int64_t)sg.seq * P.tb_st + col];
                if (page >= 0 && page < P.pool.n_pages)
                    w.from = P.pool.pages + (int64_t)page * P.pool.page_stride + (int64_t)sg.h * P.pool.head_stride + (unit - col * P.pool.units) * kUnitBytes;
                else if (P.status)
                    *P.status = kStatusBadPage;
            }
            w.all = __all_sync(0xffffffffu, kk >= w.n || w.from);
        }
        uint64_t* bar = &S.full[warp][stage];
        uint32_t there = 3u;
        if (!w.all) there = __ballot_sync(0xffffffffu, w.from != nullptr) >> (2 * (k & 15)) & 3u;
        if (lane == 0) mbar_arrive_expect_tx(bar, w.all ? kBatchBytes : (uint32_t)__popc(there) * kUnitBytes);
        // (the lanes that hold the addresses; a copy that ends before the arrival finds the phase open all the same)
        if (lane >> 1 == (k & 15) && w.from) bulk_g2s_hint(S.ring[warp][stage] + (lane & 1) * kUnitBytes, w.from, kUnitBytes, bar, policy);
        w.have = (w.have & ~(3u << (2 * stage))) | there << (2 * stage);
    };
    auto begin_copies = [&](const Segment& sg) {
        Copies w{nullptr, 0, 0, 0, false};
        // batches that no row of the block sees are left out
        const int last_row = min((sg.cb + 1) * kCols, sg.s.n * P.gqa) - 1;
        const int lim_max = P.causal ? max(0, sg.s.len - sg.s.n + 1 + last_row / P.gqa) : sg.s.len;
        const int n = min(sg.n, max(0, (lim_max + kBatchTok - 1) / kBatchTok - sg.first));
        w.n = max(0, (n - warp + kPdWarps - 1) / kPdWarps);
        if (ok)
            while (w.issued < min(w.n, kStages)) issue(sg, w, w.issued);
        return w;
    };
    Copies w = begin_copies(g);
    while (true) {
        Query<NT> Q;
        pd_query<NT, T>(P, Q, g.s, g.cb, g.h, r, c);
        // columns' limits; columns behind the last row compute whatever they like
        const int n_rows = g.s.n * P.gqa, row0 = g.cb * kCols, behind = g.s.len - g.s.n + 1;
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = row0 + 8 * nt + 2 * c + e;
                lim[nt][e] = P.causal && row < n_rows ? max(0, behind + row / P.gqa) : g.s.len;
            }
        const int lim_min = P.causal ? max(0, behind + row0 / P.gqa) : g.s.len;
        State<NT> st = {};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) st.m[nt][0] = st.m[nt][1] = st.top[nt][0] = st.top[nt][1] = -INFINITY;
        int t0 = (g.first + warp) * kBatchTok, stage = 0;
        for (int k = 0; k < w.n && ok; ++k) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&S.full[warp][stage], phases >> stage & 1u))) {
                ok = false;
                break;
            }
            phases ^= 1u << stage;
            const uint8_t* const tile = S.ring[warp][stage];
            const uint32_t there = w.have >> (2 * stage) & 3u;
            if (there == 3u && t0 + kBatchTok <= lim_min) {
                if (NT == 1) {
                    pd_units<NT, 2, false>(tile, mg, Q, st, r, c, t0, g.s.len, lim);
                } else {
                    pd_units<NT, 1, false>(tile, mg, Q, st, r, c, t0, g.s.len, lim);
                    pd_units<NT, 1, false>(tile + kUnitBytes, mg, Q, st, r, c, t0 + kUnitTok, g.s.len, lim);
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < 2; ++i)
                    if (there >> i & 1u) pd_units<NT, 1, true>(tile + i * kUnitBytes, mg, Q, st, r, c, t0 + i * kUnitTok, g.s.len, lim);
            }
            __syncwarp();
            if (w.issued < w.n) issue(g, w, stage);
            t0 += kPdWarps * kBatchTok;
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        if (!ok)             // copies in flight land before the CTA leaves; nothing more is fetched
            for (int i = 0; i < kStages; ++i)
                if (i < w.issued) mbar_wait_bounded(&S.full[warp][i], phases >> i & 1u);
        // ---- what comes next, and its first copies ----
        Segment next = g;
        bool more = false;
        uint32_t next_count = 0;
        const uint32_t this_pos = pos;
        if (kCluster) {
            next.cb += P.n_cta;              // (only where a sequence has more rows than the caller said)
            more = next.cb * kCols < g.s.n * P.gqa;
        } else {
            pos += count;
            while (pos < end && pos - seq_start >= pd_work<NT>(P, next.s)) {
                if (next.seq + 1 >= P.n_seq) {
                    pos = end;
                    break;
                }
                seq_start += pd_work<NT>(P, next.s);
                next.s = pd_seq(P, ++next.seq);
            }
            more = pos < end;
            if (more) {
                const Segment keep = g;
                g = next;
                next_count = at_pos();
                next = g;
                g = keep;
                more = next.n > 0;           // (the share's end may fall behind a triple's head)
            }
        }
        if (more) w = begin_copies(next);
        // ---- the warps' states merged by column ----
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
                    *reinterpret_cast<float4*>(&S.o[warp][col][32 * n + 4 * r]) =
                        make_float4(st.o[nt][0][n][e], st.o[nt][0][n][2 + e], st.o[nt][1][n][e], st.o[nt][1][n][2 + e]);
            }
        __syncthreads();
        if (kCluster && n_rank > 1) cluster_wait();          // (every CTA runs, and has read what it got before)
        const uint32_t xo = smem_u32(smem_raw + sizeof(Smem)), xml = xo + n_rank * kCols * kHD * 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int col = 8 * nt + warp;
            if (row0 + col >= n_rows) continue;
            float m = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kPdWarps; ++i) m = fmaxf(m, S.ml[i][col].x);
            const float z = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < kPdWarps; ++i) {
                const float2 ml = S.ml[i][col];
                const float f = ex2(ml.x - z);
                const float4 v = *reinterpret_cast<const float4*>(&S.o[i][col][4 * lane]);
                l = fmaf(f, ml.y, l);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
            if (kCluster && n_rank > 1) {                    // to the CTA that finishes this column
                const uint32_t owner = (uint32_t)col % n_rank, row = rank * kCols + col;
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr(xo + row * kHD * 4 + 16 * lane, owner)), "f"(o.x),
                             "f"(o.y), "f"(o.z), "f"(o.w)
                             : "memory");
                if (lane == 0)
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr(xml + row * 8, owner)), "f"(m), "f"(l) : "memory");
            } else if (g.whole) {
                pd_write<T>(P, g.s, g.cb, kCols, col, g.h, lane, o, m, l);
            } else {
                const size_t slot = (size_t)(2 * blockIdx.x + (this_pos == begin ? 0 : 1)) * kCols + col;
                *reinterpret_cast<float4*>(P.part_o + slot * kHD + 4 * lane) = o;
                if (lane == 0) P.part_ml[slot] = make_float2(m, l);
            }
        }
        if (kCluster && n_rank > 1) {
            cluster_arrive();
            cluster_wait();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int col = 8 * nt + warp;
                if (row0 + col >= n_rows || (uint32_t)col % n_rank != rank) continue;
                const float* po = reinterpret_cast<const float*>(smem_raw + sizeof(Smem));
                const float2* pml = reinterpret_cast<const float2*>(po + n_rank * kCols * kHD);
                float m = -INFINITY, l = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                for (uint32_t i = 0; i < n_rank; ++i) m = fmaxf(m, pml[i * kCols + col].x);
                const float z = m == -INFINITY ? 0.f : m;
#pragma unroll 4
                for (uint32_t i = 0; i < n_rank; ++i) {
                    const float2 ml = pml[i * kCols + col];
                    const float f = ex2(ml.x - z);
                    const float4 v = *reinterpret_cast<const float4*>(po + (i * kCols + col) * kHD + 4 * lane);
                    l = fmaf(f, ml.y, l);
                    o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
                }
                pd_write<T>(P, g.s, g.cb, kCols, col, g.h, lane, o, m, l);
            }
        }
        if (!more) break;
        if (kCluster && n_rank > 1) cluster_arrive();
        __syncthreads();                                     // (the states are read)
        g = next;
        count = next_count;
    }
    if (!ok && lane == 0 && P.status) *P.status = kStatusWaitTimeout;
}

// Block (i, col): column col of a triple that is cut.  kByTriple (one query row per sequence, no more triples than CTAs): of triple i.  Otherwise of
// the one that the end of CTA i's share cuts, if that is its first cut.  kWarps warps share the partials, four of a warp's requested at a
// time.  Where the triples lie is looked up before the partials are there: the lengths were complete before the attention began.
template <int NT, typename T, bool kByTriple, int kWarps>
__global__ void __launch_bounds__(32 * kWarps) pg_merge_kernel(const PdParams P) {
    __shared__ ScanSmem scan;
    __shared__ float4 sum_o[kWarps][32];
    __shared__ float sum_l[kWarps];
    constexpr int kCols = 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y;
    grid_launch_dependents();
    uint32_t total, seq_start, share = 0, triple;
    int seq;
    if (kByTriple) {
        const int wanted = blockIdx.x / P.n_kv;
        uint32_t before = 0;
        for (int i = 0; i < wanted; i += 32)
            if (i + lane < wanted) before += pd_work<NT>(P, pd_seq(P, i + lane));
        uint32_t rest = 0;
        for (int i = wanted; i < P.n_seq; i += 32)
            if (i + lane < P.n_seq) rest += pd_work<NT>(P, pd_seq(P, i + lane));
        seq_start = __reduce_add_sync(0xffffffffu, before);
        total = seq_start + __reduce_add_sync(0xffffffffu, rest);
        share = pd_share(P, total);
        seq = wanted;
        triple = blockIdx.x - (uint32_t)wanted * P.n_kv;
    } else {
        pd_find<NT>(P, scan, total, seq, seq_start, [&](uint32_t t) {
            share = pd_share(P, t);
            return ((uint32_t)blockIdx.x + 1) * share;
        });
        if (((uint64_t)blockIdx.x + 1) * share >= total || seq < 0) seq = -1;
        triple = 0;
    }
    grid_dependency_wait();
    if (seq < 0) return;
    const SeqInfo s = pd_seq(P, seq);
    if (s.len == 0) return;
    const uint32_t np = pd_places(P, s);
    if (!kByTriple) triple = ((blockIdx.x + 1) * share - seq_start) / np;
    const uint32_t a = seq_start + triple * np, b = a + np;
    const int j0 = (int)((a + kTripleCost) / share), j1 = min(P.n_cta - 1, (int)((b - 1) / share));      // the CTAs that hold a part of it
    if (j0 >= j1 || (!kByTriple && j0 != (int)blockIdx.x)) return;                                       // not cut, or not for the first time
    const int cb = (int)(triple / P.n_kv), h = (int)(triple - (uint32_t)cb * P.n_kv);
    const size_t slot0 = (size_t)(2 * j0 + (a > (uint32_t)j0 * share ? 1 : 0)) * kCols + col;
    auto slot_of = [&](int j) { return j == j0 ? slot0 : (size_t)2 * j * kCols + col; };
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = j0 + warp; j <= j1; j += 4 * kWarps) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = j + kWarps * i <= j1;
            const size_t slot = there ? slot_of(j + kWarps * i) : slot0;
            ml[i] = P.part_ml[slot];
            v[i] = *reinterpret_cast<const float4*>(P.part_o + slot * kHD + 4 * lane);
            if (!there) {
                ml[i] = make_float2(-INFINITY, 0.f);
                v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        const float top = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
        const float z = top == -INFINITY ? 0.f : top, f0 = ex2(m - z);
        l *= f0;
        o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
        m = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = ex2(ml[i].x - z);
            l = fmaf(f, ml[i].y, l);
            o.x = fmaf(f, v[i].x, o.x); o.y = fmaf(f, v[i].y, o.y); o.z = fmaf(f, v[i].z, o.z); o.w = fmaf(f, v[i].w, o.w);
        }
    }
    __shared__ float sum_m[kWarps];
    sum_o[warp][lane] = o;
    if (lane == 0) {
        sum_l[warp] = l;
        sum_m[warp] = m;
    }
    __syncthreads();
    if (warp) return;
    m = -INFINITY;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = fmaxf(m, sum_m[i]);
    const float z = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const float f = ex2(sum_m[i] - z);
        const float4 v = sum_o[i][lane];
        l = fmaf(f, sum_l[i], l);
        o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
    }
    pd_write<T>(P, s, cb, kCols, col, h, lane, o, m, l);
}

template <int NT, typename T>
int pd_launch_split(const PdParams& P, bool merge, cudaStream_t stream) {
    constexpr int kStages = NT == 1 ? 2 : 4, smem = (int)sizeof(PdSmem<NT, kStages>);
    const auto kernel = pg_attend_kernel<NT, T, false, kStages>;
    static std::atomic<uint64_t> allowed{0};
    if (!pg_allow_smem(kernel, smem, allowed)) return BGTQ_E_LAUNCH;
    if (!pg_launch_ok(launch_kernel(kernel, dim3(P.n_cta), dim3(kPdThreads), smem, stream, true, P))) return BGTQ_E_LAUNCH;
    if (!merge) return BGTQ_OK;
    const int64_t triples = (int64_t)P.n_seq * P.n_kv;
    const bool by_triple = !P.cu_q && triples <= P.n_cta;
    const dim3 grid(by_triple ? (unsigned)triples : P.n_cta - 1, P.cu_q ? 8 * NT : P.gqa);
    // As many warps as take a triple's partials in one pass, but not more: 8 triples of 37 partials 15.3 us with 8, 14.6 with 16 (20000
    // tokens); 160 of two or three 15.5 with 8 and 19.7 with 16.
    const int warps = !by_triple || P.n_cta <= 4 * triples ? 2 : P.n_cta <= 16 * triples ? 8 : 16;
    const auto merging = !by_triple ? pg_merge_kernel<NT, T, false, 2>
                         : warps == 2 ? pg_merge_kernel<NT, T, true, 2> : warps == 8 ? pg_merge_kernel<NT, T, true, 8> : pg_merge_kernel<NT, T, true, 16>;
    return pg_launch_ok(launch_kernel(merging, grid, dim3(32 * warps), 0, stream, true, P)) ? BGTQ_OK : BGTQ_E_LAUNCH;
}
template <int NT, int kStages>
struct ClusterLaunch {
    static constexpr int kBase = (int)sizeof(PdSmem<NT, kStages>), kRow = 8 * NT * (kHD * 4 + 8);
    static_assert(kBase + 8 * kRow <= 227 * 1024, "a cluster of eight fits");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    ClusterLaunch(int64_t triples, int n_rank, cudaStream_t stream) {
        cfg.gridDim = dim3((unsigned)(triples * n_rank));
        cfg.blockDim = dim3(kPdThreads);
        cfg.dynamicSmemBytes = kBase + (n_rank > 1 ? n_rank * kRow : 0);
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = n_rank;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
    }
};
template <int NT, typename T, int kStages>
int pd_launch_cluster(const PdParams& P, int64_t triples, int n_rank, cudaStream_t stream) {
    const auto kernel = pg_attend_kernel<NT, T, true, kStages>;
    ClusterLaunch<NT, kStages> L(triples, n_rank, stream);
    static std::atomic<uint64_t> allowed{0};
    if (!pg_allow_smem(kernel, L.kBase + 8 * L.kRow, allowed)) return BGTQ_E_LAUNCH;
    return pg_launch_ok(cudaLaunchKernelEx(&L.cfg, kernel, P)) && cudaGetLastError() == cudaSuccess ? BGTQ_OK : BGTQ_E_LAUNCH;
}
// Clusters of n_rank CTAs, each with an SM for itself, that the device runs at once (its groups of SMs are no multiples of eight).
template <int NT, int kStages>
int pd_clusters(int n_rank, int dev) {
    static std::atomic<int> known[64][9];
    if (dev >= 0 && dev < 64)
        if (const int n = known[dev][n_rank].load(std::memory_order_relaxed)) return n;
    const auto kernel = pg_attend_kernel<NT, __half, true, kStages>;
    ClusterLaunch<NT, kStages> L(1, n_rank, nullptr);
    L.cfg.numAttrs = 1;
    static std::atomic<uint64_t> allowed{0};
    int n = 0;
    if (!pg_allow_smem(kernel, L.kBase + 8 * L.kRow, allowed) || cudaOccupancyMaxActiveClusters(&n, kernel, &L.cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (dev >= 0 && dev < 64) known[dev][n_rank].store(n, std::memory_order_relaxed);
    return n;
}
template <int NT, typename T>
int pd_launch(const PdParams& P, const PdForm& f, cudaStream_t stream) {
    if (!f.n_rank) return pd_launch_split<NT, T>(P, f.merge, stream);
    if (NT == 1 && f.alone) return pd_launch_cluster<NT, T, NT == 1 ? 4 : 2>(P, f.triples, f.n_rank, stream);
    return pd_launch_cluster<NT, T, 2>(P, f.triples, f.n_rank, stream);
}

bool aligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

}  // namespace
}  // namespace bgtq

using namespace bgtq;

// Column tiles of a product: eight query rows are the operand's width; more of them share what is read and unpacked.
static int pd_tiles(int32_t n_q, int32_t n_kv, int32_t max_q) { return (int64_t)max_q * (n_q / n_kv) <= 8 ? 1 : 2; }

// How a call is launched, from its shape: the form that the measured costs make the cheapest (in microseconds, 300 to 131072 tokens over 2 to 64
// KV heads and sequences; a round is 256 tokens of a CTA).  The lengths lie on the device: all that is known here is how many sequences there are and
// what none of them is longer than, so a ragged batch costs what it would if all were as long, and the list, which balances it, is
// taken later than it would pay.
//   clusters  4.4 and 1.45 for each round while every CTA has an SM for itself, 2.1 where two share one; with 16 columns 5 and 1.95.
//   list      5.6, the merging launch among them, and 2.25 for each round of the CTAs that are resident and one more; with 16 columns 9.
//   tcgen05   20, unpacking at 4.2 MB (of 144 and 512 bytes per token and head) and 1.75 for each tile of a CTA.
static PdForm pd_form(int32_t n_seq, int32_t n_tok, int32_t n_q, int32_t n_kv, int32_t max_q, int64_t max_tokens, int32_t flags) {
    PdForm f{};
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int64_t gqa = n_q / n_kv;
    f.nt = pd_tiles(n_q, n_kv, max_q);
    const int64_t cols = 8 * f.nt, rounds = (max_tokens + kPdWarps * kBatchTok - 1) / (kPdWarps * kBatchTok);
    f.blocks_of_seq = (int)((max_q * gqa + cols - 1) / cols);
    f.triples = (int64_t)n_seq * n_kv * f.blocks_of_seq;
    const int64_t resident = (f.nt == 1 ? 2 : 1) * (int64_t)sms;
    // all sequences' column blocks together, at most
    const int64_t blocks = n_tok <= n_seq ? n_seq : n_tok * gqa / cols + n_seq;
    const double most = (double)blocks * n_kv * (double)rounds, places = (double)blocks * n_kv * (double)(rounds + kTripleCost / kPdWarps);
    f.n_cta = (int)(places < 1 ? 1 : places < (double)resident ? places : (double)resident);
    const int asked = (flags & BGTQ_PAGED_FORM_MASK) >> BGTQ_PAGED_FORM_SHIFT;
    f.prefill = asked == 14;
    if (f.prefill || asked == 15) return f;
    int n = 8;
    while (n > 1 && (f.triples * n > sms || f.triples > (f.nt == 1 ? pd_clusters<1, 4>(n, dev) : pd_clusters<2, 2>(n, dev)))) n /= 2;
    if (asked) n = asked;
    f.alone = f.triples * n <= sms;
    const int64_t waves = (f.triples * n + resident - 1) / resident;
    const double cluster = (f.nt == 1 ? 4.4 : 5.0) + (f.nt > 1 ? 1.95 : f.alone ? 1.45 : 2.1) * (double)(waves * ((rounds + n - 1) / n));
    const double split = (f.nt == 1 ? 5.6 : 9.0) + 2.25 * (most + (double)resident - 1) / (double)resident;
    if (!asked && f.nt > 1) {
        const double pairs = (double)n_seq * n_kv, tiles = pairs * (double)((max_q * gqa + 255) / 256) * (double)((max_tokens + 127) / 128);
        f.prefill = 20.0 + pairs * (double)max_tokens * 656e-6 / 4.2 + 1.75 * (tiles + sms - 1) / sms < (cluster < split ? cluster : split);
        if (f.prefill) return f;
    }
    if (asked || cluster < split) f.n_rank = n;
    return f;
}

extern "C" __attribute__((visibility("default"))) int64_t bgtq_paged_workspace_bytes(int32_t n_seq, int32_t n_tok, int32_t n_q, int32_t n_kv,
                                                                                      int32_t max_q, int64_t max_tokens, int32_t flags) {
    if (n_seq < 0 || n_tok < 0 || n_kv < 1 || n_q < 1 || n_q % n_kv || max_q < 1 || max_tokens < 0) return BGTQ_E_BADARG;
    if (n_q / n_kv > 8) return BGTQ_E_UNSUPPORTED;
    const PdForm f = pd_form(n_seq, n_tok, n_q, n_kv, max_q, max_tokens, flags);
    if (f.prefill) return paged_prefill_workspace(n_seq, n_tok, n_q / n_kv, n_kv, max_tokens);
    return f.n_rank ? 0 : (int64_t)f.n_cta * 2 * 8 * f.nt * (kHD * 4 + 8);
}

extern "C" __attribute__((visibility("default"))) int bgtq_paged_attend(
    const void* q, int64_t q_st, int64_t q_sh, const uint8_t* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages,
    int32_t page_tokens, const int32_t* table, int64_t table_stride, int32_t table_cols, const int32_t* seq_lens, const int32_t* cu_q,
    int32_t n_seq, int32_t n_tok, int32_t n_q, int32_t n_kv, int32_t max_q, int64_t max_tokens, float scale, int32_t flags,
    void* workspace, int64_t workspace_bytes, void* out, int64_t o_st, int64_t o_sh, float* lse, int32_t* status, void* stream) {
    const int asked = (flags & BGTQ_PAGED_FORM_MASK) >> BGTQ_PAGED_FORM_SHIFT;
    pg_launched = 0;
    if (n_seq < 0 || n_tok < 0 || n_kv < 1 || n_q < 1 || table_cols < 0 || max_q < 1 || max_tokens < 0 ||
        (flags & ~(BGTQ_PAGED_BF16 | BGTQ_PAGED_CAUSAL | BGTQ_PAGED_FORM_MASK)) || (asked & (asked - 1) && asked < 14) || (asked == 14 && !cu_q) || asked == 13)
        return BGTQ_E_BADARG;
    if (!(scale == scale) || n_q % n_kv) return BGTQ_E_BADARG;
    if (n_q / n_kv > 8) return BGTQ_E_UNSUPPORTED;
    if (!cu_q && (n_tok != n_seq || max_q != 1)) return BGTQ_E_BADARG;
    if (n_seq == 0 || n_tok == 0) return BGTQ_OK;
    if (!pages || n_pages < 1 || page_tokens < kUnitTok || page_tokens % kUnitTok || !q || !out || !seq_lens || (!table && table_cols > 0))
        return BGTQ_E_BADARG;
    int64_t cap = (int64_t)table_cols * page_tokens;
    if (cap > max_tokens) cap = max_tokens;
    if (cap > INT32_MAX - 512 || max_tokens > INT64_MAX / 1024) return BGTQ_E_TOOBIG;
    if (!aligned(pages, 16) || page_stride % 16 || head_stride % 16 || !aligned(q, 16) || q_st % 8 || q_sh % 8 || !aligned(out, 8) || o_st % 4 ||
        o_sh % 4 || !aligned(workspace, 16))
        return BGTQ_E_ALIGN;
    // CTAs write rows while others read their queries
    const PagedRows q_rows{reinterpret_cast<uintptr_t>(q), n_tok, n_q, q_st, q_sh}, o_rows{reinterpret_cast<uintptr_t>(out), n_tok, n_q, o_st, o_sh};
    if (!paged_rows_apart(o_rows) || !paged_rows_apart(q_rows, o_rows)) return BGTQ_E_BADARG;
    PdForm f = pd_form(n_seq, n_tok, n_q, n_kv, max_q, max_tokens, flags);
    const cudaStream_t st = (cudaStream_t)stream;
    if (f.prefill) {
        if (!workspace || workspace_bytes < paged_prefill_workspace(n_seq, n_tok, n_q / n_kv, n_kv, max_tokens)) return BGTQ_E_BADARG;
        return paged_prefill({{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok}, table, table_stride, seq_lens, cu_q, n_seq, n_tok, n_q,
                              n_kv, n_q / n_kv, (flags & BGTQ_PAGED_CAUSAL) ? 1 : 0, (flags & BGTQ_PAGED_BF16) ? 1 : 0, max_tokens, (int32_t)cap,
                              reinterpret_cast<uint8_t*>(workspace), q, q_st, q_sh, scale * 1.44269504088896340736f, out, o_st, o_sh, lse, status},
                             st);
    }
    f.merge = cap > kPdWarps * kBatchTok && f.n_cta > 1;
    const int64_t cols = 8 * f.nt, blocks = n_tok <= n_seq ? n_seq : (int64_t)n_tok * (n_q / n_kv) / cols + n_seq;
    // the list's positions are 32 bits, and the grid's
    if ((double)blocks * n_kv * (double)(cap / kBatchTok + 2 * kPdWarps + kTripleCost) > 2.0e9 || (double)f.triples * 8 > 2.0e9) return BGTQ_E_TOOBIG;
    const int64_t need = f.n_rank ? 0 : (int64_t)f.n_cta * 2 * cols * (kHD * 4 + 8);
    if (need && (!workspace || workspace_bytes < need)) return BGTQ_E_BADARG;
    PdParams P{{pages, page_stride, head_stride, n_pages, page_tokens / kUnitTok}, q, q_st, q_sh, table, table_stride, seq_lens, cu_q,
               (int32_t)cap, n_seq, n_tok, n_q, n_kv, n_q / n_kv, !cu_q || (flags & BGTQ_PAGED_CAUSAL) ? 1 : 0, f.merge ? 1 : kPdWarps, f.n_rank ? f.blocks_of_seq : f.n_cta,
               scale * 1.44269504088896340736f, out, o_st, o_sh, lse, reinterpret_cast<float*>(workspace),
               reinterpret_cast<float2*>(reinterpret_cast<float*>(workspace) + (int64_t)f.n_cta * 2 * cols * kHD), status};
    const bool bf16 = flags & BGTQ_PAGED_BF16;
    if (f.nt == 1) return bf16 ? pd_launch<1, __nv_bfloat16>(P, f, st) : pd_launch<1, __half>(P, f, st);
    return bf16 ? pd_launch<2, __nv_bfloat16>(P, f, st) : pd_launch<2, __half>(P, f, st);
}
