// Attention of many query rows per (sequence, KV head) over the paged 4-bit cache, on tcgen05 with accumulators in tensor memory, in two
// launches:
//
//   unpack  every 128-token tile of a sequence's pages becomes two operand tiles in a workspace: khat [token][dim] and vhat [dim][token], fp16.
//           code * scale is exactly an fp16 number, so one tile each is all there is to know, and nothing is rounded.
//   attend  one CTA owns 256 query rows of one (sequence, KV head), two blocks of 128 (row = position * group + head), and walks the tiles:
//             * one thread streams them into a ring of five 32 KB slots (khat, vhat, khat, ...);
//             * one warp issues S_m = Q_m . khat^T (8 tcgen05.mma, M = N = 128) and O_m += P_m . vhat (8, P read from tensor memory) for the
//               two blocks in turn, so that the tensor cores work on one block while the other's softmax runs;
//             * 512 threads, two per query row, take S from tensor memory, apply the row's limit and put P (fp16) over S.  The value a row
//               scales by is its maximum less 7 (P up to 2^7: what is far below it keeps its bits), and moves, with O rescaled, only
//               when P would pass 2^15.
//           Queries are brought to [2^13, 2^14) by a power of two per row, which makes bf16 queries exact in fp16.
//
// What bounds attend: per tile 32 products of 64 cycles and 32768 exponentials at 16 a cycle, 2048 cycles each.
// Every wait is bounded: one that gives up is recorded in shared memory, where the others see it, and in the caller's status word; the CTA then
// drains its copies and products, releases its tensor memory and returns.
#include "bgtq_paged_common.cuh"
#include "bgtq_paged_prefill.h"
#include "bgtq_tcgen05.cuh"

namespace bgtq {
namespace {

constexpr int kRows = 128;                      // M of a product
constexpr int kBlocks = 2;                      // row blocks of a CTA
constexpr int kBlockRows = kRows * kBlocks;
constexpr int kPart = kPfTileTok * kHD * 2;     // bytes of an operand tile (32 KB)
static_assert(2 * kPart == kPfTileBytes, "khat and vhat");

struct Pf {
    PgPool pool;
    const int32_t* table;
    int64_t tb_st;
    const int32_t *lens, *cu_q;
    int32_t cap, n_tok, n_q, n_kv, gqa, causal;
    int32_t seq0, n_seq, h0, n_h, max_tiles;    // this launch's sequences and KV heads, tiles a sequence has room for
    uint8_t* tiles;                             // (n_seq, n_h, max_tiles) operand tile pairs
    int4* nan;                                  // (n_seq, n_h, max_tiles): per group, the tile's first token whose V is no number (INT_MAX: none)
    uint8_t* valid;                             // (n_seq, max_tiles): bit u, the tile's unit u was read (0 where its page number is none)
    const void* q;
    int64_t q_st, q_sh;
    float scale_log2;
    void* out;
    int64_t o_st, o_sh;
    float* lse;
    int32_t* status;
};

struct Seq {
    int len, q0, n;
};
__device__ __forceinline__ Seq pf_seq(const Pf& P, int i) {
    Seq s;
    s.len = max(0, min(P.lens[i], P.cap));
    s.q0 = min(max(P.cu_q[i], 0), P.n_tok);
    s.n = max(0, min(P.cu_q[i + 1], P.n_tok) - s.q0);
    return s;
}

// ------------------------------------------------------------------------------------------------------------------
// unpack: a warp per unit of 16 tokens.  Operand layout (no swizzle, K-major): element (row, k) at
//     (row / 8) * 2048 + (k / 8) * 128 + (row % 8) * 16 + (k % 8) * 2.
// Bound: memory, 144 bytes in and 512 out per token and head.  Every store is 16 bytes, a warp's are whole 128-byte lines.
// ------------------------------------------------------------------------------------------------------------------
template <int G>
__device__ __forceinline__ uint32_t value2(uint32_t w, uint32_t scale) {        // the pair of codes of group G, times the scales
    const uint32_t x = ((G >= 2 ? w >> 8 : w) & ((G & 1) ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
    uint32_t d;
    if (G & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(0x2c002c00u), "r"(0xd480d480u));
    else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0xe408e408u));
    return hmul2_u32(d, scale);
}
__device__ __forceinline__ uint32_t value2(int g, uint32_t w, uint32_t scale) {
    return g == 0 ? value2<0>(w, scale) : g == 1 ? value2<1>(w, scale) : g == 2 ? value2<2>(w, scale) : value2<3>(w, scale);
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) { return pack_half2(a, b); }

__global__ void __launch_bounds__(256) pg_unpack_kernel(const Pf P) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x, hi = blockIdx.y, si = blockIdx.z;
    grid_launch_dependents();
    grid_dependency_wait();
    const Seq s = pf_seq(P, P.seq0 + si);
    const int unit = tile * (kPfTileTok / kUnitTok) + warp, left = s.len - unit * kUnitTok;
    if (s.n == 0 || tile * kPfTileTok >= s.len) return;
    const uint8_t* u = nullptr;
    if (left > 0) {
        const int col = unit / P.pool.units, page = P.table[(int64_t)(P.seq0 + si) * P.tb_st + col];
        if (page >= 0 && page < P.pool.n_pages)
            u = P.pool.pages + (int64_t)page * P.pool.page_stride + (int64_t)(P.h0 + hi) * P.pool.head_stride + (unit - col * P.pool.units) * kUnitBytes;
        else if (P.status && lane == 0)
            *P.status = kStatusBadPage;
    }
    __shared__ uint8_t there[8];
    __shared__ int first_nan[4];
    if (lane == 0) there[warp] = u || left <= 0;
    if (threadIdx.x < 4) first_nan[threadIdx.x] = INT_MAX;
    __syncthreads();
    if (hi == 0 && threadIdx.x == 0) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m |= (uint32_t)there[i] << i;
        P.valid[(int64_t)si * P.max_tiles + tile] = (uint8_t)m;
    }
    uint8_t* const kt = P.tiles + (((int64_t)si * P.n_h + hi) * P.max_tiles + tile) * kPfTileBytes;
    uint8_t* const vt = kt + kPart;
    // K: lane = (token % 8, c): dims 32 n + 8 c .. + 7 for n = 0 .. 3
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = lane & 3, t = 8 * i + (lane >> 2);
        uint4 w = make_uint4(0, 0, 0, 0);
        uint2 sc = make_uint2(0, 0);
        if (u && t < left) {
            w = *reinterpret_cast<const uint4*>(u + 64 * t + 16 * c);
            sc = *reinterpret_cast<const uint2*>(u + kUnitKs + 8 * t);
        }
        const float f[4] = {pg_lo(sc.x), pg_hi(sc.x), pg_lo(sc.y), pg_hi(sc.y)};
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t h = half2_of(f[n], f[n]);
            *reinterpret_cast<uint4*>(kt + (2 * warp + i) * 2048 + (4 * n + c) * 128 + (lane >> 2) * 16) =
                make_uint4(value2(n, w.x, h), value2(n, w.y, h), value2(n, w.z, h), value2(n, w.w, h));
        }
    }
    // V: lane = W: dims 32 n + W, eight tokens at a time; the scales of pair p, group n lie in lane 4 p + n
    uint32_t mine = 0;
    {
        const int p = lane >> 2, n = lane & 3;
        const bool a = u && 2 * p < left, b = u && 2 * p + 1 < left;
        float s0 = a ? pg_lo(*reinterpret_cast<const uint16_t*>(u + kUnitVs + 16 * p + 2 * n)) : 0.f;
        float s1 = b ? pg_lo(*reinterpret_cast<const uint16_t*>(u + kUnitVs + 16 * p + 8 + 2 * n)) : 0.f;
        // A product with it would reach the rows that do not see it, too: zero here, and the rows that do are told
        if (s1 != s1) {
            atomicMin(&first_nan[n], unit * kUnitTok + 2 * p + 1);
            s1 = 0.f;
        }
        if (s0 != s0) {
            atomicMin(&first_nan[n], unit * kUnitTok + 2 * p);
            s0 = 0.f;
        }
        mine = half2_of(s0, s1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) w[p] = u && 8 * i + 2 * p < left ? *reinterpret_cast<const uint32_t*>(u + kUnitV + 128 * (4 * i + p) + 4 * lane) : 0u;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            uint32_t x[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) x[p] = value2(n, w[p], __shfl_sync(0xffffffffu, mine, 4 * (4 * i + p) + n));
            *reinterpret_cast<uint4*>(vt + (4 * n + (lane >> 3)) * 2048 + (2 * warp + i) * 128 + (lane & 7) * 16) = make_uint4(x[0], x[1], x[2], x[3]);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0)
        P.nan[((int64_t)si * P.n_h + hi) * P.max_tiles + tile] = make_int4(first_nan[0], first_nan[1], first_nan[2], first_nan[3]);
}

// ------------------------------------------------------------------------------------------------------------------
// attend
// ------------------------------------------------------------------------------------------------------------------
constexpr int kThreads = 576;           // warps 0-7: rows of block 0 (columns 0..63, then 64..127), 8-15: block 1, 16: products, 17: copies
constexpr int kWarpMma = 16, kWarpCopy = 17;
constexpr int kSlots = 5;
constexpr uint32_t kTmemCols = 512;     // S (and P) of block m: columns [128 m, 128 m + 128); O of block m: [256 + 128 m, 384 + 128 m)
constexpr uint32_t kColS = 0, kColO = 256;
constexpr float kLift = 7.0f, kReach = 15.0f;

struct PfSmem {
    __align__(128) uint8_t q[kBlocks][kPart];
    __align__(128) uint8_t ring[kSlots][kPart];
    __align__(8) uint64_t full[kSlots], empty[kSlots], s_ready[kBlocks], p_ready[kBlocks], o_ready[kBlocks];
    float xch[kBlocks][2][kRows];       // at first the rows' factors from sums to logits; then the two threads of a row: maxima, at the end denominators
    uint32_t tmem_base;
    int32_t seq, blk;
    int32_t nan[4];                     // per group, the first token whose V is no number
    volatile int32_t failed;
};
static_assert(sizeof(PfSmem) <= 227 * 1024, "fits an SM");

__device__ __forceinline__ float pf_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_scale8(uint32_t taddr, float f) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ bool bar_or(uint32_t id, bool flag) {        // over the 256 threads of one block's rows
    uint32_t out;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, %2, 256, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(out)
        : "r"((uint32_t)flag), "r"(id)
        : "memory");
    return out != 0;
}
__device__ __forceinline__ bool pf_wait(PfSmem& S, uint64_t* bar, uint32_t parity) {     // bounded; ends when another warp gave up, too
    for (uint32_t it = 0; it < (1u << 22); ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 63u && S.failed) return false;
    }
    S.failed = 1;
    return false;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) pg_prefill_kernel(const Pf P) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PfSmem& S = *reinterpret_cast<PfSmem*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], 1);
        }
        for (int m = 0; m < kBlocks; ++m) {
            mbar_init(&S.s_ready[m], 1);
            mbar_init(&S.p_ready[m], 2 * kRows);
            mbar_init(&S.o_ready[m], 1);
        }
        mbar_fence_init();
        S.failed = 0;
        S.nan[0] = S.nan[1] = S.nan[2] = S.nan[3] = INT_MAX;
    }
    if (warp == kWarpMma) tmem_alloc(&S.tmem_base, kTmemCols);
    grid_launch_dependents();
    grid_dependency_wait();
    // ---- which 256 rows: blocks are counted over the sequences; within one the latest, with the most tiles, come first ----
    if (warp == 0) {
        int before = 0, found = -1, blk = 0;
        for (int base = 0; base < P.n_seq && found < 0; base += 32) {
            const int i = base + lane;
            int w = 0;
            if (i < P.n_seq) w = (pf_seq(P, P.seq0 + i).n * P.gqa + kBlockRows - 1) / kBlockRows;
            int x = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, d);
                if (lane >= d) x += y;
            }
            const int first = before + x - w, at = (int)blockIdx.x - first;
            const uint32_t who = __ballot_sync(0xffffffffu, at >= 0 && at < w);
            if (who) {
                found = base + __ffs(who) - 1;
                blk = __shfl_sync(0xffffffffu, w - 1 - at, __ffs(who) - 1);
            }
            before += __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) {
            S.seq = found;
            S.blk = blk;
        }
    }
    __syncthreads();
    const int si = S.seq;
    if (si < 0) {
        if (warp == kWarpMma) tmem_dealloc(S.tmem_base, kTmemCols);
        return;
    }
    const Seq s = pf_seq(P, P.seq0 + si);
    const int hi = blockIdx.y, h = P.h0 + hi, n_rows = s.n * P.gqa, row0 = S.blk * kBlockRows;
    const int behind = s.len - s.n + 1, last_pos = (min(n_rows, row0 + kBlockRows) - 1) / P.gqa;
    const int t_max = P.causal ? min(s.len, max(0, behind + last_pos)) : s.len;
    const int n_t = (t_max + kPfTileTok - 1) / kPfTileTok;
    for (int t = tid; t < n_t; t += kThreads) {
        const int4 f = P.nan[((int64_t)si * P.n_h + hi) * P.max_tiles + t];
        if (min(min(f.x, f.y), min(f.z, f.w)) != INT_MAX) {
            atomicMin(&S.nan[0], f.x);
            atomicMin(&S.nan[1], f.y);
            atomicMin(&S.nan[2], f.z);
            atomicMin(&S.nan[3], f.w);
        }
    }
    // ---- the queries as A operands: a warp takes eight rows at a time, four lanes to a row, so that its stores are contiguous (with a row's
    // pieces side by side every one of them fell into the same banks: 10000 cycles for the CTA's rows) ----
    if (warp < 16) {
        const bool neg = P.scale_log2 < 0.f, zero = P.scale_log2 == 0.f;
        uint4 w[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int g = row0 + 16 * warp + 8 * i + (lane & 7), pos = g / P.gqa, hq = h * P.gqa + g - pos * P.gqa;
            const T* src = reinterpret_cast<const T*>(P.q) + (int64_t)(s.q0 + pos) * P.q_st + (int64_t)hq * P.q_sh + 8 * (lane >> 3);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[i][k] = make_uint4(0, 0, 0, 0);
                if (g < n_rows && !zero) w[i][k] = *reinterpret_cast<const uint4*>(src + 32 * k);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 16 * warp + 8 * i + (lane & 7);
            float x[4][8], top = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t ww[4] = {w[i][k].x, w[i][k].y, w[i][k].z, w[i][k].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = PgType<T>::up(ww[e]);
                    x[k][2 * e] = v.x;
                    x[k][2 * e + 1] = v.y;
                    top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            float up0, up1;
            const float fac = pg_row_scale(top, up0, up1);
            if (neg) up0 = -up0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = pack_half2(x[k][2 * e] * up0 * up1, x[k][2 * e + 1] * up0 * up1);
                *reinterpret_cast<uint4*>(S.q[row >> 7] + ((row & 127) >> 3) * 2048 + (4 * k + (lane >> 3)) * 128 + (row & 7) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            if (lane < 8) S.xch[row >> 7][0][row & 127] = fac;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // Q: generic-proxy stores -> tensor-core reads
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = S.tmem_base;
    bool ok = true;

    if (warp == kWarpCopy) {
        if (lane == 0) {
            asm volatile("fence.proxy.async.global;" ::: "memory");     // the tiles: another launch's stores -> bulk copies
            const uint8_t* src = P.tiles + ((int64_t)si * P.n_h + hi) * P.max_tiles * kPfTileBytes;
            const int n_parts = 2 * n_t;
            int n = 0;
            for (; n < n_parts; ++n) {
                const int slot = n % kSlots;
                if (n >= kSlots && !pf_wait(S, &S.empty[slot], (uint32_t)(n / kSlots - 1) & 1u)) { ok = false; break; }
                mbar_arrive_expect_tx(&S.full[slot], kPart);
                bulk_g2s(S.ring[slot], src + (size_t)n * kPart, kPart, &S.full[slot]);
            }
            if (!ok)        // the copies in flight land before the CTA leaves
                for (int i = max(0, n - kSlots); i < n; ++i) mbar_wait_bounded(&S.full[i % kSlots], (uint32_t)(i / kSlots) & 1u);
        }
    } else if (warp == kWarpMma) {
        if (n_t > 0) {
            const uint32_t lead = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t q_desc = op_desc(smem_u32(S.q[0])), ring_desc = op_desc(smem_u32(S.ring[0]));
            auto wait_part = [&](int n) { return (bool)__all_sync(0xffffffffu, pf_wait(S, &S.full[n % kSlots], (uint32_t)(n / kSlots) & 1u)); };
            auto part_desc = [&](int n) { return ring_desc + (uint32_t)(n % kSlots) * (kPart >> 4); };
            auto commit = [&](uint64_t* bar) {
                if (lead) umma_commit(bar);
                __syncwarp();
            };
            // P in tensor memory, k-step ks: the first four steps lie in columns 0..31 of S, the others in 64..95
            auto a_of = [](uint32_t base, int ks) { return base + 64u * (uint32_t)(ks >> 2) + 8u * (uint32_t)(ks & 3); };
            auto issue_s = [&](int i, int m) {
                const uint64_t qa = q_desc + (uint32_t)m * (kPart >> 4), kd = part_desc(2 * i);
                const uint32_t dst = tm + kColS + 128u * m;
#pragma unroll
                for (int ks = 0; ks < kHD / 16; ++ks) mma_ss(dst, qa + 16u * ks, kd + 16u * ks, ks > 0, lead);
                commit(&S.s_ready[m]);
                if (m == kBlocks - 1) commit(&S.empty[(2 * i) % kSlots]);
            };
            ok = wait_part(0);
            if (ok) {
                issue_s(0, 0);
                issue_s(0, 1);
            }
            for (int i = 0; i < n_t && ok; ++i) {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    if (m == 0 && !wait_part(2 * i + 1)) { ok = false; break; }
                    if (!__all_sync(0xffffffffu, pf_wait(S, &S.p_ready[m], (uint32_t)i & 1u))) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint64_t vd = part_desc(2 * i + 1);
                    const uint32_t a = tm + kColS + 128u * m, dst = tm + kColO + 128u * m;
#pragma unroll
                    for (int ks = 0; ks < kPfTileTok / 16; ++ks) mma_ts(dst, a_of(a, ks), vd + 16u * ks, (i > 0 || ks > 0) ? 1u : 0u, lead);
                    commit(&S.o_ready[m]);
                    if (m == kBlocks - 1) commit(&S.empty[(2 * i + 1) % kSlots]);
                    if (i + 1 < n_t) {      // (products of one thread execute in order: S replaces the P that was just read)
                        if (m == 0 && !wait_part(2 * i + 2)) { ok = false; break; }
                        issue_s(i + 1, m);
                    }
                }
            }
            if (!ok) {              // products in flight end before the tensor memory is released
                commit(&S.s_ready[0]);
                mbar_wait_bounded(&S.s_ready[0], 0u);
                mbar_wait_bounded(&S.s_ready[0], 1u);
            }
        }
    } else {
        // ---- softmax: two threads per query row ----
        const int mb = warp >> 3, hf = (warp >> 2) & 1, r128 = (warp & 3) * 32 + lane;
        const int g = row0 + kRows * mb + r128;
        const bool rok = g < n_rows;
        const int pos = g / P.gqa;
        const int lim = !rok ? 0 : (P.causal ? max(0, min(s.len, behind + pos)) : s.len);
        const float sc = S.xch[mb][0][r128] * (P.scale_log2 == 0.f ? 1.f : fabsf(P.scale_log2));
        const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);   // this warp's quarter of the lanes
        const uint32_t colS = tlane + kColS + 128u * mb, colO = tlane + kColO + 128u * mb + 64u * hf;
        const uint8_t* const valid = P.valid + (int64_t)si * P.max_tiles;
        uint32_t units = n_t > 0 ? valid[0] : 0;
        float m_used = -INFINITY, lsum = 0.f;    // the maximum this row scales by (log2 domain), this half's denominator
        const uint64_t sc2 = pack_f2(sc, sc);
        for (int i = 0; i < n_t; ++i) {
            if (!__all_sync(0xffffffffu, pf_wait(S, &S.s_ready[mb], (uint32_t)i & 1u))) ok = false;
            tc_fence_after_sync();
            const uint32_t sS = colS + 64u * hf;
            const int t0 = i * kPfTileTok + 64 * hf;
            const uint32_t there = units >> (4 * hf) & 15u;
            if (i + 1 < n_t) units = valid[i + 1];
            const bool cut = !__all_sync(0xffffffffu, t0 + 64 <= lim) || there != 15u;     // tiles that reach a row's limit, or lack a page
            float sv[32];
            auto load = [&](int c0) {
                tmem_ld32(sS + (uint32_t)c0, sv);
                tmem_ld_wait();
                if (cut) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) sv[c] = t0 + c0 + c < lim && (there >> ((c0 + c) >> 4) & 1u) ? sv[c] : -INFINITY;
                }
            };
            auto top = [&]() {
                float a = max3(sv[0], sv[1], sv[2]), c = max3(sv[3], sv[4], sv[5]);
#pragma unroll
                for (int e = 6; e < 30; e += 4) {
                    a = max3(a, sv[e], sv[e + 1]);
                    c = max3(c, sv[e + 2], sv[e + 3]);
                }
                return max3(max3(a, c, c), sv[30], sv[31]);
            };
            load(32);
            float m_half = top();
            load(0);
            m_half = fmaxf(m_half, top()) * sc;
            const bool move = bar_or(1 + mb, m_half > m_used + kReach || (m_used == -INFINITY && m_half > -INFINITY) || !ok);
            if (move) {
                S.xch[mb][hf][r128] = m_half;
                const bool all_ok = bar_and(3 + mb, 256, ok);
                if (!all_ok) { ok = false; break; }              // (the same verdict for the whole block)
                const float m_new = fmaxf(m_half, S.xch[mb][hf ^ 1][r128]) - kLift;
                float alpha = 1.f;
                if (m_used == -INFINITY) m_used = m_new;         // nothing accumulated for this row yet
                else if (m_new > m_used + (kReach - kLift)) {
                    alpha = pf_exp2(m_used - m_new);
                    m_used = m_new;
                }
                lsum *= alpha;
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    // O is at rest between the previous tile's product and this tile's
                    if (!__all_sync(0xffffffffu, pf_wait(S, &S.o_ready[mb], (uint32_t)(i - 1) & 1u))) ok = false;   // (ends at the next tile)
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int ch = 0; ch < 8; ++ch) tmem_scale8(colO + 8u * ch, alpha);
                }
            }
            const float z = m_used == -INFINITY ? 0.f : m_used;
            const uint64_t nz2 = pack_f2(-z, -z);
            uint64_t ps[2] = {0ull, 0ull};
            auto put = [&](uint32_t c0) {       // P of the columns in sv -> 16 columns of the half's own part of S
                uint32_t pk[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x0, x1;
                    unpack_f2(fma_f2(pack_f2(sv[2 * e], sv[2 * e + 1]), sc2, nz2), x0, x1);
                    const float p0 = pf_exp2(x0), p1 = pf_exp2(x1);
                    ps[e & 1] = add_f2(ps[e & 1], pack_f2(p0, p1));
                    pk[e] = pack_half2(p0, p1);
                }
                tmem_st16(sS + c0, pk);
            };
            put(0u);
            load(32);
            put(16u);
            float a0, a1;
            unpack_f2(add_f2(ps[0], ps[1]), a0, a1);
            lsum += a0 + a1;
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(&S.p_ready[mb]);
        }
        // ---- normalise, write ----
        if (n_t > 0 && ok) {
            ok = __all_sync(0xffffffffu, pf_wait(S, &S.o_ready[mb], (uint32_t)(n_t - 1) & 1u));
            tc_fence_after_sync();
        }
        bar_and(3 + mb, 256, true);                // (a row's factor is read before its place takes a denominator)
        S.xch[mb][hf][r128] = lsum;
        if (!bar_and(3 + mb, 256, ok)) ok = false;
        lsum += S.xch[mb][hf ^ 1][r128];
        const float inv = lsum > 0.f ? 1.0f / lsum : lsum == 0.f ? 0.f : lsum;
        const bool wide = ((reinterpret_cast<uintptr_t>(P.out) | (uint64_t)(2 * P.o_st) | (uint64_t)(2 * P.o_sh)) & 15u) == 0;
        if (ok) {
            // through the warp's own piece of the block's query tile, which no product reads any more: 32 rows of 128 bytes, 16-byte pieces
            // exchanged by row, so that the stores are whole lines
            uint8_t* const mine = S.q[mb] + (warp & 7) * 4096;
#pragma unroll 1
            for (int ch = 0; ch < 2; ++ch) {
                float o[32];
                if (n_t > 0) {
                    tmem_ld32(colO + 32u * ch, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0.f;
                }
                const float f = S.nan[2 * hf + ch] < lim ? __uint_as_float(0x7fffffffu) : inv;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<uint4*>(mine + lane * 128 + (((4 * ch + c) ^ (lane & 7)) << 4)) =
                        make_uint4(PgType<T>::down(o[8 * c] * f, o[8 * c + 1] * f), PgType<T>::down(o[8 * c + 2] * f, o[8 * c + 3] * f),
                                   PgType<T>::down(o[8 * c + 4] * f, o[8 * c + 5] * f), PgType<T>::down(o[8 * c + 6] * f, o[8 * c + 7] * f));
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r32 = 4 * k + (lane >> 3), gr = row0 + kRows * mb + (warp & 3) * 32 + r32, pr = gr / P.gqa;
                const uint4 v = *reinterpret_cast<const uint4*>(mine + r32 * 128 + (((lane & 7) ^ (r32 & 7)) << 4));
                if (gr < n_rows) {
                    uint2* const dst = reinterpret_cast<uint2*>(reinterpret_cast<T*>(P.out) + (int64_t)(s.q0 + pr) * P.o_st +
                                                                (int64_t)(h * P.gqa + gr - pr * P.gqa) * P.o_sh + 64 * hf + 8 * (lane & 7));
                    if (wide) {
                        *reinterpret_cast<uint4*>(dst) = v;
                    } else {
                        dst[0] = make_uint2(v.x, v.y);
                        dst[1] = make_uint2(v.z, v.w);
                    }
                }
            }
            const int hq = h * P.gqa + g - pos * P.gqa;
            if (rok && hf == 0 && P.lse)
                P.lse[(int64_t)(s.q0 + pos) * P.n_q + hq] = lsum == 0.f ? -INFINITY : (m_used + log2f(lsum)) * 0.693147180559945309f;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kWarpMma) tmem_dealloc(tmem, kTmemCols);
    if (tid == 0 && S.failed && P.status) *P.status = kStatusWaitTimeout;
}

}  // namespace

// Sequences and KV heads of one launch's workspace: all of them, or fewer sequences, then fewer heads, so that their tiles stay within 2 GiB.
static void pf_parts(int n_seq, int n_kv, int64_t max_tokens, int& seqs, int& heads, int64_t& tiles) {
    constexpr int64_t kMost = 2ll << 30;
    tiles = (max_tokens + kPfTileTok - 1) / kPfTileTok;
    if (tiles < 1) tiles = 1;
    const int64_t pairs = kMost / (tiles * kPfTileBytes);
    heads = (int)(pairs >= n_kv ? n_kv : pairs > 1 ? pairs : 1);
    seqs = (int)(pairs / n_kv >= n_seq ? n_seq : pairs / n_kv > 1 ? pairs / n_kv : 1);
    if (seqs > 65535) seqs = 65535;
}

int64_t paged_prefill_workspace(int n_seq, int n_kv, int64_t max_tokens) {
    int seqs, heads;
    int64_t tiles;
    pf_parts(n_seq, n_kv, max_tokens, seqs, heads, tiles);
    return seqs * tiles * (heads * (int64_t)(kPfTileBytes + 16) + 1);
}

int paged_prefill(const PagedPrefill& A, cudaStream_t stream) {
    int seqs, heads;
    int64_t tiles;
    pf_parts(A.n_seq, A.n_kv, A.max_tokens, seqs, heads, tiles);
    const int64_t blocks = (int64_t)A.n_tok * A.gqa / kBlockRows + A.n_seq;
    if (blocks > INT32_MAX || tiles > INT32_MAX) return BGTQ_E_TOOBIG;
    const auto kernel = A.bf16 ? pg_prefill_kernel<__nv_bfloat16> : pg_prefill_kernel<__half>;
    static std::atomic<uint64_t> allowed[2];
    if (!pg_allow_smem(kernel, (int)sizeof(PfSmem), allowed[A.bf16])) return BGTQ_E_LAUNCH;
    for (int s0 = 0; s0 < A.n_seq; s0 += seqs)
        for (int h0 = 0; h0 < A.n_kv; h0 += heads) {
            const int ns = A.n_seq - s0 < seqs ? A.n_seq - s0 : seqs, nh = A.n_kv - h0 < heads ? A.n_kv - h0 : heads;
            uint8_t* const nan = A.workspace + seqs * tiles * heads * (int64_t)kPfTileBytes;
            Pf P{A.pool, A.table, A.tb_st, A.lens, A.cu_q, (int32_t)A.max_tokens, A.n_tok, A.n_q, A.n_kv, A.gqa, A.causal, s0, ns, h0, nh, (int32_t)tiles,
                 A.workspace, reinterpret_cast<int4*>(nan), nan + seqs * tiles * heads * 16, A.q, A.q_st, A.q_sh, A.scale_log2, A.out, A.o_st, A.o_sh,
                 A.lse, A.status};
            if (launch_kernel(pg_unpack_kernel, dim3((unsigned)tiles, nh, ns), dim3(256), 0, stream, true, P) != cudaSuccess) return BGTQ_E_LAUNCH;
            if (launch_kernel(kernel, dim3((unsigned)blocks, nh), dim3(kThreads), sizeof(PfSmem), stream, true, P) != cudaSuccess) return BGTQ_E_LAUNCH;
        }
    return BGTQ_OK;
}

}  // namespace bgtq
