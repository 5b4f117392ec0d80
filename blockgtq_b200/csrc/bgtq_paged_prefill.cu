// Attention of many query rows per (sequence, KV head) over the paged 4-bit cache, on tcgen05 with accumulators in tensor memory, in three
// launches:
//
//   unpack  every 128-token tile of a sequence's pages becomes two operand tiles in a workspace: khat [token][dim] and vhat [dim][token], fp16.
//           code * scale is exactly an fp16 number, so one tile each is all there is to know, and nothing is rounded.
//           One CTA more cuts the work: a block is 256 query rows of one (sequence, KV head), as two of 128 (row = position * group + head), and has
//           as many tiles as its latest row sees; the tiles of all blocks are one list, cut evenly over the CTAs of the attention.
//   attend  one CTA per SM walks its share of the list, block by block:
//             * one thread streams them into a ring of four 32 KB slots (khat, vhat, khat, ...);
//             * one warp issues S_m = Q_m . khat^T (8 tcgen05.mma, M = N = 128) and O_m += P_m . vhat (8, P read from tensor memory) for the
//               two blocks in turn, so that the tensor cores work on one block while the other's softmax runs;
//             * 512 threads, two per query row, take S from tensor memory, apply the row's limit and put P (fp16) over S.  The value a row
//               scales by is its maximum less 7 (P up to 2^7: what is far below it keeps its bits), and moves, with O rescaled, only
//               when P would pass 2^15.  Weights below 2^-21 of the largest are subnormal in fp16, and cut at 2^-32 of it.
//           Queries are brought to [2^13, 2^14) by a power of two per row, which makes bf16 queries exact in fp16.
//   merge   rows of the blocks that the shares cut.
//
// What bounds attend: per tile 32 products of 64 cycles and 32768 exponentials at 16 a cycle, 2048 cycles each; a tile takes about 3200, the chain
// of a block's S, its softmax (1900 cycles) and its P . vhat beside the other block's.  8192 positions x 32 query and 8 KV heads, causal: 493 us
// in short runs, 1.12 PFLOP/s, and 568 in long ones, 0.97 PFLOP/s, where the power limit lowers the clock.  Chunks of 195 to 700 rows behind 700
// to 9100 tokens of 2 KV heads x 8: 115 us for the three launches, every CTA's share done between 77 and 95 us.
//
// Scores that are not plain (PgScores; PgMode: a kernel for each combination).  Masks: a block's tiles are those of its sequence's prefix and those from its
// first row's window on, and only the tiles that cut a row's sight are masked, by 32 bits per row and half.  Caps and biases are made of the products by
// the softmax's threads, and add to the chain what they take: 8192 positions as above 504 us plain, 609 with slopes, 677 to 692 with a cap that logits stay
// within 3/8 of, 875 to 996 within 7/5, 2118 beyond, with both 944, 1490 and 2245; with a window of 2048 295, 326, 363 to 373, 475 to 521 and 1024, 480, 740 and 1073.  The threads issue half of the cycles then, and no pipe is
// busy for more than 42 %: two row blocks of two warps per scheduler each are too few to hide the latencies, and tensor memory holds no third.
// Every wait is bounded: one that gives up is recorded in shared memory, where the others see it, and in the caller's status word; the CTA then
// drains its copies and products, releases its tensor memory and returns.
#include "bgtq_paged_common.cuh"
#include "bgtq_paged_prefill.h"
#include "bgtq_tcgen05.cuh"

#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

namespace bgtq {
namespace {

constexpr int kRows = 128;                      // M of a product
constexpr int kBlocks = 2;                      // row blocks of a CTA
constexpr int kBlockRows = kRows * kBlocks;
static_assert(kBlockRows == kPfBlockRows, "as the form of a call is chosen for");
constexpr int kBlockCost = 7, kLeastCost = 8;   // halves of a tile's cost: of a block beside its tiles, of a share
constexpr int kPart = kPfTileTok * kHD * 2;     // bytes of an operand tile (32 KB)
static_assert(2 * kPart == kPfTileBytes, "khat and vhat");

// 256 query rows of a sequence.
struct __align__(16) Block {
    int32_t si, row0, len, q0, n;               // sequence of the launch, first row; its tokens, first query row, queries
    int32_t tiles, sees, gap;                   // tiles that its rows see, at least one; 1 + those of the prefix, 0: they see none; tiles left out behind those
    template <bool kBack> __device__ __forceinline__ int tile(int k) const {     // kBack: the last one first
        if (kBack) k = tiles - 1 - k;
        return k + (gap && k >= sees - 1 ? gap : 0);
    }
    // The same among those of its sequence that the workspace holds; first_gap: what it lacks, no more than gap
    template <bool kBack> __device__ __forceinline__ int slot(int k, int first_gap) const {
        if (kBack) k = tiles - 1 - k;
        return k + (gap && k >= sees - 1 ? gap - first_gap : 0);
    }
};

struct Pf {
    PgPool pool;
    const int32_t* table;
    int64_t tb_st;
    const int32_t *lens, *cu_q;
    int32_t cap, n_tok, n_q, n_kv, gqa, causal;
    uint32_t gqa_inv;                           // 2^32 / gqa, rounded up; 0: gqa is 1
    int32_t seq0, n_seq, h0, n_h, max_tiles;    // this launch's sequences and KV heads, tiles a sequence has room for (with a window, those that its
                                                // prefix and its rows' windows reach, one behind the other)
    uint8_t* tiles;                             // (n_seq, n_h, max_tiles) operand tile pairs
    int4* nan;                                  // (n_seq, n_h, max_tiles): per group, the tile's first token whose V is no number (INT_MAX: none)
    Block* blk;                                 // the blocks, sequence by sequence
    int32_t* first;                             // per block: the tiles of the blocks before it; one more: of all of them
    int4* start;                                // per CTA, and for the end: block, tile, KV head of its share's begin, tiles before it; behind them: the number of blocks
    int32_t max_blocks, n_cta;
    float* part_o;                              // (2 n_cta, 256, 128): blocks' rows that a CTA holds a part of (its first, its last)
    float2* part_ml;                            // (2 n_cta, 256): reference, denominator
    uint8_t* valid;                             // (n_seq, max_tiles): bit u, the tile's unit u was read (0 where its page number is none)
    const void* q;
    int64_t q_st, q_sh;
    float scale_log2;
    void* out;
    int64_t o_st, o_sh;
    float* lse;
    int32_t* status;
    PgScores sc;                                // (kernels of kMod read it)
    uint64_t low[4], mid[9], steps[16];        // the cap's polynomials (of products, of u), each coefficient twice; -31, -30 .. 0
    float low_reach2;                           // largest product's square that the first is for
    uint32_t* nan_bits;                         // kMod: (n_seq, n_h, max_tiles) x 4 groups x 128 tokens: those whose V is no number
};

struct Seq {
    int len, q0, n, pre;
};
template <bool kMod>
__device__ __forceinline__ Seq pf_seq(const Pf& P, int i) {
    Seq s;
    s.pre = 0;
    s.len = max(0, min(P.lens[i], P.cap));
    s.q0 = min(max(P.cu_q[i], 0), P.n_tok);
    s.n = max(0, min(P.cu_q[i + 1], P.n_tok) - s.q0);
    if (kMod) s.pre = pg_prefix(P.sc, i, s.len);
    return s;
}
// First token of the window of a sequence's row
__device__ __forceinline__ int pf_window(const Pf& P, const Seq& s, int pos) { return P.sc.window ? max(0, max(0, s.len - s.n + 1 + pos) - P.sc.window) : 0; }

// ------------------------------------------------------------------------------------------------------------------
// unpack: a warp per unit of 16 tokens.  Operand layout (no swizzle, K-major): element (row, k) at
//     (row / 8) * 2048 + (k / 8) * 128 + (row % 8) * 16 + (k % 8) * 2.
// Bound: memory, 144 bytes in and 512 out per token and head, at 4.2 TB/s (8192 tokens x 8 heads: 43 MB in 10 us).  Every store is 16 bytes, a
// warp's are whole 128-byte lines.
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

__device__ __forceinline__ int pf_pos(const Pf& P, int row) {      // row / gqa, rows < 2^29
    return P.gqa_inv ? (int)__umulhi((uint32_t)row, P.gqa_inv) : row;
}
// Tiles between a sequence's prefix and its first row's window: the workspace has no place for them.
__device__ __forceinline__ int pf_gap(const Pf& P, const Seq& s) {
    return max(0, pf_window(P, s, 0) / kPfTileTok - (s.pre + kPfTileTok - 1) / kPfTileTok);
}
template <bool kMod>
__device__ __forceinline__ Block pf_block(const Pf& P, int si, const Seq& s, int j) {
    const int last_pos = (min(s.n * P.gqa, (j + 1) * kBlockRows) - 1) / P.gqa;
    const int t_max = P.causal ? max(s.pre, s.len - s.n + 1 + last_pos) : s.len, tiles = (t_max + kPfTileTok - 1) / kPfTileTok;
    if (!kMod) return Block{si, j * kBlockRows, s.len, s.q0, s.n, max(1, tiles), tiles > 0, 0};
    const int head = (s.pre + kPfTileTok - 1) / kPfTileTok, gap = max(0, pf_window(P, s, j * kBlockRows / P.gqa) / kPfTileTok - head);
    return Block{si, j * kBlockRows, s.len, s.q0, s.n, max(1, tiles - gap), tiles > 0 ? 1 + head : 0, gap};
}
// The list of blocks and the CTAs' shares, by one CTA of 256 threads.
template <bool kMod>
__device__ void pf_plan(const Pf& P) {
    __shared__ int sums[8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto scan = [&](int w, int& total) {         // exclusive, over the CTA
        int x = w;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        int before = 0;
        total = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            before += i < warp ? sums[i] : 0;
            total += sums[i];
        }
        __syncthreads();
        return before + x - w;
    };
    int n_blocks = 0;
    for (int base = 0; base < P.n_seq; base += 256) {
        const int i = base + tid;
        Seq s{0, 0, 0, 0};
        if (i < P.n_seq) s = pf_seq<kMod>(P, P.seq0 + i);
        const int w = (s.n * P.gqa + kBlockRows - 1) / kBlockRows;
        int all;
        const int at = n_blocks + scan(w, all);
        for (int k = 0; k < 32; ++k) {           // a warp writes the blocks of its sequences one after another
            const int n = __shfl_sync(0xffffffffu, w, k), to = __shfl_sync(0xffffffffu, at, k);
            const Seq t{__shfl_sync(0xffffffffu, s.len, k), __shfl_sync(0xffffffffu, s.q0, k), __shfl_sync(0xffffffffu, s.n, k),
                        kMod ? __shfl_sync(0xffffffffu, s.pre, k) : 0};
            for (int j = lane; j < n && to + j < P.max_blocks; j += 32) P.blk[to + j] = pf_block<kMod>(P, base + 32 * warp + k, t, j);
        }
        n_blocks = min(P.max_blocks, n_blocks + all);
    }
    __syncthreads();
    int tiles = 0;
    for (int base = 0; base < n_blocks; base += 256) {
        const int i = base + tid, w = i < n_blocks ? P.blk[i].tiles : 0;
        int all;
        const int at = tiles + scan(w, all);
        if (i < n_blocks) P.first[i] = at;
        tiles += all;
    }
    if (tid == 0) P.first[n_blocks] = tiles;
    __syncthreads();
    // Shares of equal cost: a tile 2, a block kBlockCost more (its queries, its results, the pipeline's start)
    const int64_t head = 2ll * tiles + (int64_t)kBlockCost * n_blocks, total = head * P.n_h, share = max((int64_t)kLeastCost, (total + P.n_cta - 1) / P.n_cta);
    for (int c = tid; c <= P.n_cta; c += 256) {
        const int64_t p = min((int64_t)c * share, total);
        const int h = (int)(p / max(head, (int64_t)1)), r = (int)(p - (int64_t)h * head);
        int lo = 0, hi = max(n_blocks - 1, 0);           // the last block that starts at or before r
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (2ll * P.first[mid] + (int64_t)kBlockCost * mid <= r) lo = mid;
            else hi = mid - 1;
        }
        const int t = p < total ? max(0, (int)(r - (2ll * P.first[lo] + (int64_t)kBlockCost * lo)) - kBlockCost) >> 1 : 0;
        P.start[c] = make_int4(lo, t, h, p < total ? h * tiles + P.first[lo] + t : tiles * P.n_h);
    }
    if (tid == 0) P.start[P.n_cta + 1] = make_int4(n_blocks, 0, 0, 0);
}

template <bool kMod>
__global__ void __launch_bounds__(256) pg_unpack_kernel(const Pf P) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slot = blockIdx.x, hi = blockIdx.y, si = blockIdx.z;
    grid_launch_dependents();
    grid_dependency_wait();
    if (slot == P.max_tiles) {
        if (hi == 0 && si == 0) pf_plan<kMod>(P);
        return;
    }
    const Seq s = pf_seq<kMod>(P, P.seq0 + si);
    const int tile = kMod && slot * kPfTileTok >= s.pre ? slot + pf_gap(P, s) : slot;
    const int unit = tile * (kPfTileTok / kUnitTok) + warp, left = s.len - unit * kUnitTok;
    if (s.n == 0 || tile * kPfTileTok >= s.len) return;
    const int low = kMod ? pf_window(P, s, 0) : 0;
    const bool hidden = kMod && unit * kUnitTok >= s.pre && (unit + 1) * kUnitTok <= low;     // (no row sees this unit)
    const uint8_t* u = nullptr;
    if (left > 0 && !hidden) {
        const int col = unit / P.pool.units, page = P.table[(int64_t)(P.seq0 + si) * P.tb_st + col];
        if (page >= 0 && page < P.pool.n_pages)
            u = P.pool.pages + (int64_t)page * P.pool.page_stride + (int64_t)(P.h0 + hi) * P.pool.head_stride + (unit - col * P.pool.units) * kUnitBytes;
        else if (P.status && lane == 0)
            *P.status = kStatusBadPage;
    }
    __shared__ uint8_t there[8];
    __shared__ int first_nan[4];
    __shared__ uint32_t all_nan[16];
    if (lane == 0) there[warp] = u || left <= 0 || hidden;
    if (threadIdx.x < 4) first_nan[threadIdx.x] = INT_MAX;
    if (kMod && threadIdx.x < 16) all_nan[threadIdx.x] = 0;
    __syncthreads();
    if (hi == 0 && threadIdx.x == 0) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m |= (uint32_t)there[i] << i;
        P.valid[(int64_t)si * P.max_tiles + slot] = (uint8_t)m;
    }
    uint8_t* const kt = P.tiles + (((int64_t)si * P.n_h + hi) * P.max_tiles + slot) * kPfTileBytes;
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
        if (kMod && (s0 != s0 || s1 != s1)) atomicOr(&all_nan[4 * n + (warp >> 1)], ((s0 != s0 ? 1u : 0u) | (s1 != s1 ? 2u : 0u)) << (16 * (warp & 1) + 2 * p));
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
        P.nan[((int64_t)si * P.n_h + hi) * P.max_tiles + slot] = make_int4(first_nan[0], first_nan[1], first_nan[2], first_nan[3]);
    if (kMod && threadIdx.x < 16) P.nan_bits[16 * (((int64_t)si * P.n_h + hi) * P.max_tiles + slot) + threadIdx.x] = all_nan[threadIdx.x];
}

// ------------------------------------------------------------------------------------------------------------------
// attend
// ------------------------------------------------------------------------------------------------------------------
constexpr int kThreads = 576;           // warps 0-7: rows of block 0 (columns 0..63, then 64..127), 8-15: block 1, 16: products, 17: copies
constexpr int kWarpMma = 16, kWarpCopy = 17;
constexpr int kSlots = 4;
constexpr uint32_t kTmemCols = 512;     // S (and P) of block m: columns [128 m, 128 m + 128); O of block m: [256 + 128 m, 384 + 128 m)
constexpr uint32_t kColS = 0, kColO = 256;
constexpr float kLift = 7.0f, kReach = 15.0f;
constexpr float kHuge = 1048576.0f;     // 2^20: a fused product's rounding is 2^-4 of a power of two here
// Of 16 pairs of exponentials, those that go to the FMA pipe: 8192 positions x 32 heads 506 us with two of them, 509 with none, 510 with three,
// 517 with four.
constexpr uint32_t kPolyPairs = 0x8080;

// A CTA's share, block by block.  Every role walks it for itself.
struct Walk {
    Block b;
    int g, t0, tiles, h, left, n_blocks;         // block, first tile and tiles of it (zero: its rows see nothing), KV head of the launch; tiles from here on
    bool first;

    Walk() = default;
    __device__ __forceinline__ explicit Walk(const Pf& P) {
        const int4 v = P.start[blockIdx.x], e = P.start[blockIdx.x + 1];
        n_blocks = P.start[P.n_cta + 1].x;
        g = v.x;
        t0 = v.y;
        h = v.z;
        left = e.w - v.w;
        first = true;
        if (left > 0) b = P.blk[g];
        tiles = left > 0 && b.sees ? run() : 0;
    }
    __device__ __forceinline__ int run() const { return min(b.tiles - t0, left); }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && left >= b.tiles; }
    __device__ __forceinline__ bool more() const { return left > run(); }
    __device__ __forceinline__ int next_g() const { return g + 1 == n_blocks ? 0 : g + 1; }
    __device__ __forceinline__ int next_h() const { return h + (g + 1 == n_blocks); }
    __device__ __forceinline__ int next_tiles(const Block& n) const { return n.sees ? min(n.tiles, left - run()) : 0; }
    __device__ __forceinline__ void step(const Block& n) {     // n: the record of next_g()
        left -= run();
        first = false;
        h = next_h();
        g = next_g();
        t0 = 0;
        b = n;
        tiles = n.sees ? run() : 0;
    }
    __device__ __forceinline__ void step_from(const Walk& w) { // the same from the block before, with its own record in place
        left = w.left - w.run();
        first = false;
        h = w.next_h();
        g = w.next_g();
        t0 = 0;
        n_blocks = w.n_blocks;
        tiles = b.sees ? run() : 0;
    }
};

// Logits under a cap, pairs at a time on the FMA pipe, u = x / cap.  Most tiles' are small beside it: an odd polynomial of degree 7 up to 3/8, straight from the
// products where all rows' have one factor (no row of bf16 queries was brought to another magnitude), or of degree 17 up to 7/5, both fitted to the relative
// error (7e-8, 4.8e-8); beyond, one by one.  All of a warp's 32 tokens go one way.  (Two more values of the special function pipe for each logit would be
// twice the time of all else: it makes 16 a cycle.)
constexpr int kLowTerms = 4, kMidTerms = 9;
constexpr double kLowReach = 0.375;
constexpr float kMidReach = 1.4f;
constexpr double kCapLow[kLowTerms] = {1.0, -0.3333233349357446, 0.13289726163824672, -0.04848729069776324};
constexpr double kCapMid[kMidTerms] = {1.0, -0.33333077724742183, 0.13328956227827346, -0.053706810286391585, 0.021092473450978352, -0.007527298246243253,
                                       0.0021462715909971895, -0.0004054931883325217, 3.6238863462110705e-05};
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <typename F>
__device__ __forceinline__ void tmem_map8(uint32_t taddr, F f) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(f(__uint_as_float(r[i])));
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// A pair of products' logits by the short polynomial, over the products; v: their squares
__device__ __forceinline__ uint64_t pf_low(const Pf& P, uint64_t v) {
    uint64_t p = fma_f2(v, P.low[kLowTerms - 1], P.low[kLowTerms - 2]);
#pragma unroll
    for (int i = kLowTerms - 3; i >= 0; --i) p = fma_f2(v, p, P.low[i]);
    return p;
}
// The same by the long one; v: the squares of u
__device__ __forceinline__ uint64_t pf_mid(const Pf& P, uint64_t v) {
    uint64_t p = fma_f2(v, P.mid[kMidTerms - 1], P.mid[kMidTerms - 2]);
#pragma unroll
    for (int i = kMidTerms - 3; i >= 0; --i) p = fma_f2(v, p, P.mid[i]);
    return p;
}
__device__ __forceinline__ float abs_top(const float (&x)[32]) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
        a = max3(a, fabsf(x[c]), fabsf(x[c + 1]));
        b = max3(b, fabsf(x[c + 2]), fabsf(x[c + 3]));
    }
    return fmaxf(a, b);
}
// 32 products x[], in tensor memory at `from`, to logits: times factor (even: the one that P.low is made for), capped (alike: by pg_cap_any, as the row's
// reference was), and less slope times the distances, of which the first is `ahead` of the row's own place (apart: each by itself, as
// some lie behind it).
template <bool kCap, bool kBias>
__device__ __forceinline__ void pf_shape(float (&x)[32], const Pf& P, float factor, bool even, bool alike, float slope, float ahead, bool apart, uint32_t from) {
    auto load = [&]() {
        tmem_ld32(from, x);
        tmem_ld_wait();
    };
    const float t31 = slope * (ahead + 31.f);
    const uint64_t t2 = pack_f2(t31, t31), s2 = pack_f2(slope, slope);
    // (slopes times whole numbers below 32, on top of the nearest token's, the last: its rounding is no more than the others' own)
    auto bias = [&](int c) { return fma_f2(s2, P.steps[c >> 1], t2); };
    if (kCap) {
        bool done = false;
        if (even && !alike) {
            float most[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const uint64_t r = pack_f2(x[c], x[c + 1]), v = mul_f2(r, r), p = pf_low(P, v);
                float v0, v1;
                unpack_f2(v, v0, v1);
                most[c >> 1 & 1] = max3(most[c >> 1 & 1], v0, v1);
                unpack_f2(kBias && !apart ? fma_f2(r, p, bias(c)) : mul_f2(r, p), x[c], x[c + 1]);
            }
            done = __all_sync(0xffffffffu, fmaxf(most[0], most[1]) <= P.low_reach2);
            if (done && (!kBias || !apart)) return;
            if (!done) load();
        }
        if (!done) {
            const float g = pg_unit(factor, P.sc);
            const uint64_t g2 = pack_f2(g, g);
            float most[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const uint64_t u = mul_f2(pack_f2(x[c], x[c + 1]), g2), v = mul_f2(u, u);
                float v0, v1;
                unpack_f2(v, v0, v1);
                most[c >> 1 & 1] = max3(most[c >> 1 & 1], v0, v1);
                unpack_f2(mul_f2(u, pf_mid(P, v)), x[c], x[c + 1]);
            }
            if (alike || !__all_sync(0xffffffffu, fmaxf(most[0], most[1]) <= kMidReach * kMidReach)) {
                // (in place, a few at a time: what hardly ever runs is kept short)
#pragma unroll 1
                for (int c = 0; c < 32; c += 8) tmem_map8(from + (uint32_t)c, [&](float r) { return pg_cap_any(r * g, P.sc); });
                tmem_st_wait();
                load();
            }
        }
    }
    if (kBias) {
        const float f = kCap ? 1.f : factor;
        const uint64_t f2 = pack_f2(f, f);
        if (apart) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = fmaf(-slope, fabsf(ahead + (float)c), x[c] * f);
        } else {
#pragma unroll
            for (int c = 0; c < 32; c += 2) unpack_f2(fma_f2(pack_f2(x[c], x[c + 1]), f2, bias(c)), x[c], x[c + 1]);
        }
    }
}

struct PfSmem {
    __align__(128) uint8_t q[kBlocks][kPart];
    __align__(128) uint8_t ring[kSlots][kPart];
    __align__(16) uint8_t stage[16][2048];      // per softmax warp: 64 bytes of each of its rows on their way out
    __align__(16) Walk walk[kBlocks][2];        // the softmax's: the block that is worked on and the one behind it, in turn (not in registers,
                                                // where the tiles' loop needs them)
    __align__(8) uint64_t full[kSlots], empty[kSlots], q_ready[kBlocks], s_ready[kBlocks], p_ready[kBlocks][2], o_ready[kBlocks];
    float xch[kBlocks][2][kRows];       // the two threads of a row: maxima, at the end denominators
    int16_t ex[kBlocks][kRows];         // the rows' queries are times 2^ex
    uint32_t tmem_base;
    int32_t nan[kBlocks][4];            // per group, the first token of the segment whose V is no number
    volatile int32_t failed;
};
static_assert(sizeof(PfSmem) <= 227 * 1024, "fits an SM");

__device__ __forceinline__ float pf_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of a pair on the FMA pipe, x >= -125: x = n + f, |f| <= 1/2, the powers of f by a polynomial fitted to the relative error (3e-6, exact at
// f = 0), n added to the exponent.
__device__ __forceinline__ void pf_exp2_poly(uint64_t x, float& p0, float& p1) {
    const uint64_t magic = pack_f2(12582912.f, 12582912.f), minus = pack_f2(-12582912.f, -12582912.f), neg = pack_f2(-1.f, -1.f);
    const uint64_t t = add_f2(x, magic), f = fma_f2(add_f2(t, minus), neg, x);
    uint64_t p = fma_f2(f, pack_f2(0.009582852013409138f, 0.009582852013409138f), pack_f2(0.055906426161527634f, 0.055906426161527634f));
    p = fma_f2(p, f, pack_f2(0.24024099111557007f, 0.24024099111557007f));
    p = fma_f2(p, f, pack_f2(0.6931241750717163f, 0.6931241750717163f));
    p = fma_f2(p, f, pack_f2(1.f, 1.f));
    p0 = __uint_as_float((uint32_t)p + ((uint32_t)t << 23));
    p1 = __uint_as_float((uint32_t)(p >> 32) + ((uint32_t)(t >> 32) << 23));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {             // NaN when either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
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

__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

template <typename T, PgMode kMode>
__global__ void __launch_bounds__(kThreads, 1) pg_prefill_kernel(const Pf P) {
    constexpr bool kMod = kMode != kPlain;
    // Biases fall with the distance: from a row's own place on backwards, its reference hardly moves
    constexpr bool kBack = kMode >= kBiased;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PfSmem& S = *reinterpret_cast<PfSmem*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], 1);
        }
        for (int m = 0; m < kBlocks; ++m) {
            mbar_init(&S.q_ready[m], 8);
            mbar_init(&S.s_ready[m], 1);
            mbar_init(&S.p_ready[m][0], 8);
            mbar_init(&S.p_ready[m][1], 8);
            mbar_init(&S.o_ready[m], 1);
        }
        mbar_fence_init();
        S.failed = 0;
        for (int i = 0; i < 4; ++i) S.nan[0][i] = S.nan[1][i] = INT_MAX;
    }
    if (warp == kWarpMma) tmem_alloc(&S.tmem_base, kTmemCols);
    grid_launch_dependents();
    grid_dependency_wait();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = S.tmem_base;
    bool ok = true;

    if (warp == kWarpCopy) {
        if (lane == 0) {
            asm volatile("fence.proxy.async.global;" ::: "memory");     // the tiles: another launch's stores -> bulk copies
            int n = 0;                                                  // parts so far
            for (Walk w(P); w.left > 0 && ok;) {
                const int first_gap = kMod ? pf_gap(P, pf_seq<true>(P, P.seq0 + w.b.si)) : 0;
                const uint8_t* src = P.tiles + (((int64_t)w.b.si * P.n_h + w.h) * P.max_tiles + (kMod ? 0 : w.t0)) * kPfTileBytes;
                for (int k = 0; k < 2 * w.tiles; ++k, ++n) {
                    const int slot = n % kSlots;
                    if (n >= kSlots && !pf_wait(S, &S.empty[slot], (uint32_t)(n / kSlots - 1) & 1u)) { ok = false; break; }
                    mbar_arrive_expect_tx(&S.full[slot], kPart);
                    const int part = kMod ? 2 * w.b.slot<kBack>(w.t0 + (k >> 1), first_gap) + (k & 1) : k;
                    bulk_g2s(S.ring[slot], src + (size_t)part * kPart, kPart, &S.full[slot]);
                }
                if (!w.more()) break;
                w.step(P.blk[w.next_g()]);
            }
            if (!ok)        // the copies in flight land before the CTA leaves
                for (int i = max(0, n - kSlots); i < n; ++i) mbar_wait_bounded(&S.full[i % kSlots], (uint32_t)(i / kSlots) & 1u);
        }
    } else if (warp == kWarpMma) {
        const uint32_t lead = elect_one();
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_desc = op_desc(smem_u32(S.q[0])), ring_desc = op_desc(smem_u32(S.ring[0]));
        auto wait = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, pf_wait(S, bar, parity & 1u)); };
        auto wait_part = [&](int n) { return wait(&S.full[n % kSlots], (uint32_t)(n / kSlots)); };
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
        int i = 0, seg = 0;                                             // tiles, and segments with tiles, so far
        Walk w(P);
        bool more = w.left > 0;
        while (more && ok) {
            const int end = i + w.tiles, begin = i;
            more = w.more();
            if (more) w.step(P.blk[w.next_g()]);
            if (end == begin) continue;
            ok = wait_part(2 * i);
#pragma unroll
            for (int m = 0; m < kBlocks; ++m) {
                if (ok) ok = wait(&S.q_ready[m], (uint32_t)seg);
                if (ok) {
                    tc_fence_after_sync();
                    issue_s(i, m);
                }
            }
            ++seg;
            for (; i < end && ok; ++i) {
#pragma unroll
                for (int m = 0; m < kBlocks; ++m) {
                    if (m == 0 && !wait_part(2 * i + 1)) { ok = false; break; }
                    const uint64_t vd = part_desc(2 * i + 1);
                    const uint32_t a = tm + kColS + 128u * m, dst = tm + kColO + 128u * m;
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        if (ok) ok = wait(&S.p_ready[m][part], (uint32_t)i);
                        if (!ok) break;
                        tc_fence_after_sync();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int ks = 4 * (k >> 1) + 2 * part + (k & 1);
                            mma_ts(dst, a_of(a, ks), vd + 16u * ks, (i > begin || part > 0 || k > 0) ? 1u : 0u, lead);
                        }
                    }
                    if (!ok) break;
                    commit(&S.o_ready[m]);
                    if (m == kBlocks - 1) commit(&S.empty[(2 * i + 1) % kSlots]);
                    if (i + 1 < end) {      // (products of one thread execute in order: S replaces the P that was just read)
                        if (m == 0 && !wait_part(2 * i + 2)) { ok = false; break; }
                        issue_s(i + 1, m);
                    }
                }
            }
        }
        if (!ok) {                  // products in flight end before the tensor memory is released
            commit(&S.s_ready[0]);
            mbar_wait_bounded(&S.s_ready[0], 0u);
            mbar_wait_bounded(&S.s_ready[0], 1u);
        }
    } else {
        // ---- softmax: two threads per query row ----
        const int mb = warp >> 3, hf = (warp >> 2) & 1, r128 = (warp & 3) * 32 + lane, w8 = warp & 7;
        const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);   // this warp's quarter of the lanes
        const uint32_t colS = tlane + kColS + 128u * mb, colO = tlane + kColO + 128u * mb + 64u * hf, sS = colS + 64u * hf;
        int done = 0;                                     // tiles so far
        // A block's queries go straight to their places in the operand; a warp takes sixteen rows, eight at a time and four lanes to a row, so that
        // its pieces are contiguous there.  They are requested while the last tile before them is worked on, and bf16 ones then made fp16, so that the
        // products of the new block run while the old one's results are written.  (Loops that are not unrolled: what runs once per
        // block is not in the instruction cache, and its size is its time.)
        auto q_place = [&](int i, int k) { return S.q[mb] + (2 * w8 + i) * 2048 + (4 * k + (lane >> 3)) * 128 + (lane & 7) * 16; };
        auto fetch = [&](const Block& b, int h) {
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                const int g = b.row0 + kRows * mb + 16 * w8 + 8 * i + (lane & 7), pos = pf_pos(P, g), hq = (P.h0 + h) * P.gqa + g - pos * P.gqa;
                const bool there = pos < b.n && P.scale_log2 != 0.f;
                const T* src = reinterpret_cast<const T*>(P.q) + (there ? (int64_t)(b.q0 + pos) * P.q_st + (int64_t)hq * P.q_sh + 8 * (lane >> 3) : 0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(q_place(i, k))), "l"(src + 32 * k), "r"(there ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // bf16 queries become fp16 in place; a row whose largest magnitude is in [2^-2, 2^15) as it is (what fp16 then cuts off is 2^-23 of it)
        auto ready = [&]() {
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (!PgType<T>::kHalf || P.scale_log2 < 0.f) {
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {
                    uint4 v[4];
                    uint32_t top = 0;                  // largest magnitudes as whole numbers, two at a time
                    bool plain = P.scale_log2 >= 0.f;
                    float up0 = 1.f, up1 = 1.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const uint4*>(q_place(i, k));
                    if (!PgType<T>::kHalf) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            top = __vmaxu2(__vmaxu2(top, __vmaxu2(v[k].x & 0x7fff7fffu, v[k].y & 0x7fff7fffu)), __vmaxu2(v[k].z & 0x7fff7fffu, v[k].w & 0x7fff7fffu));
                        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const uint32_t big = max(top & 0xffffu, top >> 16);
                        const float f = __uint_as_float(big << 16);
                        const int ex = f >= 0.25f && f < 32768.f ? 0 : pg_row_exponent(f);
                        pg_pow2(ex, up0, up1);
                        plain = plain && ex == 0;
                        if (lane < 8) S.ex[mb][16 * w8 + 8 * i + lane] = (int16_t)ex;
                    }
                    if (P.scale_log2 < 0.f) up0 = -up0;
                    const bool scaled = !__all_sync(0xffffffffu, plain);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t ww[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                        uint32_t o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float2 x = PgType<T>::up(ww[e]);
                            if (scaled) x = make_float2(x.x * up0 * up1, x.y * up0 * up1);
                            o[e] = pack_half2(x.x, x.y);
                        }
                        *reinterpret_cast<uint4*>(q_place(i, k)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // Q: copies and stores -> tensor-core reads
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.q_ready[mb]);
        };
        if ((tid & 255) == 0) S.walk[mb][0] = Walk(P);
        if (PgType<T>::kHalf && (tid & 255) < kRows) S.ex[mb][tid & 127] = 0;
        bar_and(3 + mb, 256, true);
        bool more = S.walk[mb][0].left > 0;
        if (more && S.walk[mb][0].tiles > 0) {
            fetch(S.walk[mb][0].b, S.walk[mb][0].h);
            ready();
        }
        for (int turn = 0; more; turn ^= 1) {
            const Walk& w = S.walk[mb][turn];
            Walk& next = S.walk[mb][turn ^ 1];
            const int tiles = w.tiles, tile0 = w.t0;
            more = w.more();
            if (more && w8 == 0 && lane < 2)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&next.b) + 16 * lane),
                             "l"(reinterpret_cast<const uint8_t*>(P.blk + w.next_g()) + 16 * lane) : "memory");
            const int first_gap = kMod ? pf_gap(P, pf_seq<true>(P, P.seq0 + w.b.si)) : 0;
            for (int t = tid & 255; t < tiles; t += 256) {
                const int4 f = P.nan[((int64_t)w.b.si * P.n_h + w.h) * P.max_tiles + (kMod ? w.b.slot<kBack>(tile0 + t, first_gap) : tile0 + t)];
                if (min(min(f.x, f.y), min(f.z, f.w)) != INT_MAX) {
                    atomicMin(&S.nan[mb][0], f.x);
                    atomicMin(&S.nan[mb][1], f.y);
                    atomicMin(&S.nan[mb][2], f.z);
                    atomicMin(&S.nan[mb][3], f.w);
                }
            }
            bar_and(3 + mb, 256, true);                // (exponents are there)
            int lim, lo = 0, pre = 0, at = 0;        // tokens that this row sees: below lim, and from lo on or below pre; its own place
            float slope = 0.f;
            {
                // (rows behind the last one, zeros, compute what that one's limit lets them: with none of the tokens each of their tiles
                // would be one that is cut, and these blocks, 1.6 times as long as the others, the launch's end)
                const int g = w.b.row0 + kRows * mb + r128, pos = min(pf_pos(P, g), w.b.n - 1);
                lim = P.causal ? max(0, min(w.b.len, w.b.len - w.b.n + 1 + pos)) : w.b.len;
                if (kMod) {
                    const Seq s{w.b.len, w.b.q0, w.b.n, 0};
                    pre = pg_prefix(P.sc, P.seq0 + w.b.si, w.b.len);
                    lim = max(lim, pre);
                    lo = pf_window(P, s, pos);
                    at = w.b.len - w.b.n + pos;
                    const int g_pos = pf_pos(P, g);
                    if (P.sc.slopes) slope = pg_slope(P.sc.slopes[(P.h0 + w.h) * P.gqa + g - g_pos * P.gqa]);
                }
            }
            float down0, down1;
            pg_pow2(-S.ex[mb][r128], down0, down1);
            const float sc = fmaxf((P.scale_log2 == 0.f ? 1.f : fabsf(P.scale_log2)) * down0 * down1, kPgFactorMin);
            // kCapped and on: logits are finished as they are loaded, and nothing is left to be multiplied by
            const float fac = kMode >= kCapped ? 1.f : sc;
            const bool even = __all_sync(0xffffffffu, S.ex[mb][r128] == 0);
            const uint8_t* const valid = P.valid + (int64_t)w.b.si * P.max_tiles + (kMod ? 0 : tile0);
            auto place = [&](int i) { return kMod ? w.b.slot<kBack>(tile0 + i, first_gap) : i; };   // of a tile among the sequence's valid[]
            uint32_t units = tiles > 0 ? valid[place(0)] : 0;
            float m_used = -INFINITY, lsum = 0.f;    // what this row scales by (log2), this half's denominator
            const float unit = kMode == kCapped ? pg_unit(sc, P.sc) : 0.f;
            float u_lim = -INFINITY;                 // kCapped: up to here logits are within the reference's reach (they rise no faster than what is capped)
            bool huge = false;                       // logits whose steps in fp32 are no longer small beside a weight's range
            for (int i = 0; i < tiles; ++i) {
                if (!__all_sync(0xffffffffu, pf_wait(S, &S.s_ready[mb], (uint32_t)(done + i) & 1u))) ok = false;
                tc_fence_after_sync();
                const int t0 = (kMod ? w.b.tile<kBack>(tile0 + i) : tile0 + i) * kPfTileTok + 64 * hf;
                const uint32_t there = units >> (4 * hf) & 15u;
                if (i + 1 < tiles) units = valid[place(i + 1)];
                // tiles that reach a row's limit, or lack a page
                const bool cut = !__all_sync(0xffffffffu, t0 + 64 <= lim && (!kMod || t0 >= lo || t0 + 64 <= pre)) || there != 15u;
                float sv[32];
                auto hide = [&](int c0) {              // kMod: what this row does not see of the tokens in sv
                    const uint32_t seen = bits_below(lim - t0 - c0) & (~bits_below(lo - t0 - c0) | bits_below(pre - t0 - c0)) &
                                          ((there >> (c0 >> 4) & 1u ? 0xffffu : 0u) | (there >> (c0 >> 4) & 2u ? 0xffff0000u : 0u));
#pragma unroll
                    for (int c = 0; c < 32; ++c) sv[c] = seen >> c & 1u ? sv[c] : -INFINITY;
                };
                auto load = [&](int c0) {
                    tmem_ld32(sS + (uint32_t)c0, sv);
                    tmem_ld_wait();
                    if (kMode >= kCapped) return;      // (made logits, and masked, elsewhere)
                    if (kMod && cut) {
                        hide(c0);
                    } else if (cut) {
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
                float m_half;
                int way = 0;                           // kCapped, where nothing is hidden and a polynomial reaches: 1 the short one, 2 the long one, beside the exponentials
                if constexpr (kMode == kCapped) {      // caps keep the order: the largest product's logit is the largest
                    float far;
                    load(32);
                    far = abs_top(sv);
                    if (cut) hide(32);
                    m_half = top();
                    load(0);
                    far = fmaxf(far, abs_top(sv));
                    if (cut) hide(0);
                    m_half = fmaxf(m_half, top());
                    m_half *= unit;                    // (u: capped where the reference may have to move)
                    if (!cut) way = even && __all_sync(0xffffffffu, far * far <= P.low_reach2) ? 1 : __all_sync(0xffffffffu, far * unit <= kMidReach) ? 2 : 0;
                } else if constexpr (kMode >= kBiased) {       // logits take their products' places
                    m_half = -INFINITY;
#pragma unroll 1
                    for (int c0 = 32; c0 >= 0; c0 -= 32) {
                        load(c0);
                        // (tokens behind a row's own place are in its sight only where it lies in the prefix, or sees all; its own one has no bias)
                        const int first = t0 + c0 - at;
                        pf_shape<kMode == kCappedBiased, true>(sv, P, sc, even, false, slope, (float)first,
                                                               __any_sync(0xffffffffu, first + 31 > 0 && (first <= 0 || lim > at + 1)), sS + (uint32_t)c0);
                        if (cut) hide(c0);
                        m_half = fmaxf(m_half, top());
                        if (c0) tmem_st32(sS + 32u, sv);
                    }
                    tmem_st_wait();
                } else {
                    load(32);
                    m_half = top();
                    load(0);
                    m_half = fmaxf(m_half, top()) * fac;
                }
                const bool last = more && i + 1 == tiles;
                if (last && w8 == 0) {                 // (the next block's record)
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                }
                const bool move = bar_or(1 + mb, (kMode == kCapped ? m_half > u_lim : m_half - m_used > kReach) || !ok);
                if (move) {
                    S.xch[mb][hf][r128] = m_half;
                    const bool all_ok = bar_and(3 + mb, 256, ok);
                    if (!all_ok) { ok = false; break; }              // (the same verdict for the whole block)
                    float top_m = fmaxf(m_half, S.xch[mb][hf ^ 1][r128]);
                    const float top_u = top_m;
                    if (kMode == kCapped && top_u > -INFINITY) top_m = pg_cap_any(top_u, P.sc);
                    // (where fp32's steps are wider than the distance, it becomes none)
                    const float m_new = top_m - (top_m - kLift) > kReach ? top_m : top_m - kLift;
                    float alpha = 1.f;
                    if (m_used == -INFINITY) m_used = m_new;         // nothing accumulated for this row yet
                    // (kMod: where the block's rows meet anyhow, all that have grown move: with logits of 4.8 to the base of 2, window of 2048, 373 us -> 347)
                    else if (top_m - m_used > (kMod ? kLift + 1.f : kReach)) {
                        alpha = pf_exp2(m_used - m_new);
                        m_used = m_new;
                    }
                    // (a reference that is huge is looked at every time: its steps are no longer small beside the reach)
                    if (kMode == kCapped && top_u > -INFINITY) u_lim = fabsf(m_used) < kHuge ? top_u + (m_used + kReach - top_m) * P.sc.cap_inv : -INFINITY;
                    huge = __any_sync(0xffffffffu, fabsf(m_used) >= kHuge && m_used > -INFINITY);
                    lsum *= alpha;
                    if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // O is at rest between the previous tile's product and this tile's
                        if (!__all_sync(0xffffffffu, pf_wait(S, &S.o_ready[mb], (uint32_t)(done + i - 1) & 1u))) ok = false;   // (ends at the next tile)
                        tc_fence_after_sync();
                        // (32 columns at a time, in the registers of the products, which are fetched anew: 626 to 647 us instead of 662 for logits of that size)
                        if (kMode >= kBiased) tmem_st32(sS, sv);
#pragma unroll 1
                        for (int ch = 0; ch < 2; ++ch) {
                            tmem_ld32(colO + 32u * ch, sv);
                            tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 32; ++c) sv[c] *= alpha;
                            tmem_st32(colO + 32u * ch, sv);
                        }
                        if (kMode >= kBiased) tmem_st_wait();
                        load(0);
                    }
                }
                if (last && w.next_tiles(next.b) > 0) fetch(next.b, w.next_h());        // (the last product with the queries is done)
                if (kMode == kCapped) {
                    if (huge) way = 0;                 // (product and difference rounded apart, as the reference was)
                    if (!way) {                        // logits take their products' places
#pragma unroll 1
                        for (int c0 = 32; c0 >= 0; c0 -= 32) {
                            load(c0);
                            pf_shape<true, false>(sv, P, sc, even, huge, 0.f, 0.f, false, sS + (uint32_t)c0);
                            if (cut) hide(c0);
                            if (c0) tmem_st32(sS + 32u, sv);
                        }
                        tmem_st_wait();
                    }
                }
                const float z = m_used == -INFINITY ? 0.f : m_used;
                const uint64_t nz2 = pack_f2(-z, -z), sc2 = huge ? pack_f2(1.f, 1.f) : pack_f2(fac, fac);
                uint64_t ps[2] = {0ull, 0ull};
                auto put = [&](uint32_t c0) {       // P of the columns in sv -> 16 columns of the half's own part of S
                    uint32_t pk[16];
                    if (kMode == kCapped && way) {
                        // (a pair is added up and packed behind the next one's exponentials: 688 us instead of 741, with a window 356 instead of 380)
                        auto finish = [&](int e) {
                            ps[e & 1] = add_f2(ps[e & 1], pack_f2(sv[2 * e], sv[2 * e + 1]));
                            pk[e] = pack_half2(sv[2 * e], sv[2 * e + 1]);
                        };
                        auto weigh = [&](auto logit) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                unpack_f2(logit(pack_f2(sv[2 * e], sv[2 * e + 1])), sv[2 * e], sv[2 * e + 1]);
                                sv[2 * e] = pf_exp2(sv[2 * e]);
                                sv[2 * e + 1] = pf_exp2(sv[2 * e + 1]);
                                if (e > 0) finish(e - 1);
                            }
                            finish(15);
                        };
                        if (way == 1) {
                            weigh([&](uint64_t r) { return fma_f2(r, pf_low(P, mul_f2(r, r)), nz2); });
                        } else {
                            const uint64_t g2 = pack_f2(unit, unit);
                            weigh([&](uint64_t r) {
                                const uint64_t u = mul_f2(r, g2);
                                return fma_f2(u, pf_mid(P, mul_f2(u, u)), nz2);
                            });
                        }
                        tmem_st16(sS + c0, pk);
                        return;
                    }
                    if (kMode < kCapped && huge) {  // product and difference rounded apart, as the reference was
#pragma unroll
                        for (int c = 0; c < 32; ++c) sv[c] = __fmul_rn(sv[c], fac);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float x0, x1, p0, p1;
                        const uint64_t s2 = pack_f2(sv[2 * e], sv[2 * e + 1]), x = kMode >= kCapped ? add_f2(s2, nz2) : fma_f2(s2, sc2, nz2);
                        unpack_f2(x, x0, x1);
                        if (kMode <= kMasked && (kPolyPairs >> e & 1) != 0) {
                            const uint64_t y = pack_f2(max_nan(x0, -125.f), max_nan(x1, -125.f));
                            pf_exp2_poly(y, p0, p1);
                            ps[e & 1] = fma_f2(y, 0ull, ps[e & 1]);      // (what is no number stays none in the denominator)
                        } else {
                            p0 = pf_exp2(x0);
                            p1 = pf_exp2(x1);
                        }
                        ps[e & 1] = add_f2(ps[e & 1], pack_f2(p0, p1));
                        pk[e] = pack_half2(p0, p1);
                    }
                    tmem_st16(sS + c0, pk);
                };
                // (the products of the halves' first 32 tokens start while the others' exponentials are taken)
                auto tell = [&](int part) {
                    tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.p_ready[mb][part]);
                };
                if constexpr (kMode >= kCapped) {      // (one piece of code for both: what it shapes logits with is long)
#pragma unroll 1
                    for (int part = 0; part < 2; ++part) {
                        if (part) load(32);
                        put(16u * part);
                        tell(part);
                    }
                } else {
                    put(0u);
                    tell(0);
                    load(32);
                    put(16u);
                    tell(1);
                }
                float a0, a1;
                unpack_f2(add_f2(ps[0], ps[1]), a0, a1);
                lsum += a0 + a1;
            }
            done += tiles;
            // ---- what comes next, and the rows' results, or their part of them ----
            if (more) {
                if (tiles == 0) {                      // (nobody waited for the record, nor fetched)
                    if (w8 == 0) {
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        __syncwarp();
                    }
                    bar_and(3 + mb, 256, true);
                }
                if (ok && w.next_tiles(next.b) > 0) {
                    if (tiles == 0) fetch(next.b, w.next_h());
                    ready();
                }
            }
            if (tiles > 0 && ok) {
                ok = __all_sync(0xffffffffu, pf_wait(S, &S.o_ready[mb], (uint32_t)(done - 1) & 1u));
                tc_fence_after_sync();
            }
            bool bad0 = S.nan[mb][2 * hf] < lim, bad1 = S.nan[mb][2 * hf + 1] < lim;
            if (kMod && (bad0 || bad1)) {              // (the first may be hidden, and a later one not)
                bad0 = bad1 = false;
                for (int i = 0; i < tiles; ++i) {
                    const uint32_t* const bits = P.nan_bits + 16 * (((int64_t)w.b.si * P.n_h + w.h) * P.max_tiles + place(i)) + 8 * hf;
                    for (int k = 0; k < 4; ++k) {
                        const int t = w.b.tile<kBack>(tile0 + i) * kPfTileTok + 32 * k;
                        const uint32_t seen = bits_below(lim - t) & (~bits_below(lo - t) | bits_below(pre - t));
                        bad0 |= (bits[k] & seen) != 0;
                        bad1 |= (bits[4 + k] & seen) != 0;
                    }
                }
            }
            bar_and(3 + mb, 256, true);                // (maxima, and which numbers are none, are read before their places change)
            S.xch[mb][hf][r128] = lsum;
            if ((tid & 255) < 4) S.nan[mb][tid & 3] = INT_MAX;
            if ((tid & 255) == 0 && more) next.step_from(w);
            if (!bar_and(3 + mb, 256, ok)) {
                ok = false;
                break;
            }
            lsum += S.xch[mb][hf ^ 1][r128];
            const bool whole = w.whole();
            const float inv = !whole ? 1.f : lsum > 0.f ? 1.0f / lsum : lsum == 0.f ? 0.f : lsum;
            const size_t slot = (size_t)(2 * blockIdx.x + (w.first ? 0 : 1)) * kBlockRows + kRows * mb + (warp & 3) * 32;
            uint8_t* const st = S.stage[warp];         // 64 bytes per row, 16-byte pieces exchanged by row
            auto stage = [&](int c, uint4 v) { *reinterpret_cast<uint4*>(st + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)) = v; };
            auto staged = [&](int r32) { return *reinterpret_cast<const uint4*>(st + r32 * 64 + (((lane & 3) ^ (r32 >> 1 & 3)) << 4)); };
            const bool wide = ((reinterpret_cast<uintptr_t>(P.out) | (uint64_t)(2 * P.o_st) | (uint64_t)(2 * P.o_sh)) & 15u) == 0;
            T* to[4];                                  // rows lane / 4 + 8 k, this lane's piece; null: none
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int gr = w.b.row0 + kRows * mb + (warp & 3) * 32 + (lane >> 2) + 8 * k, pr = pf_pos(P, gr);
                to[k] = pr < w.b.n ? reinterpret_cast<T*>(P.out) + (int64_t)(w.b.q0 + pr) * P.o_st +
                                         (int64_t)((P.h0 + w.h) * P.gqa + gr - pr * P.gqa) * P.o_sh + 64 * hf + 8 * (lane & 3)
                                   : nullptr;
            }
#pragma unroll 1
            for (int ch = 0; ch < 2; ++ch) {
                float o[32];
                if (tiles > 0) {
                    tmem_ld32(colO + 32u * ch, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0.f;
                }
                const float f = (ch ? bad1 : bad0) ? __uint_as_float(0x7fffffffu) : inv;
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        stage(c, make_uint4(PgType<T>::down(o[8 * c] * f, o[8 * c + 1] * f), PgType<T>::down(o[8 * c + 2] * f, o[8 * c + 3] * f),
                                            PgType<T>::down(o[8 * c + 4] * f, o[8 * c + 5] * f), PgType<T>::down(o[8 * c + 6] * f, o[8 * c + 7] * f)));
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 v = staged((lane >> 2) + 8 * k);
                        if (!to[k]) continue;
                        uint2* const dst = reinterpret_cast<uint2*>(to[k] + 32 * ch);
                        if (wide) {
                            *reinterpret_cast<uint4*>(dst) = v;
                        } else {
                            dst[0] = make_uint2(v.x, v.y);
                            dst[1] = make_uint2(v.z, v.w);
                        }
                    }
                    __syncwarp();
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float* x = o + 16 * half + 4 * c;
                            stage(c, make_uint4(__float_as_uint(x[0] * f), __float_as_uint(x[1] * f), __float_as_uint(x[2] * f), __float_as_uint(x[3] * f)));
                        }
                        __syncwarp();
#pragma unroll 1
                        for (int r32 = lane >> 2; r32 < 32; r32 += 8)
                            *reinterpret_cast<uint4*>(P.part_o + (slot + r32) * kHD + 64 * hf + 32 * ch + 16 * half + 4 * (lane & 3)) = staged(r32);
                        __syncwarp();
                    }
                }
            }
            if (hf == 0) {
                const int g = w.b.row0 + kRows * mb + r128, pos = pf_pos(P, g);
                if (!whole)
                    P.part_ml[slot + lane] = make_float2(m_used, lsum);
                else if (pos < w.b.n && P.lse)
                    P.lse[(int64_t)(w.b.q0 + pos) * P.n_q + (P.h0 + w.h) * P.gqa + g - pos * P.gqa] =
                        lsum == 0.f ? -INFINITY : (m_used + log2f(lsum)) * 0.693147180559945309f;
            }
            tc_fence_before_sync();                    // (O is read before the next block's first product into it)
            bar_and(3 + mb, 256, true);                // (and this block's record, before the one after the next takes its place)
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kWarpMma) tmem_dealloc(tmem, kTmemCols);
    if (tid == 0 && S.failed && P.status) *P.status = kStatusWaitTimeout;
}

// ------------------------------------------------------------------------------------------------------------------
// merge: block (i, y) 32 rows of the block that the end of CTA i's share cuts, if that is its first cut; a warp four of them at a time, so that what
// is looked up first, three loads one behind the other, is looked up for 32 rows together.
// Bound: memory, at most 148 cuts x 256 rows x two parts of 520 bytes, 39 MB that are still in L2.
// ------------------------------------------------------------------------------------------------------------------
constexpr int kMergeRows = 4;
template <typename T>
__global__ void __launch_bounds__(256) pg_prefill_merge_kernel(const Pf P) {
    const int lane = threadIdx.x & 31, row0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * kMergeRows, j0 = blockIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    const int4 a = P.start[j0], b = P.start[j0 + 1];
    const int all = P.start[P.n_cta].w, behind = P.start[min(j0 + 2 + lane, P.n_cta)].w;
    if (b.w == all || b.y == 0) return;                         // nothing behind, or cut between blocks
    const bool same = a.x == b.x && a.z == b.z;                 // the CTA's only block
    if (same && a.y > 0) return;                                // (cut before)
    const Block bk = P.blk[b.x];
    const int end = b.w - b.y + bk.tiles;
    int j1 = j0 + 1;                                            // the last CTA that holds a part of it
    for (int w = behind;; w = P.start[min(j1 + 1 + lane, P.n_cta)].w) {
        const uint32_t more = __ballot_sync(0xffffffffu, j1 + 1 + lane < P.n_cta && w < end);
        j1 += __popc(more);
        if (more != 0xffffffffu) break;
    }
    float m[kMergeRows], l[kMergeRows];
    float4 o[kMergeRows];
#pragma unroll
    for (int i = 0; i < kMergeRows; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int j = j0; j <= j1; ++j) {
        const size_t slot = (size_t)(2 * j + (j == j0 && !same ? 1 : 0)) * kBlockRows + row0;
        float2 ml[kMergeRows];
        float4 v[kMergeRows];
#pragma unroll
        for (int i = 0; i < kMergeRows; ++i) {
            ml[i] = P.part_ml[slot + i];
            v[i] = *reinterpret_cast<const float4*>(P.part_o + (slot + i) * kHD + 4 * lane);
        }
#pragma unroll
        for (int i = 0; i < kMergeRows; ++i) {
            const float top = fmaxf(m[i], ml[i].x), z = top == -INFINITY ? 0.f : top, f = pf_exp2(m[i] - z), f1 = pf_exp2(ml[i].x - z);
            l[i] = fmaf(f1, ml[i].y, l[i] * f);
            o[i].x = fmaf(f1, v[i].x, o[i].x * f); o[i].y = fmaf(f1, v[i].y, o[i].y * f);
            o[i].z = fmaf(f1, v[i].z, o[i].z * f); o[i].w = fmaf(f1, v[i].w, o[i].w * f);
            m[i] = top;
        }
    }
#pragma unroll
    for (int i = 0; i < kMergeRows; ++i) {
        const int g = bk.row0 + row0 + i, pos = pf_pos(P, g);
        if (pos >= bk.n) return;
        const int hq = (P.h0 + b.z) * P.gqa + g - pos * P.gqa;
        const float inv = l[i] > 0.f ? 1.0f / l[i] : l[i] == 0.f ? 0.f : l[i];
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(P.out) + (int64_t)(bk.q0 + pos) * P.o_st + (int64_t)hq * P.o_sh + 4 * lane) =
            make_uint2(PgType<T>::down(o[i].x * inv, o[i].y * inv), PgType<T>::down(o[i].z * inv, o[i].w * inv));
        if (P.lse && lane == 0) P.lse[(int64_t)(bk.q0 + pos) * P.n_q + hq] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * 0.693147180559945309f;
    }
}

}  // namespace

// Sequences and KV heads of one launch's workspace: all of them, or fewer sequences, then fewer heads, so that their tiles stay within 2 GiB.
// With a window, a sequence of n rows has no more than its prefix's tiles and those of n - 1 + window tokens from any place on.
static void pf_parts(int n_seq, int n_tok, int n_kv, int64_t max_tokens, const PgScores* sc, int& seqs, int& heads, int64_t& tiles) {
    constexpr int64_t kMost = 2ll << 30;
    auto whole = [](int64_t tokens) { return (tokens + kPfTileTok - 1) / kPfTileTok; };
    tiles = whole(max_tokens);
    if (sc && sc->window) tiles = std::min(tiles, whole(sc->prefix ? sc->max_prefix : 0) + whole((int64_t)n_tok - 1 + sc->window) + 1);
    if (tiles < 1) tiles = 1;
    const int64_t pairs = kMost / (tiles * kPfTileBytes);
    heads = (int)(pairs >= n_kv ? n_kv : pairs > 1 ? pairs : 1);
    seqs = (int)(pairs / n_kv >= n_seq ? n_seq : pairs / n_kv > 1 ? pairs / n_kv : 1);
    if (seqs > 65535) seqs = 65535;
}

// Where a launch's pieces lie in the workspace.
struct PfLayout {
    int64_t nan, part_o, part_ml, start, blk, first, valid, nan_bits, total;
};
static int pf_ctas() {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}
static PfLayout pf_layout(int seqs, int heads, int64_t tiles, int64_t blocks, int n_cta, bool mod) {
    PfLayout L;
    L.nan = seqs * tiles * heads * (int64_t)kPfTileBytes;
    L.part_o = L.nan + seqs * tiles * heads * 16;
    L.part_ml = L.part_o + 2ll * n_cta * kBlockRows * kHD * 4;
    L.start = L.part_ml + 2ll * n_cta * kBlockRows * 8;
    L.blk = L.start + 16ll * (n_cta + 2);
    L.first = L.blk + (int64_t)sizeof(Block) * (blocks + 1);
    L.valid = L.first + 4 * (blocks + 1);
    L.nan_bits = (L.valid + seqs * tiles + 15) / 16 * 16;
    L.total = mod ? L.nan_bits + seqs * tiles * heads * 64 : L.valid + seqs * tiles;
    return L;
}

int64_t paged_prefill_workspace(int n_seq, int n_tok, int gqa, int n_kv, int64_t max_tokens, const PgScores* sc) {
    int seqs, heads;
    int64_t tiles;
    pf_parts(n_seq, n_tok, n_kv, max_tokens, sc, seqs, heads, tiles);
    return pf_layout(seqs, heads, tiles, (int64_t)n_tok * gqa / kBlockRows + n_seq, pf_ctas(), sc != nullptr).total;
}

// What pf_shape takes from the launch's parameters.
static void pf_constants(Pf& P) {
    auto pair = [](double a, double b) {
        const float f[2] = {(float)a, (float)b};
        uint64_t bits;
        memcpy(&bits, f, 8);
        return bits;
    };
    for (int i = 0; i < 16; ++i) P.steps[i] = pair(2 * i - 31, 2 * i - 30);
    for (int i = 0; i < kMidTerms; ++i) P.mid[i] = pair(kCapMid[i] * P.sc.cap, kCapMid[i] * P.sc.cap);
    // u = product * g; where fp32 has no normal numbers for the coefficients, the polynomial is for no product
    const double factor = P.scale_log2 == 0.f ? 1.0 : fabs((double)P.scale_log2), g = factor * P.sc.cap_inv;
    double k = factor;
    bool good = true;
    for (int i = 0; i < kLowTerms; ++i, k *= g * g) {
        P.low[i] = pair(kCapLow[i] * k, kCapLow[i] * k);
        good = good && k > 1e-35 && k < 1e35;
    }
    P.low_reach2 = good ? (float)(kLowReach / g * (kLowReach / g)) : -1.f;
}

int paged_prefill(const PagedPrefill& A, cudaStream_t stream) {
    int seqs, heads;
    int64_t tiles;
    pf_parts(A.n_seq, A.n_tok, A.n_kv, A.max_tokens, A.mod ? &A.sc : nullptr, seqs, heads, tiles);
    const int64_t blocks = (int64_t)A.n_tok * A.gqa / kBlockRows + A.n_seq;
    // (a launch's tiles are counted in 32 bits, rows to 2^29)
    if (2 * (double)blocks * (double)(tiles + 2) * heads > INT32_MAX || (int64_t)A.n_tok * A.gqa > 1 << 29) return BGTQ_E_TOOBIG;
    const int n_cta = pf_ctas();
    const PfLayout L = pf_layout(seqs, heads, tiles, blocks, n_cta, A.mod);
    uint8_t* const ws = A.workspace;
    const auto unpack = A.mod ? pg_unpack_kernel<true> : pg_unpack_kernel<false>;
    const PgMode mode = pg_mode(A.sc, A.mod);
    constexpr decltype(&pg_prefill_kernel<__half, kPlain>) kernels[5][2] = {{pg_prefill_kernel<__half, kPlain>, pg_prefill_kernel<__nv_bfloat16, kPlain>},
                                                                            {pg_prefill_kernel<__half, kMasked>, pg_prefill_kernel<__nv_bfloat16, kMasked>},
                                                                            {pg_prefill_kernel<__half, kCapped>, pg_prefill_kernel<__nv_bfloat16, kCapped>},
                                                                            {pg_prefill_kernel<__half, kBiased>, pg_prefill_kernel<__nv_bfloat16, kBiased>},
                                                                            {pg_prefill_kernel<__half, kCappedBiased>, pg_prefill_kernel<__nv_bfloat16, kCappedBiased>}};
    const auto kernel = kernels[mode][A.bf16];
    const auto merge = A.bf16 ? pg_prefill_merge_kernel<__nv_bfloat16> : pg_prefill_merge_kernel<__half>;
    static std::atomic<uint64_t> allowed[10];
    if (!pg_allow_smem(kernel, (int)sizeof(PfSmem), allowed[2 * mode + A.bf16])) return BGTQ_E_LAUNCH;
    for (int s0 = 0; s0 < A.n_seq; s0 += seqs)
        for (int h0 = 0; h0 < A.n_kv; h0 += heads) {
            const int ns = A.n_seq - s0 < seqs ? A.n_seq - s0 : seqs, nh = A.n_kv - h0 < heads ? A.n_kv - h0 : heads;
            Pf P{};
            P.pool = A.pool;
            P.table = A.table; P.tb_st = A.tb_st; P.lens = A.lens; P.cu_q = A.cu_q;
            P.cap = A.cap; P.n_tok = A.n_tok; P.n_q = A.n_q; P.n_kv = A.n_kv; P.gqa = A.gqa; P.causal = A.causal;
            P.gqa_inv = A.gqa > 1 ? (uint32_t)(0x100000000ull / A.gqa + (0x100000000ull % A.gqa != 0)) : 0;
            P.seq0 = s0; P.n_seq = ns; P.h0 = h0; P.n_h = nh; P.max_tiles = (int32_t)tiles;
            P.tiles = ws;
            P.nan = reinterpret_cast<int4*>(ws + L.nan);
            P.part_o = reinterpret_cast<float*>(ws + L.part_o);
            P.part_ml = reinterpret_cast<float2*>(ws + L.part_ml);
            P.start = reinterpret_cast<int4*>(ws + L.start);
            P.blk = reinterpret_cast<Block*>(ws + L.blk);
            P.first = reinterpret_cast<int32_t*>(ws + L.first);
            P.valid = ws + L.valid;
            P.max_blocks = (int32_t)blocks; P.n_cta = n_cta;
            P.q = A.q; P.q_st = A.q_st; P.q_sh = A.q_sh; P.scale_log2 = A.scale_log2;
            P.out = A.out; P.o_st = A.o_st; P.o_sh = A.o_sh; P.lse = A.lse; P.status = A.status;
            P.sc = A.sc;
            pf_constants(P);
            P.nan_bits = reinterpret_cast<uint32_t*>(ws + L.nan_bits);
            if (!pg_launch_ok(launch_kernel(unpack, dim3((unsigned)tiles + 1, nh, ns), dim3(256), 0, stream, true, P))) return BGTQ_E_LAUNCH;
            if (!pg_launch_ok(launch_kernel(kernel, dim3(n_cta), dim3(kThreads), sizeof(PfSmem), stream, true, P))) return BGTQ_E_LAUNCH;
            if (!pg_launch_ok(launch_kernel(merge, dim3(n_cta - 1, kBlockRows / (8 * kMergeRows)), dim3(256), 0, stream, true, P))) return BGTQ_E_LAUNCH;
        }
    return BGTQ_OK;
}

}  // namespace bgtq
