// Copying pages of the paged 4-bit cache: page dst[i] of every layer and KV head becomes page src[i], or the units that hold its first tokens.
//
// The pairs lie on the host, where the pages are handed out, and travel as the launch's parameters: no transfer of their own, and the host has seen
// that no page is written twice or read and written.
//
// A row is what lies in one piece of a pair: a layer's page of all heads where the heads follow one another and pages are whole, otherwise of one head.
// A block copies a piece of a row, 16 KB: each thread four times 16 bytes, all of them on their way before the first is stored.
// Bound: memory, every byte once in and once out.  256 pages of 64 tokens in 32 layers of 8 KV heads, 604 MB: 185 us, 6.52 TB/s, what a plain copy of such a
// size gets.  32 half-filled pages in 36 layers of 2 heads, 13 MB: 5.2 us, a launch and one round of loads and stores.
#include "bgtq_paged_common.cuh"
#include "bgtq_paged_rows.h"

#include <limits.h>
#include <stdlib.h>
#include <string.h>

namespace bgtq {
namespace {

constexpr int kPcThreads = 256, kPcEach = 4;
constexpr int kPcPiece = kPcThreads * kPcEach * 16;

struct PcPair {
    int32_t src, dst, units;
};
struct PcPool {
    int64_t layer, page, head;       // bytes from one to the next
};
template <int N>
struct PcParams {
    const uint8_t* from;
    uint8_t* to;
    PcPool f, t;
    int32_t layers, heads, pieces;   // heads: rows of a layer's page; pieces of the longest row
    int32_t unit_bytes;              // of a row
    PcPair pair[N];
};

template <int N>
__global__ void __launch_bounds__(kPcThreads) pg_copy_kernel(const __grid_constant__ PcParams<N> P) {
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t piece = blockIdx.x % (uint32_t)P.pieces, row = blockIdx.x / (uint32_t)P.pieces;
    const uint32_t head = row % (uint32_t)P.heads, rest = row / (uint32_t)P.heads, layer = rest % (uint32_t)P.layers;
    const PcPair p = P.pair[rest / (uint32_t)P.layers];
    const int64_t bytes = (int64_t)p.units * P.unit_bytes, at = (int64_t)piece * kPcPiece + threadIdx.x * 16;
    const uint8_t* const src = P.from + layer * P.f.layer + p.src * P.f.page + head * P.f.head + at;
    uint8_t* const dst = P.to + layer * P.t.layer + p.dst * P.t.page + head * P.t.head + at;
    uint4 v[kPcEach];
#pragma unroll
    for (int i = 0; i < kPcEach; ++i)
        if (at + i * kPcThreads * 16 < bytes) v[i] = *reinterpret_cast<const uint4*>(src + i * kPcThreads * 16);
#pragma unroll
    for (int i = 0; i < kPcEach; ++i)
        if (at + i * kPcThreads * 16 < bytes) *reinterpret_cast<uint4*>(dst + i * kPcThreads * 16) = v[i];
}

// Whether a number of b is among those of a, or (a == b) there twice.  Few are compared with one another, many marked in a set of bits; < 0: no memory.
int pc_common(const int32_t* a, const int32_t* b, int32_t n, int32_t n_pages) {
    const bool same = a == b;
    if (n <= 48) {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < (same ? i : n); ++j)
                if (b[i] == a[j]) return 1;
        return 0;
    }
    uint64_t* const seen = static_cast<uint64_t*>(calloc(((size_t)n_pages + 63) / 64, 8));
    if (!seen) return -1;
    int found = 0;
    auto mark = [&](int32_t x) {
        const uint64_t bit = 1ull << (x & 63);
        const bool was = seen[x >> 6] & bit;
        seen[x >> 6] |= bit;
        return was;
    };
    if (same) {
        for (int i = 0; i < n && !found; ++i) found = mark(a[i]);
    } else {
        for (int i = 0; i < n; ++i) mark(a[i]);
        for (int i = 0; i < n && !found; ++i) found = (seen[b[i] >> 6] >> (b[i] & 63)) & 1;
    }
    free(seen);
    return found;
}

// The places of a pool, (layers, pages, heads) of `row` bytes, do not overlap: along the strides in order, each step is past all that lies within it.
bool pc_apart(const PcPool& s, int64_t layers, int64_t pages, int64_t heads, int64_t row) {
    int64_t n[3] = {layers, pages, heads}, st[3] = {s.layer, s.page, s.head};
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2 - i; ++j)
            if ((n[j] > 1 && st[j] > st[j + 1]) || n[j + 1] <= 1) {
                const int64_t a = n[j], b = st[j];
                n[j] = n[j + 1]; st[j] = st[j + 1];
                n[j + 1] = a; st[j + 1] = b;
            }
    int64_t span = row;
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (st[i] < span) return false;
        span += (n[i] - 1) * st[i];
    }
    return true;
}
int64_t pc_span(const PcPool& s, int64_t layers, int64_t pages, int64_t heads, int64_t row) {
    return (layers - 1) * s.layer + (pages - 1) * s.page + (heads - 1) * s.head + row;
}

template <int N>
bool pc_launch(PcParams<N>& P, const int32_t* src, const int32_t* dst, const int32_t* n_tokens, int32_t n, int32_t units, int64_t blocks_of_pair, cudaStream_t stream) {
    for (int32_t i = 0; i < n; ++i) P.pair[i] = PcPair{src[i], dst[i], n_tokens ? (n_tokens[i] + kUnitTok - 1) / kUnitTok : units};
    return pg_launch_ok(launch_kernel(pg_copy_kernel<N>, dim3((unsigned)(n * blocks_of_pair)), dim3(kPcThreads), 0, stream, true, P));
}

}  // namespace
}  // namespace bgtq

using namespace bgtq;

extern "C" __attribute__((visibility("default"))) int bgtq_paged_copy(
    const uint8_t* from, int64_t f_layer, int64_t f_page, int64_t f_head, int32_t n_from, uint8_t* to, int64_t t_layer, int64_t t_page, int64_t t_head,
    int32_t n_to, int32_t page_tokens, int32_t n_layers, int32_t n_kv, const int32_t* src, const int32_t* dst, const int32_t* n_tokens, int32_t n, void* stream) {
    pg_launched = 0;
    if (!from || !to || n < 0 || n_from < 1 || n_to < 1 || n_layers < 1 || n_kv < 1 || page_tokens < kUnitTok || page_tokens % kUnitTok) return BGTQ_E_BADARG;
    if (n == 0) return BGTQ_OK;
    if (!src || !dst) return BGTQ_E_BADARG;
    if ((reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to) | (uint64_t)(f_layer | f_page | f_head | t_layer | t_page | t_head)) & 15u) return BGTQ_E_ALIGN;
    if (f_layer < 0 || f_page < 0 || f_head < 0 || t_layer < 0 || t_page < 0 || t_head < 0) return BGTQ_E_BADARG;
    const int32_t units = page_tokens / kUnitTok;
    const int64_t page_bytes = (int64_t)units * kUnitBytes;
    const PcPool f{f_layer, f_page, f_head}, t{t_layer, t_page, t_head};
    for (int32_t i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= n_from || dst[i] < 0 || dst[i] >= n_to || (n_tokens && (n_tokens[i] < 0 || n_tokens[i] > page_tokens))) return BGTQ_E_BADARG;
    if (!pc_apart(t, n_layers, n_to, n_kv, page_bytes)) return BGTQ_E_BADARG;
    const bool same = from == to && (n_layers == 1 || f_layer == t_layer) && (n_from == 1 || f_page == t_page) && (n_kv == 1 || f_head == t_head);
    if (!same) {         // pools of their own, apart from one another
        const uintptr_t a = reinterpret_cast<uintptr_t>(from), b = reinterpret_cast<uintptr_t>(to);
        if (a < b + pc_span(t, n_layers, n_to, n_kv, page_bytes) && b < a + pc_span(f, n_layers, n_from, n_kv, page_bytes)) return BGTQ_E_BADARG;
    }
    int found = pc_common(dst, dst, n, n_to);
    if (!found && same) found = pc_common(src, dst, n, n_to);
    if (found) return found < 0 ? BGTQ_E_TOOBIG : BGTQ_E_BADARG;

    const bool joined = !n_tokens && (n_kv == 1 || (f_head == page_bytes && t_head == page_bytes));
    const int32_t heads = joined ? 1 : n_kv;
    const int64_t unit_bytes = joined ? (int64_t)n_kv * kUnitBytes : kUnitBytes, pieces = (units * unit_bytes + kPcPiece - 1) / kPcPiece;
    if (unit_bytes > INT32_MAX) return BGTQ_E_TOOBIG;
    const int64_t blocks = pieces * heads * n_layers;           // of a pair
    if (blocks > INT32_MAX) return BGTQ_E_TOOBIG;
    auto fill = [&](auto& P) {
        P.from = from; P.to = to; P.f = f; P.t = t;
        P.layers = n_layers; P.heads = heads; P.pieces = (int32_t)pieces; P.unit_bytes = (int32_t)unit_bytes;
    };
    // As many pairs as the launch's parameters hold: 4 KB of them in most calls, 32 KB where there are more.
    constexpr int kFew = 320, kMany = 2700;
    PcParams<kFew> few;
    fill(few);
    static_assert(sizeof(PcParams<kFew>) <= 4096 && sizeof(PcParams<kMany>) <= 32764, "what a launch's parameters hold");
    const int64_t most = INT32_MAX / blocks;
    for (int32_t i = 0; i < n;) {
        int64_t take = n - i < most ? n - i : most;
        const int32_t* const count = n_tokens ? n_tokens + i : nullptr;
        bool ok;
        if (take <= kFew) {
            ok = pc_launch(few, src + i, dst + i, count, (int32_t)take, units, blocks, (cudaStream_t)stream);
        } else {
            static thread_local PcParams<kMany> many;
            fill(many);
            if (take > kMany) take = kMany;
            ok = pc_launch(many, src + i, dst + i, count, (int32_t)take, units, blocks, (cudaStream_t)stream);
        }
        if (!ok) return BGTQ_E_LAUNCH;
        i += (int32_t)take;
    }
    return BGTQ_OK;
}
