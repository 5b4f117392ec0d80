// The tcgen05 form of the paged attention (bgtq_paged_prefill.cu), called by bgtq_paged_attend where there are rows enough.
#pragma once
#include "bgtq_paged_common.cuh"

namespace bgtq {

constexpr int kPfTileTok = 128;                             // cache tokens of a tile
constexpr int kPfTileBytes = 2 * kPfTileTok * kHD * 2;      // its khat and vhat in the workspace

struct PagedPrefill {
    PgPool pool;
    const int32_t* table;
    int64_t tb_st;
    const int32_t *lens, *cu_q;
    int32_t n_seq, n_tok, n_q, n_kv, gqa, causal, bf16;
    int64_t max_tokens;             // the workspace's
    int32_t cap;                    // sequences are held to it: max_tokens and what the table holds
    uint8_t* workspace;
    const void* q;
    int64_t q_st, q_sh;             // elements; rows on 16-byte boundaries
    float scale_log2;
    void* out;
    int64_t o_st, o_sh;
    float* lse;
    int32_t* status;
};
int64_t paged_prefill_workspace(int n_seq, int n_tok, int gqa, int n_kv, int64_t max_tokens);
int paged_prefill(const PagedPrefill& A, cudaStream_t stream);

}  // namespace bgtq
