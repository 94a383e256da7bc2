// vox_kv_observe: what its kernels share.  One query per stream, windows of few query rows: kv_observe.cu; others: kv_observe_window.cu.
#pragma once

#include "kv_cache.cuh"

#include <algorithm>

namespace vox {

constexpr int kObserveMaxQ = 64;

struct ObserveParams {
    const uint8_t * k;         // f16: the layer's K rows; q8_0: the layer's tiles
    size_t          k_nb_head, k_nb_stream;
    const int32_t * kv_len;
    const int32_t * n_seen;
    const uint8_t * q;
    size_t          q_nb_head, q_nb_tok, q_nb_stream;
    const float2 *  rope;
    const float *   lse;
    float           scale_log2, decay;
    int             n_streams, n_heads, n_kv_heads, gqa, layer, n_q, n_new, kv_bound, n_chunks;
    int             run;       // one query: chunks of a CTA
    uint8_t *       score;
    uint8_t *       row_pos;
    size_t          nb_head, nb_stream;
    uint32_t        gqa_magic; // row * gqa_magic >> 16 = row / gqa for rows below 512
    float2 *        stats;     // (max, sum) of every row over a part of the keys
    int *           status;
};

size_t observe_window_bytes(int n_streams, int n_kv_heads, int rows, int kv_bound);
int    launch_observe_window(vox_engine * e, const vox_kv_cache * c, const ObserveParams & p, cudaStream_t st);

}  // namespace vox
