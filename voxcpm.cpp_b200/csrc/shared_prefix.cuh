// What the kernel of the shared rows (shared_decode.cu) and the decode kernel that folds its results agree on.
//
// Streams that share a prefix are packed into row tiles: the queries of up to 128 / gqa streams of one prefix, gqa rows per
// stream (row = place in the tile * gqa + head of the group), per kv head.  The keys of a prefix are cut into chunks; one
// (row tile, kv head, chunk) is one partial result: per row (max, sum) in units of log2 and the unnormalised output.
#pragma once

#include "kv_cache.cuh"

namespace vox {

constexpr int kPrefixRows = 128;       // rows of a row tile
constexpr int kPrefixMaxChunks = 64;   // partials per row at most
// DecodeParams::early of a decode launch whose predecessor on the stream is the kernel of the shared rows
constexpr int kBehindPrefix = 2;

struct PrefixFold {
    const float2 *  ml;       // [slot][kPrefixRows] (max, sum); NULL: no shared rows in this call
    const float4 *  acc;      // [slot][16][kPrefixRows]: output columns 4c .. 4c+3 of a row at [c][row]
    const int32_t * place;    // [stream] row tile * kPrefixRows + place in the tile, -1: the stream shares nothing
    const int32_t * of;       // [stream] its prefix
    const int32_t * len;      // [prefix] rows
    int             max_len;  // rows the prefix cache holds
    int             chunk, max_chunks;
};

// what a decode launch takes beside the arguments of vox_attn_decode
struct SharedRows {
    PrefixFold fold;  // fold.ml == NULL: no shared rows
    float *    lse;
};
int    check_decode(const vox_engine * e, const vox_decode_args * a, const char * who);
int    launch_decode_shared(vox_engine * e, const vox_decode_args * a, const SharedRows & rows, void * workspace, size_t workspace_bytes,
                            cudaStream_t stream);
size_t decode_workspace_bytes(int n_streams, int n_heads, int n_kv_heads, int kv_bound);

// chunks that hold rows of a prefix of `len` rows: the last one takes whatever lies past max_chunks * chunk
__host__ __device__ inline int prefix_chunks(int len, int chunk, int max_chunks) {
    const int n = (len + chunk - 1) / chunk;
    return n < max_chunks ? n : max_chunks;
}

#ifdef __CUDACC__
// Folds the partials of one row, output columns d0 .. d0+3, into (M, L, acc), in key order whatever order they were made in.
__device__ __forceinline__ void prefix_fold(const PrefixFold & f, int stream, int kvh, int hh, int n_kv_heads, int gqa, int d0, float & M,
                                            float & L, float (&acc)[4]) {
    const int place = f.place[stream];
    if (place < 0) return;
    const int n    = prefix_chunks(max(0, min(f.len[f.of[stream]], f.max_len)), f.chunk, f.max_chunks);
    const int tile = place / kPrefixRows;
    const int    row  = (place - tile * kPrefixRows) * gqa + hh;
    const size_t slot = (size_t) (tile * n_kv_heads + kvh) * f.max_chunks;
    constexpr int W = 4;  // partials in flight: each is a round trip to L2
    for (int c = 0; c < n; c += W) {
        float2 ml[W];
        float4 o[W];
#pragma unroll
        for (int u = 0; u < W; ++u) {
            const size_t at = slot + min(c + u, n - 1);
            ml[u] = __ldcg(f.ml + at * kPrefixRows + row);
            o[u]  = __ldcg(f.acc + (at * 16 + (d0 >> 2)) * kPrefixRows + row);
        }
#pragma unroll
        for (int u = 0; u < W; ++u) {
            if (c + u >= n || (ml[u].x == -INFINITY && ml[u].y == 0.0f)) continue;
            const float Mn = fmaxf(M, ml[u].x), fo = exp2f(M - Mn), fw = exp2f(ml[u].x - Mn);
            M      = Mn;
            L      = L * fo + ml[u].y * fw;
            acc[0] = acc[0] * fo + o[u].x * fw;
            acc[1] = acc[1] * fo + o[u].y * fw;
            acc[2] = acc[2] * fo + o[u].z * fw;
            acc[3] = acc[3] * fo + o[u].w * fw;
        }
    }
}
#endif

}  // namespace vox
