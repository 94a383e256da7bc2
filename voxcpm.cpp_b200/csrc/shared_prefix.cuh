// What vox_attn_decode_shared asks of the decode kernel (decode_attn.cu) for the streams' own rows.
#pragma once

#include "kv_cache.cuh"

namespace vox {

// results beside dst: per (stream, head) the natural log-sum-exp and the (max, sum) in units of log2 (NULL: not wanted)
struct OwnRows {
    float *  lse;
    float2 * ml;
    int      wave;    // CTAs per SM at most, where the prefix kernel is to run beside it (0: all that fit)
};
int    check_decode(const vox_engine * e, const vox_decode_args * a, const char * who);
int    launch_decode_shared(vox_engine * e, const vox_decode_args * a, const OwnRows & rows, void * workspace, size_t workspace_bytes,
                            cudaStream_t stream);
size_t decode_shared_workspace_bytes(int n_streams, int n_heads, int n_kv_heads, int kv_bound);

}  // namespace vox
