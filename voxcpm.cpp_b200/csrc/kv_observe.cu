// The attention weight that every cache row receives, summed over the queries and heads that look at it (vox_kv_observe).
//
//   score[j] = (j new ? 0 : decay * score[j]) + sum_rows 2^(s[row][j] - lse[row]),   s = scale * log2 e * q.k
//
// V plays no part, so a call reads K (128 or 68 bytes a row) and 8 bytes of score: bound by HBM for a decode step, by the
// exponentials and products for a window of queries.
#include "kv_cache.cuh"

#include <algorithm>

using namespace vox;

namespace {

constexpr int kWarps     = 8;
constexpr int kThreads   = kWarps * 32;
constexpr int kWarpKeys  = 64;                  // keys a warp keeps as operands
constexpr int kChunk     = kWarps * kWarpKeys;  // keys of a CTA
constexpr int kMaxQ      = 64;
constexpr int kMaxRows   = kMaxQ * 8;

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
    int             n_heads, n_kv_heads, gqa, n_q, n_new, kv_bound, n_chunks;
    uint8_t *       score;
    uint8_t *       row_pos;
    size_t          nb_head, nb_stream;
    float2 *        stats;     // [pair][chunk][n_q * gqa] (max, sum)
    int *           status;
};

// One 16-row operand of the queries: rows 16 * group + g and + 8 as value and remainder.  For one query (at most 8 rows)
// the remainders take rows 8 .. 15 of the same operand and `lo` is unused.
// The 64 head dimensions go to the k-steps in the order in which a lane's 16-byte loads (q8_0: 8-byte loads) of a K row
// deliver them: any order will do as long as both operands use the same one.
//   f16 : k-step c, d = 32 (c / 2) + 8t + 4 (c % 2) + {0 .. 3}         (a lane's two loads start at d = 8t and 32 + 8t)
//   q8_0: the same order, from 8 bytes at 8t of either block
__device__ __forceinline__ int step_d(int c, int t) { return 32 * (c >> 1) + 8 * t + 4 * (c & 1); }

// the f16 operands of a K row group of 8 keys: b[c][0], b[c][1] for k-step c; q8_0 bytes stay bytes (two 8-byte words)
template <bool Q8> struct KeyTile;
template <> struct KeyTile<false> { uint4 x[2]; };
template <> struct KeyTile<true>  { uint2 x[2]; uint32_t d; };

template <bool Q8>
__device__ __forceinline__ KeyTile<Q8> load_keys(const uint8_t * pair, int row, int t, bool live) {
    KeyTile<Q8> k;
    if constexpr (!Q8) {
        const uint4 * src = reinterpret_cast<const uint4 *>(pair + (size_t) row * 128) + t;
        k.x[0] = live ? __ldg(src) : make_uint4(0u, 0u, 0u, 0u);
        k.x[1] = live ? __ldg(src + 4) : make_uint4(0u, 0u, 0u, 0u);
    } else {
        const uint8_t * tile = pair + q8_tile_off(row);
#pragma unroll
        for (int b = 0; b < 2; ++b)
            k.x[b] = live ? __ldg(reinterpret_cast<const uint2 *>(tile + q8_byte_off(row, 32 * b + 8 * t))) : make_uint2(0u, 0u);
        k.d = live ? __ldg(reinterpret_cast<const uint32_t *>(tile + kQ8KScaleOff + q8_scale_off(row, 0))) : 0u;
    }
    return k;
}

// scores of 16 rows x 8 keys.  One query: sc[0], sc[1] are row g, keys 2t and 2t + 1 (value and remainder added);
// otherwise sc[2], sc[3] are row g + 8.
template <bool Q8, bool kOne>
__device__ __forceinline__ void score_tile(float (&sc)[4], const uint32_t (&hi)[4][4], const uint32_t (&lo)[4][4], const float (&bias)[2][2],
                                           const KeyTile<Q8> & k, int lane) {
    if constexpr (!Q8) {
        sc[0] = sc[1] = sc[2] = sc[3] = 0.0f;
        const uint32_t b[4][2] = {{k.x[0].x, k.x[0].y}, {k.x[0].z, k.x[0].w}, {k.x[1].x, k.x[1].y}, {k.x[1].z, k.x[1].w}};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            mma_16816(sc, hi[c], b[c][0], b[c][1]);
            if (!kOne) mma_16816(sc, lo[c], b[c][0], b[c][1]);
        }
        if (kOne) { sc[0] += sc[2]; sc[1] += sc[3]; }
    } else {
        // keys 2t and 2t + 1 of this tile: their scales are with the lanes that hold those keys' bytes (lane = 4 * key)
        const uint32_t d0 = __shfl_sync(0xffffffffu, k.d, 8 * (lane & 3)), d1 = __shfl_sync(0xffffffffu, k.d, 8 * (lane & 3) + 4);
        float part[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            part[b][0] = part[b][1] = -bias[0][b];
            part[b][2] = part[b][3] = kOne ? 0.0f : -bias[1][b];
            const uint32_t x0 = u8_pair_to_half2(k.x[b].x, 0x4140), x1 = u8_pair_to_half2(k.x[b].x, 0x4342);
            const uint32_t y0 = u8_pair_to_half2(k.x[b].y, 0x4140), y1 = u8_pair_to_half2(k.x[b].y, 0x4342);
            mma_16816(part[b], hi[2 * b], x0, x1);
            mma_16816(part[b], hi[2 * b + 1], y0, y1);
            if (!kOne) {
                mma_16816(part[b], lo[2 * b], x0, x1);
                mma_16816(part[b], lo[2 * b + 1], y0, y1);
            } else {
                part[b][0] += part[b][2];
                part[b][1] += part[b][3];
            }
        }
        sc[0] = (part[0][0] * half_lo(d0) + part[1][0] * half_hi(d0)) * kTwo24;
        sc[1] = (part[0][1] * half_lo(d1) + part[1][1] * half_hi(d1)) * kTwo24;
        if (!kOne) {
            sc[2] = (part[0][2] * half_lo(d0) + part[1][2] * half_hi(d0)) * kTwo24;
            sc[3] = (part[0][3] * half_lo(d1) + part[1][3] * half_hi(d1)) * kTwo24;
        }
    }
}

// One row's 16 values of this lane, rotated and scaled, as value and remainder.
__device__ __forceinline__ void load_query(const ObserveParams & p, int stream, int kvh, int row, bool live, int t, float (&hi)[4][4], float (&lo)[4][4]) {
    const int     i = live ? row / p.gqa : 0, head = kvh * p.gqa + (live ? row - i * p.gqa : 0);
    const float * src = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) i * p.q_nb_tok + (size_t) head * p.q_nb_head);
    float x[4][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float2 a = *reinterpret_cast<const float2 *>(src + step_d(c, t)), b = *reinterpret_cast<const float2 *>(src + step_d(c, t) + 2);
        x[c][0] = a.x; x[c][1] = a.y; x[c][2] = b.x; x[c][3] = b.y;
    }
    if (p.rope != nullptr) {  // k-steps c and c + 2 hold each other's partners (d and d + 32)
        const float2 * tb = p.rope + (size_t) stream * (kHeadDim / 2);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 r = tb[step_d(c, t) + e];
                const float  x0 = x[c][e], x1 = x[c + 2][e];
                x[c][e]     = __fsub_rn(__fmul_rn(x0, r.x), __fmul_rn(x1, r.y));
                x[c + 2][e] = __fadd_rn(__fmul_rn(x0, r.y), __fmul_rn(x1, r.x));
            }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) split_hi_lo(live ? x[c][e] * p.scale_log2 : 0.0f, hi[c][e], lo[c][e]);
}

// the operands of rows 16 * group + g (and + 8), and what the +128 of the K bytes adds to their scores
template <bool Q8, bool kOne>
__device__ __forceinline__ void load_group(const ObserveParams & p, int stream, int kvh, int group, int rows, int lane, uint32_t (&hi)[4][4],
                                           uint32_t (&lo)[4][4], float (&bias)[2][2]) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < (kOne ? 1 : 2); ++h) {
        const int row = 16 * group + g + 8 * h;
        float     xh[4][4], xl[4][4];
        load_query(p, stream, kvh, row, row < rows, t, xh, xl);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            hi[c][h]     = pack_half2(xh[c][0], xh[c][1]);
            hi[c][h + 2] = pack_half2(xh[c][2], xh[c][3]);
            if (kOne) {
                hi[c][1] = pack_half2(xl[c][0], xl[c][1]);
                hi[c][3] = pack_half2(xl[c][2], xl[c][3]);
            } else {
                lo[c][h]     = pack_half2(xl[c][0], xl[c][1]);
                lo[c][h + 2] = pack_half2(xl[c][2], xl[c][3]);
            }
        }
        if constexpr (Q8) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float sum = 0.0f;
#pragma unroll
                for (int c = 2 * b; c < 2 * b + 2; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += xh[c][e] + xl[c][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                bias[h][b] = sum * (128.0f * kTwoM24);
            }
        }
    }
}

// kWeights = false: the (max, sum) of every row over the CTA's keys.  kWeights = true: the weights' sums over the rows.
template <bool Q8, bool kOne, bool kWeights>
__global__ void __launch_bounds__(kThreads, kOne ? 2 : 1) observe_kernel(const ObserveParams p) {
    __shared__ float2 row_stat[kMaxRows];           // kWeights: (max, 1 / sum) of every row of the pair
    __shared__ float2 warp_stat[kWarps][kMaxRows];  // otherwise: (max, sum) of every row over a warp's keys
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int chunk = blockIdx.x, kvh = blockIdx.y % p.n_kv_heads, stream = blockIdx.y / p.n_kv_heads;
    const int rows = p.n_q * p.gqa;
    pdl_wait();
    pdl_launch_dependents();
    const int len = p.kv_len[stream];
    if (len > p.kv_bound) {  // longer than the call said: nothing of it is touched
        if (tid == 0 && kvh == 0 && chunk == 0) atomicOr(p.status, kStatusBadState);
        return;
    }
    const int first = chunk * kChunk + warp * kWarpKeys;
    if (chunk * kChunk >= len) return;
    const float2 * all = p.stats + (size_t) blockIdx.y * p.n_chunks * rows;
    if (kWeights) {
        const int n = (len + kChunk - 1) / kChunk;
        for (int r = tid; r < rows; r += kThreads) {
            if (p.lse != nullptr) {
                // kept as the scores are, in units of log2, in two parts: one would lose 2^-24 of its size
                const float x = p.lse[(size_t) stream * p.n_heads + kvh * p.gqa + r], hi = x * 1.4426950408889634f;
                const float rest = fmaf(x, 1.4426950408889634f, -hi) + x * 1.9259629911266175e-8f;
                row_stat[r] = make_float2(hi, ex2_approx(-rest));
                if (isinf(hi)) row_stat[r].y = 1.0f;
                continue;
            }
            float M = -INFINITY, L = 0.0f;
            for (int c = 0; c < n; ++c) {
                const float2 x  = __ldcg(all + (size_t) c * rows + r);
                const float  mn = fmaxf(M, x.x);
                if (x.x == -INFINITY && x.y == 0.0f) continue;
                L = L * exp2f(M - mn) + x.y * exp2f(x.x - mn);
                M = mn;
            }
            row_stat[r] = L == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(M, 1.0f / L);  // a row that sees nothing adds nothing
        }
        __syncthreads();
    }
    KeyTile<Q8> keys[kWarpKeys / 8];
    const uint8_t * pair = p.k + (size_t) stream * p.k_nb_stream + (size_t) kvh * p.k_nb_head;
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n) keys[n] = load_keys<Q8>(pair, first + 8 * n + g, t, first + 8 * n + g < len);
    float colsum[kWarpKeys / 8][2];
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n) colsum[n][0] = colsum[n][1] = 0.0f;
    if (first < len) {
        for (int group = 0; 16 * group < rows; ++group) {
            uint32_t hi[4][4], lo[4][4];
            float    bias[2][2];
            load_group<Q8, kOne>(p, stream, kvh, group, rows, lane, hi, lo, bias);
            int    last[2];  // last key that rows g and g + 8 see
            float2 st[2];
            float  m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = 16 * group + g + 8 * h;
                last[h] = row < rows && !(kOne && h) ? len - p.n_q + row / p.gqa : -1;
                if (kWeights) st[h] = row < rows ? row_stat[row] : make_float2(0.0f, 0.0f);
            }
            float sc[kWarpKeys / 8][4];
#pragma unroll
            for (int n = 0; n < kWarpKeys / 8; ++n) {
                score_tile<Q8, kOne>(sc[n], hi, lo, bias, keys[n], lane);
                const int key = first + 8 * n + 2 * t;
#pragma unroll
                for (int h = 0; h < (kOne ? 1 : 2); ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (key + e > last[h]) sc[n][2 * h + e] = -INFINITY;
                        if (kWeights) colsum[n][e] += ex2_approx(sc[n][2 * h + e] - st[h].x) * st[h].y;
                        else          m[h] = fmaxf(m[h], sc[n][2 * h + e]);
                    }
            }
            if (!kWeights) {
#pragma unroll
                for (int h = 0; h < (kOne ? 1 : 2); ++h) {
                    m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
                    m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
                    const float ref = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
                    for (int n = 0; n < kWarpKeys / 8; ++n) l[h] += ex2_approx(sc[n][2 * h] - ref) + ex2_approx(sc[n][2 * h + 1] - ref);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                    const int row = 16 * group + g + 8 * h;
                    if (t == 0 && row < rows) warp_stat[warp][row] = make_float2(m[h], l[h]);
                }
            }
        }
    } else if (!kWeights) {
        for (int r = lane; r < rows; r += 32) warp_stat[warp][r] = make_float2(-INFINITY, 0.0f);
    }
    if (!kWeights) {
        __syncthreads();
        for (int r = tid; r < rows; r += kThreads) {
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, warp_stat[w][r].x);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 x = warp_stat[w][r];
                L += x.x == -INFINITY ? x.y : x.y * exp2f(x.x - M);
            }
            p.stats[((size_t) blockIdx.y * p.n_chunks + chunk) * rows + r] = make_float2(M, L);
        }
        return;
    }
    float *   score   = reinterpret_cast<float *>(p.score + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head);
    int32_t * row_pos = p.row_pos ? reinterpret_cast<int32_t *>(p.row_pos + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head) : nullptr;
    const int base = (p.n_seen ? p.n_seen[stream] : len) - len;
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float w = colsum[n][e];
            w += __shfl_xor_sync(0xffffffffu, w, 4);
            w += __shfl_xor_sync(0xffffffffu, w, 8);
            w += __shfl_xor_sync(0xffffffffu, w, 16);
            const int key = first + 8 * n + 2 * t + e;
            if (g == n && key < len) {  // eight row groups of lanes hold the same sum: each writes one tile
                const bool fresh = key >= len - p.n_new;
                score[key] = fresh ? w : fmaf(p.decay, score[key], w);
                if (fresh && row_pos != nullptr) row_pos[key] = base + key;
            }
        }
}

int check_observe(const vox_engine * e, const vox_kv_observe_args * a) {
    VOX_REQUIRE(e && a && a->cache && a->q && a->score && a->kv_len, VOX_ATTN_INVALID_ARGUMENT, "vox_kv_observe: null argument");
    const vox_kv_cache * c = a->cache;
    VOX_REQUIRE(c->e == e, VOX_ATTN_INVALID_ARGUMENT, "cache belongs to another engine");
    VOX_REQUIRE(a->layer >= 0 && a->layer < c->cfg.n_layers, VOX_ATTN_INVALID_ARGUMENT, "layer %d out of range", a->layer);
    VOX_REQUIRE(a->n_streams > 0 && a->n_streams <= c->cfg.n_streams, VOX_ATTN_INVALID_ARGUMENT, "n_streams %d out of range (cache holds %d)",
                a->n_streams, c->cfg.n_streams);
    VOX_REQUIRE(a->n_heads > 0 && a->n_heads % c->cfg.n_kv_heads == 0, VOX_ATTN_INVALID_ARGUMENT, "n_heads %d is not a multiple of n_kv_heads %d",
                a->n_heads, c->cfg.n_kv_heads);
    VOX_REQUIRE(a->n_heads / c->cfg.n_kv_heads <= 8, VOX_ATTN_UNSUPPORTED, "GQA ratio above 8 is not supported");
    VOX_REQUIRE(a->n_q >= 1, VOX_ATTN_INVALID_ARGUMENT, "n_q %d must be positive", a->n_q);
    VOX_REQUIRE(a->n_q <= kMaxQ, VOX_ATTN_UNSUPPORTED, "n_q %d: at most %d queries look back at once", a->n_q, kMaxQ);
    VOX_REQUIRE(a->n_q == 1 || (a->lse == nullptr && a->rope_table == nullptr), VOX_ATTN_UNSUPPORTED, "lse and rope_table are taken with n_q == 1 only");
    VOX_REQUIRE(a->kv_bound >= 0 && a->kv_bound <= c->cfg.max_len, VOX_ATTN_INVALID_ARGUMENT, "kv_bound %d exceeds the cache capacity %d",
                a->kv_bound, c->cfg.max_len);
    VOX_REQUIRE(a->n_new >= 0, VOX_ATTN_INVALID_ARGUMENT, "n_new %d must not be negative", a->n_new);
    VOX_REQUIRE((reinterpret_cast<uintptr_t>(a->q) & 7) == 0 && a->q_nb_head % 8 == 0 && a->q_nb_tok % 8 == 0 && a->q_nb_stream % 8 == 0,
                VOX_ATTN_INVALID_ARGUMENT, "q rows must be 8-byte aligned");
    VOX_REQUIRE((reinterpret_cast<uintptr_t>(a->rope_table) & 7) == 0, VOX_ATTN_INVALID_ARGUMENT, "rope_table must be 8-byte aligned");
    VOX_REQUIRE(((reinterpret_cast<uintptr_t>(a->score) | reinterpret_cast<uintptr_t>(a->row_pos) | reinterpret_cast<uintptr_t>(a->lse)) & 3) == 0 &&
                    a->nb_head % 4 == 0 && a->nb_stream % 4 == 0,
                VOX_ATTN_INVALID_ARGUMENT, "score, row_pos and lse must be 4-byte aligned");
    VOX_REQUIRE((long long) a->n_streams * c->cfg.n_kv_heads <= 65535, VOX_ATTN_UNSUPPORTED, "more than 65535 (stream, kv head) pairs in one call");
    return VOX_ATTN_OK;
}

template <bool Q8, bool kOne>
int launch_observe(vox_engine * e, const ObserveParams & p, dim3 grid, cudaStream_t st) {
    if (p.lse == nullptr) {
        launch_pdl(observe_kernel<Q8, kOne, false>, grid, dim3(kThreads), 0, st, p);
        const int rc = check_launch(e, "observe_kernel<stats>");
        if (rc != VOX_ATTN_OK) return rc;
    }
    launch_pdl(observe_kernel<Q8, kOne, true>, grid, dim3(kThreads), 0, st, p);
    return check_launch(e, "observe_kernel<weights>");
}

}  // namespace

extern "C" {

size_t vox_kv_observe_workspace_bytes(const vox_kv_observe_args * a) {
    if (a == nullptr || a->cache == nullptr || a->n_streams <= 0 || a->n_heads <= 0 || a->n_q <= 0 || a->kv_bound < 0 || a->lse != nullptr) return 0;
    const size_t chunks = ((size_t) a->kv_bound + kChunk - 1) / kChunk;
    return (size_t) a->n_streams * a->n_heads * a->n_q * chunks * sizeof(float2);
}

int vox_kv_observe(vox_engine * e, const vox_kv_observe_args * a, void * workspace, size_t workspace_bytes, void * stream) {
    const int rc = check_observe(e, a);
    if (rc != VOX_ATTN_OK) return rc;
    int current = -1;
    VOX_CUDA_TRY(cudaGetDevice(&current));
    VOX_REQUIRE(current == e->device, VOX_ATTN_INVALID_ARGUMENT, "the engine's device %d must be the current device (current is %d)", e->device, current);
    const size_t need = vox_kv_observe_workspace_bytes(a);
    VOX_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
                VOX_ATTN_WORKSPACE_TOO_SMALL, "vox_kv_observe needs %zu workspace bytes (16-byte aligned), got %zu", need, workspace_bytes);
    const vox_kv_cache * c = a->cache;
    const bool           q8 = c->cfg.type == VOX_TYPE_Q8_0;
    ObserveParams        p;
    p.k = c->k_data + (size_t) a->layer * c->nb_layer;
    p.k_nb_head = c->nb_head; p.k_nb_stream = c->nb_stream;
    p.kv_len = a->kv_len; p.n_seen = a->n_seen;
    p.q = reinterpret_cast<const uint8_t *>(a->q);
    p.q_nb_head = a->q_nb_head; p.q_nb_tok = a->q_nb_tok; p.q_nb_stream = a->q_nb_stream;
    p.rope = reinterpret_cast<const float2 *>(a->rope_table); p.lse = a->lse;
    p.scale_log2 = a->scale * 1.4426950408889634f; p.decay = a->decay;
    p.n_heads = a->n_heads; p.n_kv_heads = c->cfg.n_kv_heads; p.gqa = a->n_heads / c->cfg.n_kv_heads;
    p.n_q = a->n_q; p.n_new = a->n_new; p.kv_bound = a->kv_bound; p.n_chunks = (std::max(a->kv_bound, 1) + kChunk - 1) / kChunk;
    p.score = reinterpret_cast<uint8_t *>(a->score); p.row_pos = reinterpret_cast<uint8_t *>(a->row_pos);
    p.nb_head = a->nb_head; p.nb_stream = a->nb_stream;
    p.stats = static_cast<float2 *>(workspace);
    p.status = e->status_dev;
    const dim3   grid((unsigned) p.n_chunks, (unsigned) (a->n_streams * p.n_kv_heads));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->n_q == 1) return q8 ? launch_observe<true, true>(e, p, grid, st) : launch_observe<false, true>(e, p, grid, st);
    return q8 ? launch_observe<true, false>(e, p, grid, st) : launch_observe<false, false>(e, p, grid, st);
}

}  // extern "C"
