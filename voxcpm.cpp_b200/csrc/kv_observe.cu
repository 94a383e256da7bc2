// The attention weight that every cache row receives from the query of a step (vox_kv_observe with n_q == 1).
//
//   score[j] = (j new ? 0 : decay * score[j]) + sum over heads of 2^(s[head][j] - lse[head]),   s = scale * log2 e * q.k
//
// V plays no part, so a call reads K (128 or 68 bytes a row) and 8 bytes of score: bound by HBM.  A CTA takes 512 keys of a
// (stream, kv head), a warp 64 of them, from global memory straight into the operands of the products (a lane's 16-byte
// loads; nothing is shared between warps, so nothing passes through shared memory).  The softmax's (max, sum) are
//   given:    the log-sum-exp is an input; every CTA for itself;
//   cluster:  up to 24576 keys: the CTAs of a pair are a cluster and exchange (max, sum) through distributed shared memory
//             while the scores wait in registers and shared memory: K is read once, in one launch;
//   two:      longer streams: a launch that finds the (max, sum) of every CTA's keys, and one that joins them.
// 256 streams of 4096 f16 rows, given the log-sum-exp: 32.5 us = 5.5 TB/s, 84 % of the copy bandwidth; without it 53.4 us (a CTA
// waits for its cluster with its loads done); 64 streams 12.7 / 15.9 us.  Four streams of 300 rows: 4.7 us, the latency of a launch.
// q8_0 rows: 34.0 us at 256 x 4096, 2.9 TB/s.  HBM is a third busy (f16: 63 %), issue slots 54 % (f16: 32 %): per byte there are twice
// the instructions, the conversion of every byte among them, and with half the bytes in a lane's registers half of them in flight.
// (For smaller pieces and more CTAs of fewer registers: 32 keys of a warp 42 - 53 us, three CTAs per SM 43 us, against 40.4 us before a
// CTA took several chunks.)
#include "kv_observe.cuh"
#include "row_lists.h"

using namespace vox;

namespace {

constexpr int kWarps     = 8;
constexpr int kThreads   = kWarps * 32;
constexpr int kWarpKeys  = 64;                  // keys a warp keeps as operands
constexpr int kChunk     = kWarps * kWarpKeys;  // keys of a CTA
constexpr int kMaxGroup  = 8;                   // query heads of a kv head
constexpr int kFewRows    = 96;                  // query rows of a kv head up to which a window is taken here
constexpr int kMaxCluster = 8;
constexpr int kMaxRun     = 6;                   // chunks of a CTA of a cluster: the scores of two CTAs fit an SM

enum { kGiven, kCluster, kFind, kJoin };        // which launch (see above); kFind and kJoin are the two

// The query rows of the group (at most 8) as value and remainder: the values are rows 0 .. 7 of the products' A operand, the
// remainders rows 8 .. 15.
// The 64 head dimensions go to the k-steps in the order in which a lane's 16-byte loads (q8_0: 8-byte loads) of a K row
// deliver them: any order will do as long as both operands use the same one.
//   f16 : k-step c, d = 32 (c / 2) + 8t + 4 (c % 2) + {0 .. 3}         (a lane's two loads start at d = 8t and 32 + 8t)
//   q8_0: the same order, from 8 bytes at 8t of either block
__device__ __forceinline__ int step_d(int c, int t) { return 32 * (c >> 1) + 8 * t + 4 * (c & 1); }

// the f16 operands of a K row group of 8 keys: b[c][0], b[c][1] for k-step c; q8_0 bytes stay bytes (two 8-byte words)
template <bool Q8> struct KeyTile;
template <> struct KeyTile<false> { uint4 x[2]; };
template <> struct KeyTile<true>  { uint2 x[2]; uint32_t d; };

// Ordinary loads: the rows are read-only to this kernel, but its CTAs may be on the SMs while the launch in front still appends some
// (they wait for it before they read), and the non-coherent path asks for memory that nobody writes while the kernel lives.  q8_0 from L2,
// f16 through L1: the other way round the compiler orders them worse (a window of 4 queries over 128 streams of 4096 q8_0 rows 97
// against 86 us, a step over 256 f16 streams 32.5 against 32.2 us).
template <bool Q8>
__device__ __forceinline__ KeyTile<Q8> load_keys(const uint8_t * pair, int row, int t, bool live) {
    KeyTile<Q8> k;
    if constexpr (!Q8) {
        const uint4 * src = reinterpret_cast<const uint4 *>(pair + (size_t) row * 128) + t;
        k.x[0] = live ? *src : make_uint4(0u, 0u, 0u, 0u);
        k.x[1] = live ? src[4] : make_uint4(0u, 0u, 0u, 0u);
    } else {
        const uint8_t * tile = pair + q8_tile_off(row);
#pragma unroll
        for (int b = 0; b < 2; ++b)
            k.x[b] = live ? __ldcg(reinterpret_cast<const uint2 *>(tile + q8_byte_off(row, 32 * b + 8 * t))) : make_uint2(0u, 0u);
        k.d = live ? __ldcg(reinterpret_cast<const uint32_t *>(tile + kQ8KScaleOff + q8_scale_off(row, 0))) : 0u;
    }
    return k;
}

// scores of 8 rows x 8 keys: sc[0], sc[1] are row g, keys 2t and 2t + 1
template <bool Q8>
__device__ __forceinline__ void score_tile(float (&sc)[2], const uint32_t (&q)[4][4], const KeyTile<Q8> & k, int lane) {
    if constexpr (!Q8) {
        float          x[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t b[4][2] = {{k.x[0].x, k.x[0].y}, {k.x[0].z, k.x[0].w}, {k.x[1].x, k.x[1].y}, {k.x[1].z, k.x[1].w}};
#pragma unroll
        for (int c = 0; c < 4; ++c) mma_16816(x, q[c], b[c][0], b[c][1]);
        sc[0] = x[0] + x[2];
        sc[1] = x[1] + x[3];
    } else {
        // keys 2t and 2t + 1 of this tile: their scales are with the lanes that hold those keys' bytes (lane = 4 * key)
        const uint32_t d0 = __shfl_sync(0xffffffffu, k.d, 8 * (lane & 3)), d1 = __shfl_sync(0xffffffffu, k.d, 8 * (lane & 3) + 4);
        float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // one accumulator per 32-value block
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            mma_16816(x[b], q[2 * b], s8_pair_to_half2(k.x[b].x, 0x4140), s8_pair_to_half2(k.x[b].x, 0x4342));
            mma_16816(x[b], q[2 * b + 1], s8_pair_to_half2(k.x[b].y, 0x4140), s8_pair_to_half2(k.x[b].y, 0x4342));
        }
        sc[0] = (x[0][0] + x[0][2]) * half_lo(d0) + (x[1][0] + x[1][2]) * half_hi(d0);
        sc[1] = (x[0][1] + x[0][3]) * half_lo(d1) + (x[1][1] + x[1][3]) * half_hi(d1);
    }
}

// the operand, from the query rows rotated and scaled
__device__ __forceinline__ void load_query(const ObserveParams & p, int stream, int kvh, int lane, uint32_t (&op)[4][4]) {
    const int     g = lane >> 2, t = lane & 3;
    const bool    live = g < p.gqa;
    const float * src = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) (kvh * p.gqa + (live ? g : 0)) * p.q_nb_head);
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
    for (int c = 0; c < 4; ++c) {
        float h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_hi_lo(live ? x[c][e] * p.scale_log2 : 0.0f, h[e], l[e]);
        op[c][0] = pack_half2(h[0], h[1]);
        op[c][1] = pack_half2(l[0], l[1]);
        op[c][2] = pack_half2(h[2], h[3]);
        op[c][3] = pack_half2(l[2], l[3]);
    }
}

// two parts' (max, sum) as one; (-inf, 0) is a part that saw nothing, (-inf, NaN) one of NaN
__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {
    const float M = fmaxf(a.x, b.x);
    const float fa = a.x == -INFINITY ? 1.0f : exp2f(a.x - M), fb = b.x == -INFINITY ? 1.0f : exp2f(b.x - M);  // a sum of 0 or NaN stays so
    return make_float2(M, fmaf(a.y, fa, b.y * fb));
}
// as the weights take them: (max, 1 / sum); a row that saw nothing adds nothing
__device__ __forceinline__ float2 as_weights(float2 s) { return s.y == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(s.x, 1.0f / s.y); }

// A warp's 64 keys from `from` on: the weights w (of keys 8n + 2t + e, n and e the index's parts, by the row g of this lane) are added up
// over the rows and go to the scores.  Halving the keys as it halves the rows: lane (g, t) ends with keys 2t and 2t + 1 of tile g (14
// shuffles; each sum by itself in every lane would be 48).
__device__ __forceinline__ void add_weights(const ObserveParams & p, float (&w)[16], float * score, int32_t * row_pos, int stream, int len, int from,
                                            const float (&old)[2], int g, int t) {
    static_assert(kWarpKeys == 64, "a tile of keys to a row of lanes");
#pragma unroll
    for (int half = 8; half >= 2; half >>= 1) {
        const bool upper = g & (half >> 1);
#pragma unroll
        for (int n = 0; n < half; ++n) w[n] = (upper ? w[n + half] : w[n]) + __shfl_xor_sync(0xffffffffu, upper ? w[n] : w[n + half], 2 * half);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int key = from + 8 * g + 2 * t + e;
        if (key >= len) break;
        const bool fresh = key >= len - p.n_new;
        score[key] = fresh ? w[e] : fmaf(p.decay, old[e], w[e]);
        if (fresh && row_pos != nullptr) row_pos[key] = (p.n_seen ? p.n_seen[stream] : len) - len + key;
    }
}

template <bool Q8, int kMode>
__global__ void __launch_bounds__(kThreads, 2) observe_kernel(const ObserveParams p) {
    extern __shared__ float4 kept_scores[];  // kCluster: [chunk][4][thread], of all chunks of a CTA but the last
    __shared__ float2 row_stat[kMaxGroup], cta_stat[kMaxGroup], warp_stat[kWarps][kMaxGroup];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int chunk = blockIdx.x, kvh = blockIdx.y % p.n_kv_heads, stream = blockIdx.y / p.n_kv_heads;
    pdl_wait();
    pdl_launch_dependents();
    const int len = p.kv_len[stream];
    if (len > p.kv_bound || len <= 0) {  // longer than the call said: nothing of it is touched (the same for a whole cluster)
        if (len > 0 && tid == 0 && kvh == 0 && chunk == 0) atomicOr(p.status, kStatusBadState);
        return;
    }
    // A CTA takes p.run chunks one after the other; the next one's keys are asked for as soon as the products have taken this one's.
    const int chunk0 = chunk * p.run, end = min(len, (chunk0 + p.run) * kChunk);
    int       first  = chunk0 * kChunk + warp * kWarpKeys;
    if (kMode != kCluster && chunk0 * kChunk >= len) return;
    // everything the CTA reads is asked for before anything is waited for
    KeyTile<Q8>     keys[kWarpKeys / 8];
    const uint8_t * pair = p.k + (size_t) stream * p.k_nb_stream + (size_t) kvh * p.k_nb_head;
    float * const   score = reinterpret_cast<float *>(p.score + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head);
    float           old[2], next_old[2] = {0.0f, 0.0f};
    auto ask = [&](int from) {
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n) keys[n] = load_keys<Q8>(pair, from + 8 * n + g, t, from + 8 * n + g < len);
    };
    auto ask_old = [&](int from) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (from + 8 * g + 2 * t + e < len - p.n_new) next_old[e] = score[from + 8 * g + 2 * t + e];
    };
    ask(first);
    if (kMode == kGiven || kMode == kJoin || first + kChunk >= end) ask_old(first);
    if (kMode == kGiven && tid < p.gqa) {
        // kept as the scores are, in units of log2, in two parts: one would lose 2^-24 of its size
        const float x = p.lse[(size_t) stream * p.n_heads + kvh * p.gqa + tid], hi = x * 1.4426950408889634f;
        const float rest = fmaf(x, 1.4426950408889634f, -hi) + x * 1.9259629911266175e-8f;
        row_stat[tid] = make_float2(hi, isinf(hi) ? 1.0f : ex2_approx(-rest));
    }
    if (kMode == kJoin && tid < p.gqa) {
        const float2 * all = p.stats + (size_t) blockIdx.y * gridDim.x * p.gqa + tid;
        float2         s = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
        for (int c = 0; c * p.run * kChunk < len; ++c) s = join_stats(s, __ldcg(all + (size_t) c * p.gqa));
        row_stat[tid] = as_weights(s);
    }
    uint32_t q[4][4];
    load_query(p, stream, kvh, lane, q);
    if (kMode == kGiven || kMode == kJoin) __syncthreads();
    int32_t * const row_pos = p.row_pos ? reinterpret_cast<int32_t *>(p.row_pos + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head) : nullptr;
    auto write = [&](const float (&sc)[kWarpKeys / 8][2], float2 st, int from, const float (&old)[2]) {
        float w[16];
#pragma unroll
        for (int n = 0; n < 16; ++n) w[n] = ex2_approx(sc[n >> 1][n & 1] - st.x) * st.y;
        add_weights(p, w, score, row_pos, stream, len, from, old, g, t);
    };
    float m = -INFINITY, l = 0.0f;  // kFind, kCluster: of the row's keys in this lane
    for (int n_kept = 0;; first += kChunk) {
        float sc[kWarpKeys / 8][2];
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n) {
            score_tile<Q8>(sc[n], q, keys[n], lane);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (first + 8 * n + 2 * t + e >= len) sc[n][e] = -INFINITY;
        }
        old[0] = next_old[0];
        old[1] = next_old[1];
        const bool more = first + kChunk < end;
        if (more) {
            ask(first + kChunk);
            if (kMode == kGiven || kMode == kJoin || (kMode == kCluster && first + 2 * kChunk >= end)) ask_old(first + kChunk);
        }
        if (kMode == kFind || kMode == kCluster) {
            const float before = m;
#pragma unroll
            for (int n = 0; n < kWarpKeys / 8; ++n) m = fmaxf(m, fmaxf(sc[n][0], sc[n][1]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float ref = m == -INFINITY ? 0.0f : m;
            if (before != -INFINITY) l *= ex2_approx(before - ref);
#pragma unroll
            for (int n = 0; n < kWarpKeys / 8; ++n) l += ex2_approx(sc[n][0] - ref) + ex2_approx(sc[n][1] - ref);
            if (more) {
                if (kMode == kCluster) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) kept_scores[(4 * n_kept + n) * kThreads + tid] = make_float4(sc[2 * n][0], sc[2 * n][1], sc[2 * n + 1][0], sc[2 * n + 1][1]);
                    ++n_kept;
                }
                continue;
            }
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (t == 0) warp_stat[warp][g] = make_float2(m, l);
            __syncthreads();
            if (tid < p.gqa) {
                float2 s = warp_stat[0][tid];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) s = join_stats(s, warp_stat[w][tid]);
                if (kMode == kFind) p.stats[((size_t) blockIdx.y * gridDim.x + chunk) * p.gqa + tid] = s;
                else                cta_stat[tid] = s;
            }
            if (kMode == kFind) return;
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            if (tid < p.gqa) {
                const uint32_t at = smem_u32(&cta_stat[tid]);
                float2         all[kMaxCluster], s = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {  // all on their way together
                    all[r] = s;
                    if (r < (int) gridDim.x) {
                        uint32_t peer;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(r));
                        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(all[r].x), "=f"(all[r].y) : "r"(peer) : "memory");
                    }
                }
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) s = join_stats(s, all[r]);
                row_stat[tid] = as_weights(s);
            }
            __syncthreads();
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for at the end: nobody leaves while its memory is read
        }
        const float2 st = g < p.gqa ? row_stat[g] : make_float2(0.0f, 0.0f);
        if (kMode == kCluster) {  // the last chunk's scores are here; back over the others
            while (n_kept > 0) {
                --n_kept;
                ask_old(first - kChunk);
                write(sc, st, first, old);
                first -= kChunk;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float4 x = kept_scores[(4 * n_kept + n) * kThreads + tid];
                    sc[2 * n][0] = x.x; sc[2 * n][1] = x.y; sc[2 * n + 1][0] = x.z; sc[2 * n + 1][1] = x.w;
                }
                old[0] = next_old[0];
                old[1] = next_old[1];
            }
        }
        write(sc, st, first, old);
        if (!more) break;
    }
    if (kMode == kCluster) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// A window of few query rows (at most kFewRows, queries times the heads of a group): as above, with the rows in groups of eight.  A
// warp's keys stay in its registers while the groups' operands come from shared memory one after the other.  Two launches: the
// rows' (max, sum) over every CTA's keys, and the weights.  Bound by latency: a group is a chain of products, shuffles, exponentials and
// the join of its statistics, 0.3 us of it where nothing else runs, and 16 warps an SM do not hide it: 128 streams of 4096 rows, 4
// queries of 8 heads take 60 us, of which K twice from HBM or L2 would be 28, with no unit much busier than a third (issue 32 %, tensor
// 29 %, special functions 20 %, DRAM 31 %).  q8_0, whose bytes are converted for every group, 86 us: issue 47 and 39 %; the kernel
// of the weights spills 304 bytes a thread.
template <bool Q8, bool kWeights>
__global__ void __launch_bounds__(kThreads, 2) observe_rows_kernel(const ObserveParams p) {
    __shared__ uint4  q_op[kFewRows / 8][4][32];
    __shared__ float2 row_stat[kFewRows], warp_stat[kWarps][kFewRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int chunk = blockIdx.x, kvh = blockIdx.y % p.n_kv_heads, stream = blockIdx.y / p.n_kv_heads;
    const int rows = p.n_q * p.gqa, n_groups = (rows + 7) >> 3;
    // (the second launch reads one thing that the first has written, the statistics: it waits for them alone)
    if (!kWeights) {
        pdl_wait();
        pdl_launch_dependents();
    }
    const int len = p.kv_len[stream], first0 = chunk * p.run * kChunk, end = min(len, first0 + p.run * kChunk);
    if (len > p.kv_bound || first0 >= len) {
        if (kWeights) pdl_wait();  // no launch of the next call ends before the first one of this call
        else if (len > p.kv_bound && tid == 0 && kvh == 0 && chunk == 0) atomicOr(p.status, kStatusBadState);
        return;
    }
    int             first = first0 + warp * kWarpKeys;
    KeyTile<Q8>     keys[kWarpKeys / 8];
    const uint8_t * pair = p.k + (size_t) stream * p.k_nb_stream + (size_t) kvh * p.k_nb_head;
    float * const   score = reinterpret_cast<float *>(p.score + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head);
    int32_t * const row_pos = p.row_pos ? reinterpret_cast<int32_t *>(p.row_pos + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head) : nullptr;
    auto ask = [&](int from) {
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n) keys[n] = load_keys<Q8>(pair, from + 8 * n + g, t, from + 8 * n + g < len);
    };
    ask(first);
    for (int i = warp; i < n_groups; i += kWarps) {
        const int     row = 8 * i + g, at = min(row, rows - 1), q = (int) ((uint32_t) at * p.gqa_magic >> 16);
        const float * src = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) q * p.q_nb_tok +
                                                            (size_t) (kvh * p.gqa + at - q * p.gqa) * p.q_nb_head);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float2 a = *reinterpret_cast<const float2 *>(src + step_d(c, t)), b = *reinterpret_cast<const float2 *>(src + step_d(c, t) + 2);
            const float  x[4] = {a.x, a.y, b.x, b.y};
            float        h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) split_hi_lo(row < rows ? x[e] * p.scale_log2 : 0.0f, h[e], l[e]);
            q_op[i][c][lane] = make_uint4(pack_half2(h[0], h[1]), pack_half2(l[0], l[1]), pack_half2(h[2], h[3]), pack_half2(l[2], l[3]));
        }
    }
    if (kWeights) {
        pdl_wait();
        pdl_launch_dependents();
        if (tid < kFewRows) {
            const float2 * all = p.stats + (size_t) blockIdx.y * gridDim.x * rows + tid;
            float2         s = make_float2(-INFINITY, 0.0f);
            if (tid < rows)
#pragma unroll 4
                for (int c = 0; c * p.run * kChunk < len; ++c) s = join_stats(s, __ldcg(all + (size_t) c * rows));
            row_stat[tid] = as_weights(s);
        }
    } else if (t == 0) {
        for (int i = 0; i < n_groups; ++i) warp_stat[warp][8 * i + g] = make_float2(-INFINITY, 0.0f);
    }
    __syncthreads();
    for (;; first += kChunk) {
        const bool cut = first + kWarpKeys > len - p.n_q;  // keys that not every query sees, and keys past the end
        float      w[16], old[2] = {0.0f, 0.0f};
        if (kWeights) {
#pragma unroll
            for (int n = 0; n < 16; ++n) w[n] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (first + 8 * g + 2 * t + e < len - p.n_new) old[e] = score[first + 8 * g + 2 * t + e];
        }
#pragma unroll 1
        for (int i = 0; i < n_groups; ++i) {
            uint32_t q[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint4 x = q_op[i][c][lane];
                q[c][0] = x.x; q[c][1] = x.y; q[c][2] = x.z; q[c][3] = x.w;
            }
            float sc[kWarpKeys / 8][2];
#pragma unroll
            for (int n = 0; n < kWarpKeys / 8; ++n) score_tile<Q8>(sc[n], q, keys[n], lane);
            const int last = len - p.n_q + (int) ((uint32_t) (8 * i + g) * p.gqa_magic >> 16) - first - 2 * t;
            if (cut) {
#pragma unroll
                for (int n = 0; n < 16; ++n)
                    if (8 * (n >> 1) + (n & 1) > last) sc[n >> 1][n & 1] = -INFINITY;
            }
            if (kWeights) {
                const float2 st = row_stat[8 * i + g];
                if (cut) {  // (the sum of a row that does not see a key may be NaN)
#pragma unroll
                    for (int n = 0; n < 16; ++n)
                        if (8 * (n >> 1) + (n & 1) <= last) w[n] = fmaf(ex2_approx(sc[n >> 1][n & 1] - st.x), st.y, w[n]);
                } else {
#pragma unroll
                    for (int n = 0; n < 16; ++n) w[n] = fmaf(ex2_approx(sc[n >> 1][n & 1] - st.x), st.y, w[n]);
                }
            } else {
                float m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int n = 0; n < kWarpKeys / 8; ++n) m = fmaxf(m, fmaxf(sc[n][0], sc[n][1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int n = 0; n < 16; ++n) l += ex2_approx(sc[n >> 1][n & 1] - ref);
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (t == 0) warp_stat[warp][8 * i + g] = join_stats(warp_stat[warp][8 * i + g], make_float2(m, l));
            }
        }
        const bool more = first + kChunk < end;
        if (more) ask(first + kChunk);
        if (kWeights) add_weights(p, w, score, row_pos, stream, len, first, old, g, t);
        if (!more) break;
    }
    if (!kWeights) {
        __syncthreads();
        if (tid < rows) {
            float2 s = warp_stat[0][tid];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) s = join_stats(s, warp_stat[w][tid]);
            p.stats[((size_t) blockIdx.y * gridDim.x + chunk) * rows + tid] = s;
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
    VOX_REQUIRE(a->n_q <= kObserveMaxQ, VOX_ATTN_UNSUPPORTED, "n_q %d: at most %d queries look back at once", a->n_q, kObserveMaxQ);
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
    const size_t row_bytes = (size_t) a->kv_bound * sizeof(float);
    const RowLists lists(a->score, row_bytes, {{c->cfg.n_kv_heads, a->nb_head}, {a->n_streams, a->nb_stream}});
    VOX_REQUIRE(!lists.overlap(), VOX_ATTN_INVALID_ARGUMENT, "the scores of %d rows overlap (strides %zu, %zu bytes)", a->kv_bound, a->nb_head, a->nb_stream);
    VOX_REQUIRE(a->row_pos == nullptr || !lists.overlap_shifted(a->row_pos), VOX_ATTN_INVALID_ARGUMENT, "score and row_pos overlap");
    const RowLists positions(a->row_pos, a->row_pos ? row_bytes : 0, {{c->cfg.n_kv_heads, a->nb_head}, {a->n_streams, a->nb_stream}});
    for (const int32_t * in : {a->kv_len, a->n_seen})
        VOX_REQUIRE(!lists.meets(in, a->n_streams * sizeof(int32_t)) && !positions.meets(in, a->n_streams * sizeof(int32_t)), VOX_ATTN_INVALID_ARGUMENT,
                    "score and row_pos must not overlap kv_len or n_seen");
    VOX_REQUIRE(!lists.meets(a->lse, (size_t) a->n_streams * a->n_heads * sizeof(float)) &&
                    !positions.meets(a->lse, (size_t) a->n_streams * a->n_heads * sizeof(float)),
                VOX_ATTN_INVALID_ARGUMENT, "score and row_pos must not overlap lse");
    VOX_REQUIRE((long long) a->n_streams * c->cfg.n_kv_heads <= 65535, VOX_ATTN_UNSUPPORTED, "more than 65535 (stream, kv head) pairs in one call");
    return VOX_ATTN_OK;
}

int chunks_of(int kv_bound) { return (std::max(kv_bound, 1) + kChunk - 1) / kChunk; }
// Windows of few query rows are this file's: up to 40 rows, or 96 where there is work for more than two rounds of CTAs (the kernel for
// the others takes a pair or a part of one per SM, with nothing beside it to hide its latency).  24 / 48 / 64 / 96 / 128 rows, f16:
// 4 streams of 4096 rows 9.8 / 13.0 / 15.6 / 20.3 / 25.1 us against 13.9 / 13.9 / 13.9 / 14.5 / 14.5 us there; 128 streams of
// 2048 rows 35 / 49 / 59 / 80 / 100 against 74 / 74 / 74 / 83 / 84 us.  q8_0: 11.8 / 16.8 / 19.9 / 26.2 / 32.3 against 18.6 / 18.8 /
// 18.6 / 19.3 / 19.5 us, and 46 / 66 / 79 / 108 / 135 against 113 / 114 / 114 / 125 / 126 us.
bool few_rows(const vox_kv_observe_args * a) {
    const int HK = a->cache->cfg.n_kv_heads;
    return a->n_heads / HK * a->n_q <= ((long long) chunks_of(a->kv_bound) * a->n_streams * HK > 4LL * a->cache->e->sm_count ? kFewRows : 40);
}

template <bool Q8>
int launch_rows(vox_engine * e, const ObserveParams & p, cudaStream_t st) {
    const dim3 grid((unsigned) ((p.n_chunks + p.run - 1) / p.run), (unsigned) (p.n_streams * p.n_kv_heads));
    launch_pdl(observe_rows_kernel<Q8, false>, grid, dim3(kThreads), 0, st, p);
    const int rc = check_launch(e, "observe_rows_kernel<statistics>");
    if (rc != VOX_ATTN_OK) return rc;
    launch_pdl(observe_rows_kernel<Q8, true>, grid, dim3(kThreads), 0, st, p);
    return check_launch(e, "observe_rows_kernel<weights>");
}

template <bool Q8>
int launch_observe(vox_engine * e, const ObserveParams & p, cudaStream_t st) {
    const dim3 grid((unsigned) ((p.n_chunks + p.run - 1) / p.run), (unsigned) (p.n_streams * p.n_kv_heads));
    if (p.lse == nullptr && p.n_chunks > kMaxCluster * kMaxRun) {
        launch_pdl(observe_kernel<Q8, kFind>, grid, dim3(kThreads), 0, st, p);
        const int rc = check_launch(e, "observe_kernel<statistics>");
        if (rc != VOX_ATTN_OK) return rc;
        launch_pdl(observe_kernel<Q8, kJoin>, grid, dim3(kThreads), 0, st, p);
        return check_launch(e, "observe_kernel<weights>");
    }
    if (p.lse != nullptr) {
        launch_pdl(observe_kernel<Q8, kGiven>, grid, dim3(kThreads), 0, st, p);
        return check_launch(e, "observe_kernel<given>");
    }
    const size_t   most = (size_t) (kMaxRun - 1) * kChunk * kMaxGroup * sizeof(float);
    const uint32_t bit  = 1u << (Q8 ? 11 : 10);
    if (!(e->attr_mask & bit)) {
        VOX_CUDA_TRY(cudaFuncSetAttribute(observe_kernel<Q8, kCluster>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) most));
        e->attr_mask |= bit;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(kThreads); cfg.stream = st;
    cfg.dynamicSmemBytes = (size_t) (p.run - 1) * kChunk * kMaxGroup * sizeof(float);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = grid.x; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, observe_kernel<Q8, kCluster>, p);
    return check_launch(e, "observe_kernel<cluster>");
}

}  // namespace

extern "C" {

size_t vox_kv_observe_workspace_bytes(const vox_kv_observe_args * a) {
    if (a == nullptr || a->cache == nullptr || a->n_streams <= 0 || a->n_heads <= 0 || a->n_q <= 0 || a->kv_bound < 0 || a->lse != nullptr) return 0;
    const int HK = a->cache->cfg.n_kv_heads;
    if (a->n_q > 1 && few_rows(a)) return (size_t) a->n_streams * a->n_heads * a->n_q * chunks_of(a->kv_bound) * sizeof(float2);
    if (a->n_q > 1) return observe_window_bytes(a->n_streams, HK, a->n_heads / HK * a->n_q, a->kv_bound);
    const int chunks = chunks_of(a->kv_bound);
    return chunks <= kMaxCluster * kMaxRun ? 0 : (size_t) a->n_streams * a->n_heads * chunks * sizeof(float2);
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
    p.gqa_magic = 65536u / (uint32_t) p.gqa + 1u;
    p.n_streams = a->n_streams; p.layer = a->layer;
    p.n_q = a->n_q; p.n_new = a->n_new; p.kv_bound = a->kv_bound; p.n_chunks = chunks_of(a->kv_bound);
    p.score = reinterpret_cast<uint8_t *>(a->score); p.row_pos = reinterpret_cast<uint8_t *>(a->row_pos);
    p.nb_head = a->nb_head; p.nb_stream = a->nb_stream;
    // Chunks of a CTA, 256 streams of 4096 rows.  Given the log-sum-exp: several while every SM is left two rounds of its two CTAs (1 / 2
    // / 4 / 8 chunks 41.5 / 35.6 / 33.9 / 36.2 us).  In a cluster a CTA waits for the others once, whatever it holds: as many as make
    // one round of all CTAs, if they fit (1 / 4 / 6 chunks 86.7 / 53.4 / 53.4 us; 64 streams 1 / 4 chunks 23.8 / 15.9 us), and what
    // eight CTAs need.
    const long long chunks  = (long long) p.n_chunks * a->n_streams * p.n_kv_heads, slots = 2LL * e->sm_count;
    const bool      cluster = p.n_q == 1 && p.lse == nullptr && p.n_chunks <= kMaxCluster * kMaxRun;
    const int       most    = cluster ? std::max((p.n_chunks + kMaxCluster - 1) / kMaxCluster, (int) std::min<long long>(kMaxRun, (chunks + slots - 1) / slots))
                                      : (int) std::max(1LL, std::min<long long>(8, chunks / (2 * slots)));
    const int       ctas    = (p.n_chunks + most - 1) / most;
    p.run = (p.n_chunks + ctas - 1) / ctas;
    p.stats = static_cast<float2 *>(workspace);
    p.status = e->status_dev;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->n_q > 1 && few_rows(a)) return q8 ? launch_rows<true>(e, p, st) : launch_rows<false>(e, p, st);
    if (a->n_q > 1) return launch_observe_window(e, c, p, st);
    return q8 ? launch_observe<true>(e, p, st) : launch_observe<false>(e, p, st);
}

}  // extern "C"
