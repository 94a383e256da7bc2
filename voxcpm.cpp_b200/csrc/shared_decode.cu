// Decode attention over rows that many streams share (a voice prompt), computed once for all of them.
//
//   out[s] = softmax over (prefix rows of s, own rows of s) of scale * q[s].k, times v
//
// A stream's softmax splits into the part over its own rows and the part over its prefix; each part is a (max, sum,
// unnormalised output), and two parts join as two chunks of split-KV decode do.  The own rows are the decode kernel's work
// (decode_attn.cu, bound by HBM): it runs first and leaves its result in dst with the (max, sum) of every row beside it.
// The prefix rows are this file's: the queries of all streams that share a prefix are the rows of one matrix product
// against it, so the prefix leaves HBM once for all of them instead of once per stream.  Its kernel starts as soon as the
// decode kernel's CTAs have started, runs beside them (on small calls) or in the room they leave as they finish (on large
// ones; decode CTAs end up to 20 us apart on 256 ragged streams), and waits for the decode kernel only to join the results.
//
// Streams are packed into row tiles of up to 128 rows (128 / gqa streams of one prefix, gqa rows each).  A (row tile, kv
// head) is the work of one thread-block cluster of up to eight CTAs, which share out the prefix's 128-key tiles; their
// partial results meet through distributed shared memory, every CTA joining a share of the rows.  Nothing goes through
// global memory but the inputs and the result.
// 256 streams under two prompts of 4096 rows with up to 2048 rows of their own: 49 us, of which the own rows (151 MB) are the bound: 3.1
// TB/s; each stream reading its prefix would be 690 MB.  32 streams under four of 700: 11.4 us, latency.
// (Built first: the prefix kernel in front, partials in global memory, folded by the decode kernel as it wrote every result: 61.7 and
// 16.9 us; the folds' round trips to L2 and the decode kernel's late start were a third of it.)
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <exception>
#include <new>
#include <vector>

using namespace vox;

namespace {
constexpr int kRows = 128;       // rows of a full row tile
constexpr int kHalfRows = 64;    // of the largest one for the mma.sync kernel
constexpr int kArrangements = 4; // row tiles of 128, 64, 32 and 16 rows
constexpr int kJoin = 128;       // threads that join results
constexpr int kKeys = 128;       // keys of a tile
constexpr int kMaxCluster = 8;
}

// The streams of a call, arranged by prefix into row tiles of 128 >> k rows, k = 0 .. 3: few streams are cut into small tiles,
// whose products take less time.  Host copy and device arrays (one allocation), per k:
//   tiles [max_tiles][2] = prefix, streams (0: not in use);  members [max_tiles][rows / gqa]: their streams
struct vox_prefix_plan {
    vox_engine *         e = nullptr;
    int                  n_streams = 0, n_prefixes = 0, gqa = 0;
    int                  max_tiles[kArrangements] = {}, n_tiles[kArrangements] = {};
    size_t               at[kArrangements + 1] = {};  // where an arrangement starts
    bool                 full = false;  // the tiles of 128 rows are more than half full on average
    int                  first = 0;     // the lowest prefix in use
    std::vector<int32_t> host, next;    // next: scratch of the arrangement
    int32_t *            dev = nullptr;
    int    per_tile(int k) const { return (kRows >> k) / gqa; }
    size_t members_at(int k) const { return at[k] + (size_t) max_tiles[k] * 2; }
    size_t words() const { return at[kArrangements]; }
};

namespace {

struct SharedParams {
    const uint8_t * q;
    size_t          q_nb_head, q_nb_stream;
    const float2 *  rope;
    const int2 *    tiles;
    const int32_t * members;   // [tile][per_tile]
    const int32_t * len;       // [prefix]
    int             per_tile, n_kv_heads, n_heads, gqa, layer, max_len, cluster;
    float           scale_log2;
    const uint8_t * q8_tiles;
    size_t          q8_nb_head, q8_nb_stream;
    float *         dst;       // the own rows' results, and then the joined ones
    const float2 *  ml;        // (max, sum) of the own rows
    float *         lse;
    int *           status;
};

// The work of a CTA.  What the plan says of it is read before any wait (the plan changes only in stream order and never by a
// kernel); the length of the prefix is as old as the other inputs of the call, which were complete before the decode
// kernel in front let this one start.
struct Item {
    int             prefix, rows, kvh, rank, key0, key1;
    const int32_t * streams;
};
__device__ __forceinline__ Item load_item(const SharedParams & p) {
    Item      w;
    const int pair = (int) blockIdx.x / p.cluster, tile = pair / p.n_kv_heads;
    const int2 t = p.tiles[tile];
    w.kvh     = pair - tile * p.n_kv_heads;
    w.rank    = (int) blockIdx.x - pair * p.cluster;
    w.prefix  = t.x;
    w.rows    = t.y * p.gqa;
    w.streams = p.members + (size_t) tile * p.per_tile;
    const int given = t.y > 0 ? p.len[t.x] : 0, len = max(0, min(given, p.max_len)), n = (len + kKeys - 1) / kKeys;
    if (given > p.max_len && threadIdx.x == 0) atomicOr(p.status, kStatusBadState);
    if (len == 0) w.rows = 0;
    w.key0 = (w.rank * n / p.cluster) * kKeys;
    w.key1 = min(len, ((w.rank + 1) * n / p.cluster) * kKeys);
    return w;
}

// ---- the join.  A CTA's partial results lie in its shared memory: part[v][17] float4 (a row's 64 columns, padded by 16
// bytes against bank conflicts) and ml[v], where v = group * stride + row and a row has a result from every one of
// `groups` groups of warps.  kJoin threads take part; the others only arrive at the cluster barriers.
constexpr int kPartPitch = 17;

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 peer_ld2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_ld4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// The weight of a part with maximum m against the maximum M over all parts; a part that saw nothing (-inf) has none.  (A row of
// NaN has the maximum -inf and the sum NaN, which stays NaN.)
__device__ __forceinline__ float part_weight(float m, float M) { return m == -INFINITY ? 0.0f : ex2_approx(m - M); }

// Called by all threads of the CTA; `tid` < kJoin do the work.  joined: one more ml array of kRows entries; rows_at: where the rows
// of the tile lie in dst (stream * n_heads + head); share: memory for this CTA's share of the rows, apart from `part`.
// All that can be done before the decode kernel has ended is done before it: the parts of the CTA's warps and then of the
// cluster's CTAs are joined, every CTA taking a share of the rows, so that only one part is left to join with the own rows'.
// The loops are kept short: this code runs once per CTA, and what it costs cold is fetching its instructions (8 us of a
// call when the joins of four rows and eight CTAs were written out).
__device__ __forceinline__ void join_and_write(const SharedParams & p, const Item & w, float4 * part, float2 * ml, float2 * joined, const int * rows_at,
                                               float4 * share, int groups, int stride, bool ok, int tid) {
    const bool mine = tid < kJoin;
    __syncwarp();
    if (mine) {
        named_bar_sync(1, kJoin);
        if (!ok || w.key0 >= w.key1) {
            if (tid < w.rows) joined[tid] = make_float2(-INFINITY, 0.0f);
        } else if (groups == 1) {
            if (tid < w.rows) joined[tid] = ml[tid];
        } else {
            if (tid < w.rows) {
                float M = -INFINITY, L = 0.0f;
                for (int g = 0; g < groups; ++g) M = fmaxf(M, ml[g * stride + tid].x);
                for (int g = 0; g < groups; ++g) {
                    const float2 x = ml[g * stride + tid];
                    const float  f = part_weight(x.x, M);
                    L = fmaf(x.y, f, L);
                    ml[g * stride + tid].x = f;
                }
                joined[tid] = make_float2(M, L);
            }
            named_bar_sync(1, kJoin);
            for (int i = tid; i < w.rows * 16; i += kJoin) {
                const int row = i >> 4, c = i & 15;
                float4    a = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int g = 0; g < groups; ++g) {
                    const float4 x = part[(g * stride + row) * kPartPitch + c];
                    const float  f = ml[g * stride + row].x;
                    a = make_float4(fmaf(x.x, f, a.x), fmaf(x.y, f, a.y), fmaf(x.z, f, a.z), fmaf(x.w, f, a.w));
                }
                part[row * kPartPitch + c] = a;  // only this thread looks at column group c of this row
            }
        }
    }
    // this CTA's share of the rows: row0 .. row0 + n_rows - 1, in share[] and ml[] (row 0 first)
    const int row0 = w.rank * w.rows / p.cluster, n_rows = (w.rank + 1) * w.rows / p.cluster - row0;
    if (p.cluster > 1) {
        cluster_sync_all();
        if (mine) {
            const uint32_t joined0 = smem_u32(joined), part0 = smem_u32(part);
#pragma unroll 1
            for (int i = tid; i < n_rows * 16; i += kJoin) {
                const int row = i >> 4, c = i & 15;
                float2    m[kMaxCluster];
                float4    x[kMaxCluster];
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {  // all on their way together
                    m[r] = make_float2(-INFINITY, 0.0f);
                    x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < p.cluster) {
                        m[r] = peer_ld2(peer_addr(joined0 + (row0 + row) * 8, r));
                        x[r] = peer_ld4(peer_addr(part0 + ((row0 + row) * kPartPitch + c) * 16, r));
                    }
                }
                float  M = -INFINITY, L = 0.0f;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) M = fmaxf(M, m[r].x);
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {
                    if (m[r].x == -INFINITY && m[r].y == 0.0f) continue;  // a part without keys was never written
                    const float f = part_weight(m[r].x, M);
                    L = fmaf(m[r].y, f, L);
                    a = make_float4(fmaf(x[r].x, f, a.x), fmaf(x[r].y, f, a.y), fmaf(x[r].z, f, a.z), fmaf(x[r].w, f, a.w));
                }
                share[row * kPartPitch + c] = a;
                if (c == 0) ml[row] = make_float2(M, L);
            }
            named_bar_sync(1, kJoin);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for at the end: nobody leaves while its memory is read
    } else {
        share = part;
        ml    = joined;
        if (mine) named_bar_sync(1, kJoin);
    }
    pdl_wait();  // the decode kernel's results
    pdl_launch_dependents();
    constexpr int W = 4;  // a thread's rows in flight: a row at a time would wait for L2 once per row
#pragma unroll 1
    for (int i0 = tid; mine && i0 < n_rows * 16; i0 += W * kJoin) {
        float2 own_ml[W];
        float4 own[W];
#pragma unroll
        for (int u = 0; u < W; ++u) {
            const int i = min(i0 + u * kJoin, n_rows * 16 - 1), at = rows_at[row0 + (i >> 4)];
            own_ml[u] = __ldcg(p.ml + at);
            own[u]    = __ldcg(reinterpret_cast<const float4 *>(p.dst + (size_t) at * kHeadDim) + (i & 15));
        }
#pragma unroll
        for (int u = 0; u < W; ++u) {
            const int i = i0 + u * kJoin, row = i >> 4, c = i & 15;
            if (i >= n_rows * 16) break;
            const float2 b = ml[row];
            const float4 x = share[row * kPartPitch + c];
            const float  M = fmaxf(own_ml[u].x, b.x), fa = part_weight(own_ml[u].x, M) * own_ml[u].y, fb = part_weight(b.x, M);
            const float  L = fmaf(b.y, fb, fa), inv = L > 0.0f ? 1.0f / L : L == 0.0f ? 0.0f : L;  // NaN stays NaN
            const int    at = rows_at[row0 + row];
            // the own rows' result is normalised: its sum is taken back in
            reinterpret_cast<float4 *>(p.dst + (size_t) at * kHeadDim)[c] =
                make_float4(fmaf(own[u].x, fa, x.x * fb) * inv, fmaf(own[u].y, fa, x.y * fb) * inv, fmaf(own[u].z, fa, x.z * fb) * inv, fmaf(own[u].w, fa, x.w * fb) * inv);
            if (c == 0 && p.lse != nullptr) p.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
        }
    }
    __syncwarp();
    if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// Row tiles of 64 rows, of any fill and either cache type, on mma.sync: four warps, arranged as row groups of 16 x key groups
// (a tile of few rows has the 128 keys of a ring stage spread over the warps), and a warp that copies.
constexpr int kWarps   = 4;
constexpr int kThreads = (kWarps + 1) * 32;

template <bool Q8> struct Ring {
    static constexpr int kStages     = Q8 ? 4 : 2;  // room for two CTAs of the decode kernel on the SM
    static constexpr int kBoxBytes   = Q8 ? 9 * 1024 : 2 * kKvTile * 128;  // 64 rows of K and V
    static constexpr int kBoxTx      = Q8 ? kQ8TileBytes : kBoxBytes;
    static constexpr int kVOff       = Q8 ? kQ8VBytesOff : kKvTile * 128;
    static constexpr int kStageBytes = 2 * kBoxBytes;
    static constexpr int kSmemBytes  = kStages * kStageBytes + 1024;
    static_assert(kStages * kStageBytes >= kHalfRows * kPartPitch * 16, "the partial results take the ring's memory");
    static_assert(kStages * kStageBytes >= (kHalfRows + kHalfRows / 2) * kPartPitch * 16, "and a share of them with it");
};
constexpr float kShift = 10.0f;  // f16 caches: weights up to 2^10, so that the remainders of small ones are normal f16 numbers

// what a warp holds of its 16 rows: row g of a lane is [0], row g + 8 is [1]
struct Rows {
    uint32_t qh[4][4], ql[4][4];
    float    o[8][4], m[2], l[2];
    float    to_units[2];      // q8_0: 32 / the unit of the weights that take V's scales in (inverse_unit)
};

// One step of the online softmax: NK * 16 keys from row r0 of the 64-row box at `box`; `pos` is the first one's place, `end`
// where the keys end.
template <bool Q8, int NK>
__device__ __forceinline__ void step(Rows & x, uint32_t box, int r0, int pos, int end, int lane) {
    using R = Ring<Q8>;
    const int g = lane >> 2, t = lane & 3;
    float     sc[2 * NK][4];
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        if constexpr (!Q8) {
            const int k_row = r0 + 16 * k + ((lane >> 4) << 3) + (lane & 7), k_chk = (lane >> 3) & 1;
            float     small[2][4];  // the remainders' products apart: the accumulator truncates at the size of what it holds
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[2 * k + j][e] = small[j][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t b0, b1, b2, b3;
                ldmatrix_x4(box + k_row * 128 + (((2 * c + k_chk) ^ (k_row & 7)) << 4), b0, b1, b2, b3);
                mma_16816(sc[2 * k], x.qh[c], b0, b1);
                mma_16816(sc[2 * k + 1], x.qh[c], b2, b3);
                mma_16816(small[0], x.ql[c], b0, b1);
                mma_16816(small[1], x.ql[c], b2, b3);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[2 * k + j][e] += small[j][e];
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float     part[2][4];  // one accumulator per 32-value block
                const int row = r0 + 16 * k + 8 * j + g;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    part[b][0] = part[b][1] = part[b][2] = part[b][3] = 0.0f;
                    const uint2 raw = lds64(box + row * 64 + (((2 * b + (t >> 1)) ^ ((row >> 1) & 3)) << 4) + ((t & 1) << 3));
                    const uint32_t x0 = s8_pair_to_half2(raw.x, 0x4140), x1 = s8_pair_to_half2(raw.x, 0x4342);
                    const uint32_t y0 = s8_pair_to_half2(raw.y, 0x4140), y1 = s8_pair_to_half2(raw.y, 0x4342);
                    mma_16816(part[b], x.ql[2 * b], x0, x1);
                    mma_16816(part[b], x.ql[2 * b + 1], y0, y1);
                    mma_16816(part[b], x.qh[2 * b], x0, x1);
                    mma_16816(part[b], x.qh[2 * b + 1], y0, y1);
                }
                const uint2 ds = lds64(box + kQ8KScaleOff + (r0 + 16 * k + 8 * j + 2 * t) * 4);
                sc[2 * k + j][0] = part[0][0] * half_lo(ds.x) + part[1][0] * half_hi(ds.x);
                sc[2 * k + j][1] = part[0][1] * half_lo(ds.y) + part[1][1] * half_hi(ds.y);
                sc[2 * k + j][2] = part[0][2] * half_lo(ds.x) + part[1][2] * half_hi(ds.x);
                sc[2 * k + j][3] = part[0][3] * half_lo(ds.y) + part[1][3] * half_hi(ds.y);
            }
        }
    }
    const bool edge = pos + 16 * NK > end;
    if (edge) {
#pragma unroll
        for (int j = 0; j < 2 * NK; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (pos + 8 * j + 2 * t + (e & 1) >= end) sc[j][e] = -INFINITY;
    }
    float alpha[2], m_exp[2], rise[2];
    bool  first[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2 * NK; ++j) top = max3(top, sc[j][2 * h], sc[j][2 * h + 1]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(x.m[h], top);
        first[h] = x.m[h] == -INFINITY;
        rise[h]  = m_new == -INFINITY ? 0.0f : fmaxf(m_new - x.m[h], 0.0f);
        alpha[h] = m_new == -INFINITY ? 1.0f : ex2_approx(x.m[h] - m_new);
        m_exp[h] = (m_new == -INFINITY ? 0.0f : m_new) - (Q8 ? 0.0f : kShift);
        x.m[h]   = m_new;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
        if constexpr (!Q8) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                x.o[n][0] *= alpha[0]; x.o[n][1] *= alpha[0]; x.o[n][2] *= alpha[1]; x.o[n][3] *= alpha[1];
            }
        } else {  // the accumulators' unit instead
            x.to_units[0] *= ex2_approx(rise[0]);
            x.to_units[1] *= ex2_approx(rise[1]);
        }
        x.l[0] *= alpha[0];
        x.l[1] *= alpha[1];
    }
    if constexpr (Q8) {
        // V's scales go into the weights; rows past the end count as zeros.  A row's unit is looked at again where a scale could
        // outgrow it by 2^8.  At first the largest weight is 1, and the smallest scale no more than the largest product.
        auto scale_at = [&](int j, int e) {
            const uint2 ds = lds64(box + kQ8VScaleOff + (r0 + 8 * j + 2 * t) * 4);
            return pos + 8 * j + 2 * t + e < end ? larger_scale(e ? ds.y : ds.x) : 0.0f;
        };
        float dm = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * NK; ++j) dm = fmaxf(dm, fmaxf(scale_at(j, 0), scale_at(j, 1)));
        if (__any_sync(0xffffffffu, first[0] || first[1])) {
            float low = INFINITY;
#pragma unroll
            for (int j = 0; j < 2 * NK; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) low = pos + 8 * j + 2 * t + e < end ? fminf(low, scale_at(j, e)) : low;
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 1));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, 2));
#pragma unroll
            for (int h = 0; h < 2; ++h) x.to_units[h] = first[h] ? 32.0f * inverse_unit(low) : x.to_units[h];
        }
        const float top = fmaxf(x.to_units[0], x.to_units[1]);
        if (__any_sync(0xffffffffu, dm * top > 8192.0f || !(top < 32.0f * kMostInverse))) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float most = 0.0f;
#pragma unroll
                for (int j = 0; j < 2 * NK; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float w;  // volatile: or the weights would be made for this rare branch in every step and kept
                        asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(sc[j][2 * h + e] - m_exp[h]));
                        most = fmaxf(most, w * scale_at(j, e));
                    }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                if (most * x.to_units[h] > 8192.0f || !(x.to_units[h] < 32.0f * kMostInverse)) {
                    const float now = 32.0f * inverse_unit(most), f = now / x.to_units[h];
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        x.o[n][2 * h] *= f;
                        x.o[n][2 * h + 1] *= f;
                    }
                    x.to_units[h] = now;
                }
            }
        }
    }
    // A product's sums start from zero and are added up in f32: the tensor core truncates at the size of what it accumulates, and over
    // the 900 keys of a long prefix's share the results came out 4e-6 too small.
    const uint32_t vb = box + R::kVOff;
    uint32_t       ph[NK][4], pl[NK][4];  // f16
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        float pr[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[j][e] = ex2_approx(sc[2 * k + j][e] - m_exp[e >> 1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) x.l[h] += (pr[0][2 * h] + pr[0][2 * h + 1]) + (pr[1][2 * h] + pr[1][2 * h + 1]);
        if constexpr (!Q8) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float h0, l0, h1, l1;
                    split_hi_lo(pr[j][2 * h], h0, l0);
                    split_hi_lo(pr[j][2 * h + 1], h1, l1);
                    ph[k][2 * j + h] = pack_half2(h0, h1);
                    pl[k][2 * j + h] = pack_half2(l0, l1);
                }
        } else {
            const int v_row = r0 + 16 * k + (((lane >> 3) & 1) << 3) + (lane & 7), v_chk = lane >> 4, pos_k = pos + 16 * k + 2 * t;
            uint2     ds[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                ds[j] = lds64(box + kQ8VScaleOff + (r0 + 16 * k + 8 * j + 2 * t) * 4);
                if (pos_k + 8 * j >= end) ds[j].x = 0u;
                if (pos_k + 8 * j + 1 >= end) ds[j].y = 0u;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) pr[j][e] *= x.to_units[e >> 1];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t bh[4], bl[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float s0 = b ? half_hi(ds[j].x) : half_lo(ds[j].x), s1 = b ? half_hi(ds[j].y) : half_lo(ds[j].y);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float h0, l0, h1, l1;
                        split_hi_lo(pr[j][2 * h] * s0, h0, l0);
                        split_hi_lo(pr[j][2 * h + 1] * s1, h1, l1);
                        bh[2 * j + h] = pack_half2(h0, h1);
                        bl[2 * j + h] = pack_half2(l0, l1);
                    }
                }
                uint32_t r[4];
                ldmatrix_x4_trans(vb + v_row * 64 + (((v_chk + 2 * b) ^ ((v_row >> 1) & 3)) << 4), r[0], r[1], r[2], r[3]);
#pragma unroll
                for (int n = 0; n < 4; ++n) {  // chunk n / 2 of 16 columns, even or odd ones
                    const uint32_t sel = n & 1 ? 0x4341 : 0x4240;
                    const uint32_t b0 = s8_pair_to_half2(r[2 * (n >> 1)], sel), b1 = s8_pair_to_half2(r[2 * (n >> 1) + 1], sel);
                    float          a[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_16816(a, bl, b0, b1);
                    mma_16816(a, bh, b0, b1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x.o[4 * b + n][e] += a[e];
                }
            }
        }
    }
    if constexpr (!Q8) {
#pragma unroll
        for (int n2 = 0; n2 < 4; ++n2) {
            float a0[4] = {0.f, 0.f, 0.f, 0.f}, a1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                const int v_row = r0 + 16 * k + (((lane >> 3) & 1) << 3) + (lane & 7), v_chk = lane >> 4, pos_k = pos + 16 * k + 2 * t;
                uint32_t  b0, b1, b2, b3;
                ldmatrix_x4_trans(vb + v_row * 128 + (((2 * n2 + v_chk) ^ (v_row & 7)) << 4), b0, b1, b2, b3);
                if (edge) {  // rows past the end may hold anything: zero times a NaN is none
                    const uint32_t keep0 = keep_rows(pos_k, end), keep1 = keep_rows(pos_k + 8, end);
                    b0 &= keep0; b1 &= keep1; b2 &= keep0; b3 &= keep1;
                }
                mma_16816(a0, pl[k], b0, b1);
                mma_16816(a1, pl[k], b2, b3);
                mma_16816(a0, ph[k], b0, b1);
                mma_16816(a1, ph[k], b2, b3);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.o[2 * n2][e] += a0[e];
                x.o[2 * n2 + 1][e] += a1[e];
            }
        }
    }
}

template <bool Q8>
__global__ void __maxnreg__(152)  // room for two CTAs of the decode kernel (2 x 160 x 128 registers) on the SM
shared_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedParams p) {
    using R = Ring<Q8>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * R::kStages];
    __shared__ int      abort_flag;
    __shared__ float2   ml[kRows], joined[kRows];
    __shared__ int      rows_at[kRows];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float4 * const part      = reinterpret_cast<float4 *>(smem_raw + (smem_base - smem_u32(smem_raw)));
    const int      tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[R::kStages]);
    const Item     w = load_item(p);
    if (w.rows == 0) {  // the same for the whole cluster
        pdl_wait();
        return;
    }
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < R::kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, kWarps);
        }
        fence_mbar_init();
    }
    if (tid < w.rows) rows_at[tid] = w.streams[tid / p.gqa] * p.n_heads + w.kvh * p.gqa + tid % p.gqa;
    __syncthreads();
    const int n_tiles = (w.key1 - w.key0 + kKeys - 1) / kKeys;
    bool      ok = true;
    // Warps of a row tile: groups of 16 rows, and as many key groups as that leaves
    const int groups = (w.rows + 15) >> 4;
    const int rg     = groups <= 1 ? 1 : groups <= 2 ? 2 : 4;
    const int kg = kWarps / rg;

    if (warp == kWarps) {
        // ------------------------------------------------------------------ copies: one lane
        if (lane == 0) {
            int it = 0;
            for (; it < n_tiles; ++it) {
                const int s = it % R::kStages, key = w.key0 + it * kKeys;
                if (it >= R::kStages && !mbar_wait_bounded(empty0 + 8 * s, ((it / R::kStages) - 1) & 1)) {
                    atomicOr(p.status, kStatusTimeout);
                    atomicExch(&abort_flag, 1);
                }
                if (*reinterpret_cast<volatile int *>(&abort_flag)) break;
                const int      boxes = w.key1 - key > kKvTile ? 2 : 1;
                const uint32_t bar   = full0 + 8 * s;
                mbar_expect_tx(bar, boxes * R::kBoxTx);
                for (int b = 0; b < boxes; ++b) {
                    const uint32_t dst = smem_base + s * R::kStageBytes + b * R::kBoxBytes;
                    const int      row = key + b * kKvTile;
                    if constexpr (Q8) {
                        const uint8_t * src = p.q8_tiles + (size_t) w.prefix * p.q8_nb_stream + (size_t) w.kvh * p.q8_nb_head + q8_tile_off(row);
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                                     "l"(src), "r"((uint32_t) kQ8TileBytes), "r"(bar)
                                     : "memory");
                    } else {
                        tma_load_5d(dst, &map_k, bar, 0, row, w.kvh, w.prefix, p.layer);
                        tma_load_5d(dst + R::kVOff, &map_v, bar, 0, row, w.kvh, w.prefix, p.layer);
                    }
                }
            }
            if (*reinterpret_cast<volatile int *>(&abort_flag))  // copies already issued land before the CTA retires
                for (int i = max(0, it - R::kStages); i < it; ++i) mbar_wait_bounded(full0 + 8 * (i % R::kStages), (i / R::kStages) & 1);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ consumers
        const int  g = lane >> 2, t = lane & 3;
        const int  wr = warp % rg, wk = warp / rg, span = kKeys / kg;
        const bool busy = wr < groups;
        Rows       x;
        // Q: rows g and g + 8 of this warp's 16, as value + remainder (the order of the head dimensions as in the decode kernel)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int  row  = 16 * wr + g + 8 * h;
            const bool live = row < w.rows;
            const int  at   = live ? row : 0;
            const int  stream = rows_at[at] / p.n_heads, head = rows_at[at] % p.n_heads;
            const float * qrow = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) head * p.q_nb_head);
            float xs[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int d0 = Q8 ? 32 * (c >> 1) + 8 * t + 4 * (c & 1) : 16 * c + 2 * t;
                const int d1 = Q8 ? d0 + 2 : d0 + 8;
                const float2 a = *reinterpret_cast<const float2 *>(qrow + d0);
                const float2 b = *reinterpret_cast<const float2 *>(qrow + d1);
                xs[c][0] = a.x; xs[c][1] = a.y; xs[c][2] = b.x; xs[c][3] = b.y;
            }
            if (p.rope != nullptr) {
                const float2 * tb = p.rope + (size_t) stream * (kHeadDim / 2);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int d0 = Q8 ? 8 * t + 4 * c : 16 * c + 2 * t;
                    const int d1 = Q8 ? d0 + 2 : d0 + 8;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 r  = tb[(e < 2 ? d0 : d1) + (e & 1)];
                        const float  x0 = xs[c][e], x1 = xs[c + 2][e];
                        xs[c][e]     = __fsub_rn(__fmul_rn(x0, r.x), __fmul_rn(x1, r.y));
                        xs[c + 2][e] = __fadd_rn(__fmul_rn(x0, r.y), __fmul_rn(x1, r.x));
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split_hi_lo(live ? xs[c][e] * p.scale_log2 : 0.0f, hi[e], lo[e]);
                x.qh[c][h]     = pack_half2(hi[0], hi[1]);
                x.qh[c][h + 2] = pack_half2(hi[2], hi[3]);
                x.ql[c][h]     = pack_half2(lo[0], lo[1]);
                x.ql[c][h + 2] = pack_half2(lo[2], lo[3]);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) x.o[n][0] = x.o[n][1] = x.o[n][2] = x.o[n][3] = 0.0f;
        x.m[0] = x.m[1] = -INFINITY;
        x.l[0] = x.l[1] = 0.0f;
        x.to_units[0] = x.to_units[1] = kMostInverse;
        for (int it = 0; it < n_tiles; ++it) {
            const int s = it % R::kStages, key = w.key0 + it * kKeys;
            if (!mbar_wait_bounded(full0 + 8 * s, (it / R::kStages) & 1)) {
                *reinterpret_cast<volatile int *>(&abort_flag) = 1;
                ok = false;
                break;
            }
            if (busy) {
                const int k0 = wk * span;
                const uint32_t box = smem_base + s * R::kStageBytes + (k0 >> 6) * R::kBoxBytes;
#pragma unroll 1
                for (int b = 0; b < span && key + k0 + b < w.key1; b += 32)
                    step<Q8, 2>(x, box + (((k0 & 63) + b) >> 6) * R::kBoxBytes, (k0 + b) & 63, key + k0 + b, w.key1, lane);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * s);
        }
        if (*reinterpret_cast<volatile int *>(&abort_flag)) ok = false;
        if (!ok && lane == 0) atomicOr(p.status, kStatusTimeout);
        ok = named_bar_all(1, kWarps * 32, ok);  // and the ring is no longer read
        if (ok) {
            const int v0 = (wk * rg + wr) * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float l = x.l[h];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int row = v0 + g + 8 * h;
                if (t == 0) ml[row] = make_float2(x.m[h] - (Q8 ? 0.0f : kShift), l);
                float * out = reinterpret_cast<float *>(part + row * kPartPitch);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    if constexpr (Q8) {  // tile n: chunk n / 2, this lane 16 (n / 2) + 4t + (n % 2) and two further
                        const int d = 16 * (n >> 1) + 4 * t + (n & 1);
                        out[d]     = x.o[n][2 * h] * (1.0f / x.to_units[h]);
                        out[d + 2] = x.o[n][2 * h + 1] * (1.0f / x.to_units[h]);
                    } else {
                        *reinterpret_cast<float2 *>(out + 8 * n + 2 * t) = make_float2(x.o[n][2 * h], x.o[n][2 * h + 1]);
                    }
                }
            }
        }
    }
    join_and_write(p, w, part, ml, joined, rows_at, part + kHalfRows * kPartPitch, kg, 16 * rg, ok, tid);
}

// ---------------------------------------------------------------------------------------------------------------------
// Full row tiles on the 5th-generation tensor cores.
//
// Q (scaled by scale * log2 e) lies in shared memory as two f16 tiles, value and remainder; scores S = Q_lo.K + Q_hi.K (the
// small part first: the accumulator truncates) come 64 keys at a time into one of four score buffers in TMEM.  Four softmax
// warps, a thread per row: 64 scores out of TMEM, weights 2^(S - ref) back over them as two packed f16 tiles (value and
// remainder, 22 bits), from where the tensor core takes them as the A operand of P.V.  The output has four accumulators,
// values and remainders of even and of odd tiles, added up in f32 at the end: the tensor core truncates every sum it
// makes, and one accumulator for all came out 2.2e-6 too small after 1024 keys.  The reference of a row is raised only
// when a maximum exceeds it by 2^8 (its accumulators are then rescaled in TMEM).
//   warps 0 .. 4 kGroups - 1  softmax      then one warp  issues S = Q.K, one  O += P.V, and that one, or a third of two
//   groups, the copies of K and V
// One softmax group (192 threads of 128 registers, 81 KB of shared memory; q8_0 107 KB): the CTA runs beside two CTAs of the decode
// kernel, whose time is HBM's, and takes about 1.1 us for 64 keys (q8_0 2.3 us), most of it latency that nothing hides: 0.5 us of
// it are products and exponentials.  Two groups, which take tiles in turn with a reference and accumulators of their own, hide
// some of it (256 streams under two prompts of 2048 / 4096 rows, one row of their own: 23.5 / 28.6 -> 19.8 / 27.6 us; q8_0 34.9 / 54.8
// -> 33.3 / 43.4 us), but leave room for one decode CTA per SM only: taken where the streams' own rows are few against the prefix (see
// vox_attn_decode_shared).
//
// q8_0: the softmax warps turn a tile's bytes into f16 numbers q (exact; a tile ahead of the scores they work on) and keep the
// scales apart.  Either 32-value block has a score accumulator of its own (s = d0 S0 + d1 S1), and its 32 output columns have
// weights of their own, with V's scale of the block taken in, in units (inverse_unit; a thread's row has its own).
constexpr int kSub       = 64;                    // keys of a score tile and of a stage
constexpr int kQTile     = kRows * 128;
constexpr int kTcStage   = 2 * kSub * 128;        // 64 rows of K, 64 rows of V, in f16
template <bool Q8, int kGroups> struct Tc {
    static constexpr int kThreads = (4 * kGroups + 1 + kGroups) * 32;
    // A stage is held from the copy until P.V has retired, about 3500 clocks; beside two decode CTAs there is room for three.
    static constexpr int kStages  = kGroups == 1 ? 3 : Q8 ? 5 : 6;
    static constexpr int kSCols  = Q8 ? 2 * kSub : kSub;   // TMEM columns of a score tile
    static constexpr int kSBufs  = Q8 ? 2 : 4;             // the accumulators, 4 x 64 columns, lie behind the buffers
    static constexpr int kOCol   = kSBufs * kSCols;
    static constexpr int kRaw    = Q8 ? 2 + kGroups : 0;   // q8_0: stages of tiles as the cache holds them
    static constexpr int kRawBytes = 8704;
    static constexpr int kSmem   = 2 * kQTile + kStages * kTcStage + kRaw * kRawBytes + 1024;
    // the partial results, and behind those of one group its CTA's share of the rows, take the queries' and the ring's memory
    static_assert(kRawBytes == kQ8TileBytes && 2 * kQTile + kStages * kTcStage >= 2 * kRows * kPartPitch * 16, "shared memory");
};
constexpr float kTcShift = 6.0f;                  // weights up to 2^(8 + 6): their remainders stay normal f16 numbers
// q8_0: a row's largest product of weight and scale is made 2^4 .. 2^5.  Its unit is looked at where one could be 2^13, and follows if one is
// 2^11.
constexpr float kUnitFirst = 16.0f, kUnitMost = 2048.0f;

// multiply this thread's row of the accumulators by f; rare, kept out of line so that its registers do not weigh on the loop
__device__ __noinline__ void rescale_row(uint32_t t_o, int blocks, float f) {
    tc_fence_after();
#pragma unroll 1
    for (int h = 0; h < blocks; ++h) {  // of 32 columns
        float o[32];
        tmem_ld32(t_o + 32 * h, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= f;
        tmem_st32(t_o + 32 * h, o);
    }
    tc_fence_before();
}

// q8_0: the inverse unit of this thread's row for a tile whose scores lie at t_s (S0, and S1 behind it), whatever its scales (shared memory); where
// it changes, the accumulators at t_o (0: there are none yet) follow.  Rare; it reads the scores again, so that nothing is kept for it.
template <int kBlocks> __device__ __forceinline__ float refit_row(uint32_t t_s, uint32_t scales, float m, uint32_t t_o, float to_units) {
    float most = 0.0f;  // the largest product of weight and V scale (keys past the end have scales of 0)
#pragma unroll 1
    for (int c = 0; c < kSub; c += 8) {
        uint32_t a[8], b[8];
        tmem_ld8_sync(t_s + c, a);
        tmem_ld8_sync(t_s + kSub + c, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint2 k = lds64(scales + 16 * (c + i)), v = lds64(scales + 16 * (c + i) + 8);
            const float e = ex2_approx(fmaf(__uint_as_float(b[i]), __uint_as_float(k.y), __uint_as_float(a[i]) * __uint_as_float(k.x)) - m);
            most = fmaxf(most, e * fmaxf(fabsf(__uint_as_float(v.x)), fabsf(__uint_as_float(v.y))));
        }
    }
    float now = to_units;
    if (most * to_units > kUnitMost || !(to_units < kUnitFirst * kMostInverse)) now = kUnitFirst * inverse_unit(most);
    if (t_o != 0 && __any_sync(0xffffffffu, now != to_units)) rescale_row(t_o, kBlocks, now / to_units);
    return now;
}

// one row of a q8_0 tile: 64 bytes to 64 f16 at their swizzled places; zeros where the row does not exist
__device__ __forceinline__ void expand_row(const uint8_t * bytes, uint8_t * out, int row, bool here) {
#pragma unroll 2
    for (int c = 0; c < 4; ++c) {
        const uint4    x    = *reinterpret_cast<const uint4 *>(bytes + q8_byte_off(row, 16 * c));
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
        uint32_t       h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            h[2 * e]     = here ? s8_pair_to_half2(v[e], 0x4140) : 0u;
            h[2 * e + 1] = here ? s8_pair_to_half2(v[e], 0x4342) : 0u;
        }
        *reinterpret_cast<uint4 *>(out + row * 128 + (((2 * c) ^ (row & 7)) << 4))     = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(out + row * 128 + (((2 * c + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
    }
}

template <bool Q8, int kGroups>
__global__ void __maxnreg__(128)
shared_rows_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedParams p) {
    using Z = Tc<Q8, kGroups>;
    constexpr int kTcStages = Z::kStages, kSBufs = Z::kSBufs, kSCols = Z::kSCols, kTcOCol = Z::kOCol, kRaw = Q8 ? Z::kRaw : 1;
    constexpr int kSoftmax = 4 * kGroups, kScoreWarp = kSoftmax, kOutWarp = kSoftmax + 1, kCopyWarp = kSoftmax + kGroups;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * kTcStages + 3 * kSBufs + 1 + 2 * kRaw];
    __shared__ float4   scales[Q8 ? kTcStages : 1][kSub];   // q8_0: of a row's K and V blocks
    __shared__ uint32_t largest[kTcStages], smallest[kGroups];  // q8_0: the largest of a stage's V scales, the smallest of a group's first tile, as bits
    __shared__ const uint8_t * row_q[kRows];
    __shared__ const float2 *  row_rope[kRows];
    __shared__ uint32_t tmem_slot;
    __shared__ int      abort_flag;
    __shared__ float2   ml[kGroups * kRows], joined[kRows];
    __shared__ int      rows_at[kRows];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *      smem_gen  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t sQ = smem_base, sKV = sQ + 2 * kQTile, sRaw = sKV + kTcStages * kTcStage;
    const int      tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // full: a stage holds its tile in f16; S: scores ready; P: weights ready; F: P.V retired (the score buffer is free, f16: the
    // stage too); empty (q8_0, and two groups): the stage is free (F of a score buffer may complete twice between two looks at it, that of a stage
    // cannot); rfull, rempty: a tile's bytes have landed, are expanded
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = full0 + 8 * kTcStages, bS0 = empty0 + 8 * kTcStages, bP0 = bS0 + 8 * kSBufs,
                   bF0 = bP0 + 8 * kSBufs, bO = bF0 + 8 * kSBufs, rfull0 = bO + 8, rempty0 = rfull0 + 8 * kRaw;
    const Item     w = load_item(p);
    if (w.rows == 0) {  // the same for the whole cluster
        pdl_wait();
        return;
    }
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < kTcStages; ++s) {
            mbar_init(full0 + 8 * s, Q8 ? 4 : 1);
            mbar_init(empty0 + 8 * s, 1);
            largest[s] = 0;
        }
        for (int g = 0; g < kGroups; ++g) smallest[g] = 0x7f800000u;
        for (int s = 0; s < kRaw; ++s) {
            mbar_init(rfull0 + 8 * s, 1);
            mbar_init(rempty0 + 8 * s, 4);
        }
        for (int s = 0; s < kSBufs; ++s) {
            mbar_init(bS0 + 8 * s, 1);
            mbar_init(bP0 + 8 * s, 4);  // one arrival per warp of the group that took the tile
            mbar_init(bF0 + 8 * s, 1);
        }
        mbar_init(bO, 1);
        fence_mbar_init();
    }
    if (warp == kScoreWarp) tmem_alloc(smem_u32(&tmem_slot), 512);
    if (tid < kRows) {  // once per row: the loops below would divide over and over
        const bool live   = tid < w.rows;
        const int  stream = live ? w.streams[tid / p.gqa] : w.streams[0], head = w.kvh * p.gqa + (live ? tid % p.gqa : 0);
        rows_at[tid]   = stream * p.n_heads + head;
        row_q[tid]     = p.q + (size_t) stream * p.q_nb_stream + (size_t) head * p.q_nb_head;
        row_rope[tid]  = p.rope + (size_t) stream * (kHeadDim / 2);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_slot);
    const int n_keys = w.key1 - w.key0, n_sub = (n_keys + kSub - 1) / kSub;

    auto give_up = [&]() {
        atomicOr(p.status, kStatusTimeout);
        atomicExch(&abort_flag, 1);
    };
    auto aborted   = [&]() { return *reinterpret_cast<volatile int *>(&abort_flag) != 0; };
    auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity)) != 0; };
    auto warp_wait2 = [&](uint32_t a, uint32_t pa, uint32_t b, bool two, uint32_t pb) {
        return __all_sync(0xffffffffu, mbar_wait_bounded(a, pa) && (!two || mbar_wait_bounded(b, pb))) != 0;
    };
    auto retired = [&](int U) { return mbar_wait_bounded(bF0 + 8 * (U % kSBufs), (U / kSBufs) & 1); };  // tile U's P.V
    constexpr int kAhead = Q8 ? kRaw : kTcStages;  // tiles on their way
    auto load_tile = [&](int U) {  // one lane
        if constexpr (Q8) {
            const uint32_t  bar = rfull0 + 8 * (U % kRaw), dst = sRaw + (U % kRaw) * Z::kRawBytes;
            const uint8_t * src = p.q8_tiles + (size_t) w.prefix * p.q8_nb_stream + (size_t) w.kvh * p.q8_nb_head + q8_tile_off(w.key0 + U * kSub);
            mbar_expect_tx(bar, kQ8TileBytes);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                         "r"((uint32_t) kQ8TileBytes), "r"(bar)
                         : "memory");
            return;
        }
        const uint32_t bar = full0 + 8 * (U % kTcStages), dst = sKV + (U % kTcStages) * kTcStage;
        mbar_expect_tx(bar, kTcStage);
        tma_load_5d(dst, &map_k, bar, 0, w.key0 + U * kSub, w.kvh, w.prefix, p.layer);
        tma_load_5d(dst + kSub * 128, &map_v, bar, 0, w.key0 + U * kSub, w.kvh, w.prefix, p.layer);
    };
    if (warp == kCopyWarp) {
        if (lane == 0)
            for (int U = 0; U < min(n_sub, kAhead); ++U) load_tile(U);
    } else if (warp < kSoftmax) {
        // Q: 16 threads per row, four head dimensions each; eight loads of a warp in flight.  (Two threads per row, a
        // float2 at a time, took 4 us: every load of a warp touched 16 rows.)
        const int c = lane & 15;
#pragma unroll 1
        for (int half = warp >> 2; half < 2; half += kGroups) {
        float4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float * src = reinterpret_cast<const float *>(row_q[32 * (warp & 3) + 16 * half + 2 * i + (lane >> 4)]) + 4 * c;
            const float2  a = *reinterpret_cast<const float2 *>(src), b = *reinterpret_cast<const float2 *>(src + 2);
            x[i] = make_float4(a.x, a.y, b.x, b.y);
        }
        if (p.rope != nullptr) {  // elements d and d + 32 are partners: lanes c and c ^ 8
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 * tb = row_rope[32 * (warp & 3) + 16 * half + 2 * i + (lane >> 4)] + 4 * (c & 7);
                const float *  xi = &x[i].x;
                float          y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 r = tb[e];
                    const float  other = __shfl_xor_sync(0xffffffffu, xi[e], 8);
                    y[e] = c & 8 ? __fadd_rn(__fmul_rn(other, r.y), __fmul_rn(xi[e], r.x)) : __fsub_rn(__fmul_rn(xi[e], r.x), __fmul_rn(other, r.y));
                }
                x[i] = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int    row = 32 * (warp & 3) + 16 * half + 2 * i + (lane >> 4);
            const bool   live = row < w.rows;
            float        h[4], l[4];
            split_hi_lo(live ? x[i].x * p.scale_log2 : 0.0f, h[0], l[0]);
            split_hi_lo(live ? x[i].y * p.scale_log2 : 0.0f, h[1], l[1]);
            split_hi_lo(live ? x[i].z * p.scale_log2 : 0.0f, h[2], l[2]);
            split_hi_lo(live ? x[i].w * p.scale_log2 : 0.0f, h[3], l[3]);
            uint8_t * dst = smem_gen + row * 128 + (((c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8;
            *reinterpret_cast<uint2 *>(dst)          = make_uint2(pack_half2(h[0], h[1]), pack_half2(h[2], h[3]));
            *reinterpret_cast<uint2 *>(dst + kQTile) = make_uint2(pack_half2(l[0], l[1]), pack_half2(l[2], l[3]));
        }
        }
        fence_proxy_async_smem();
    }
    __syncthreads();

    bool all_ok = true;  // of the softmax warps
    if (warp == kScoreWarp) {
        // ------------------------------------------------------------------ scores (all lanes in the loop, one issues)
        constexpr uint32_t idesc = idesc_f16(kSub, false);
        const uint64_t     dQ = smem_desc_sw128(sQ), dQlo = smem_desc_sw128(sQ + kQTile), dK = smem_desc_sw128(sKV);
        const bool         leader = elect_one();
        bool               ok = true;
        for (int U = 0; U < n_sub && ok; ++U) {
            const int st = U % kTcStages, sb = U % kSBufs;
            if (!warp_wait2(full0 + 8 * st, (U / kTcStages) & 1, bF0 + 8 * sb, U >= kSBufs, ((U / kSBufs) - 1) & 1)) { ok = false; break; }
            tc_fence_after();
            if (leader) {
                const uint32_t dS = tmem + kSCols * sb;
                const uint64_t k0 = dK + (uint64_t) (st * (kTcStage >> 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16(Q8 ? dS + (k >> 1) * kSub : dS, dQlo + k * 2, k0 + k * 2, idesc, (Q8 ? k & 1 : k) > 0);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16(Q8 ? dS + (k >> 1) * kSub : dS, dQ + k * 2, k0 + k * 2, idesc, 1);
                tc_commit(bS0 + 8 * sb);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) give_up();
    } else if (warp == kOutWarp) {
        // ------------------------------------------------------------------ output, and the copies behind it
        constexpr uint32_t idesc = idesc_f16(Q8 ? 32 : kHeadDim, true);
        const uint64_t     dV = smem_desc_sw128_mn(sKV + kSub * 128, 16);
        const bool         leader = elect_one();
        bool               ok = true;
        int                loaded = min(n_sub, kAhead);
        for (int U = 0; U < n_sub && ok; ++U) {
            const int st = U % kTcStages, sb = U % kSBufs;
            if (!warp_wait2(full0 + 8 * st, (U / kTcStages) & 1, bP0 + 8 * sb, true, (U / kSBufs) & 1)) { ok = false; break; }
            tc_fence_after();
            if (leader) {
                const uint64_t v0 = dV + (uint64_t) (st * (kTcStage >> 4));
#pragma unroll
                for (int b = 0; b < (Q8 ? 2 : 1); ++b) {
                    // q8_0: block b's 32 columns of V, 64 bytes into the swizzle atom
                    const uint32_t tP = tmem + kSCols * sb + kSub * b, tO = tmem + kTcOCol + 2 * kHeadDim * (U & 1) + 32 * b;
                    const uint64_t vb = v0 + b * (64 >> 4);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_f16_ts(tO, tP + 8 * k, vb + k * (2048 >> 4), idesc, U > 1 || k > 0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc_mma_f16_ts(tO + kHeadDim, tP + kSub / 2 + 8 * k, vb + k * (2048 >> 4), idesc, U > 1 || k > 0);
                }
                tc_commit(bF0 + 8 * sb);
                if (Q8 || kGroups == 2) tc_commit(empty0 + 8 * st);
                if (U == n_sub - 1) tc_commit(bO);
            }
            __syncwarp();
            // f16: the stage of the tile before this one is free as soon as its P.V has retired, which was issued a tile ago;
            // q8_0: the bytes of this tile were expanded before its scores were made
            if (kGroups == 1 && (Q8 || U > 0) && loaded < n_sub) {
                const bool free = Q8 ? warp_wait(rempty0 + 8 * (U % kRaw), (U / kRaw) & 1) : __all_sync(0xffffffffu, retired(U - 1)) != 0;
                if (!free || __any_sync(0xffffffffu, aborted())) { ok = false; break; }
                if (lane == 0) load_tile(loaded);
                ++loaded;
            }
        }
        if (!ok) {
            if (lane == 0) give_up();
            for (int i = kGroups == 1 ? max(0, loaded - kAhead) : loaded; i < loaded; ++i)  // copies in flight land
                warp_wait(Q8 ? rfull0 + 8 * (i % kRaw) : full0 + 8 * (i % kTcStages), (i / kAhead) & 1);
        }
    } else if (kGroups == 2 && warp == kCopyWarp) {
        // ------------------------------------------------------------------ copies (issuing one costs the output warp 500 clocks)
        if (lane == 0) {
            bool ok = true;
            int  U  = min(n_sub, kAhead);
            for (; U < n_sub; ++U) {  // the stage's last tile has retired, q8_0: has been expanded
                const uint32_t bar = Q8 ? rempty0 + 8 * (U % kRaw) : empty0 + 8 * (U % kTcStages);
                if (!mbar_wait_bounded(bar, ((U / kAhead) - 1) & 1) || aborted()) { ok = false; break; }
                load_tile(U);
            }
            if (!ok) give_up();
            if (aborted())
                for (int i = max(0, U - kAhead); i < U; ++i)  // copies in flight land
                    mbar_wait_bounded(Q8 ? rfull0 + 8 * (i % kRaw) : full0 + 8 * (i % kTcStages), (i / kAhead) & 1);
        }
    } else {
        // ------------------------------------------------------------------ softmax: a thread per row
        const int      group = warp >> 2, row = tid & 127;
        // accumulators: [parity of the tile][value, remainder][64]; with two groups a group has those of one parity
        const uint32_t t_row = tmem + ((uint32_t) (32 * (warp & 3)) << 16), t_o = t_row + kTcOCol + (kGroups == 2 ? 2 * kHeadDim * group : 0);
        float          m = -INFINITY, l = 0.0f, to_units = 1.0f;  // q8_0: see inverse_unit
        bool           ok = true;
        // q8_0: tile U's bytes to f16, K by the group's first two warps, V by the others; its scales, and the largest of V's
        auto expand = [&](int U) {
            const int rs = U % kRaw, st = U % kTcStages, key = row & 63, left = n_keys - U * kSub;
            if (!mbar_wait_bounded(rfull0 + 8 * rs, (U / kRaw) & 1) ||
                (U >= kTcStages && !mbar_wait_bounded(empty0 + 8 * st, ((U / kTcStages) - 1) & 1))) return false;
            const uint8_t * raw = smem_gen + (sRaw - smem_base) + rs * Z::kRawBytes;
            uint8_t *       out = smem_gen + (sKV - smem_base) + st * kTcStage;
            const bool      v   = row >= kSub, here = key < left;
            expand_row(raw + (v ? kQ8VBytesOff : 0), out + (v ? kSub * 128 : 0), key, here);
            const uint32_t d  = here ? *reinterpret_cast<const uint32_t *>(raw + (v ? kQ8VScaleOff : kQ8KScaleOff) + key * 4) : 0u;
            reinterpret_cast<float2 *>(&scales[Q8 ? st : 0][key])[v] = make_float2(half_lo(d), half_hi(d));
            if (v) {
                const __half2  a   = __habs2(as_half2(d));
                const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(__low2float(a), __high2float(a))));
                if (lane == 0) atomicMax(&largest[st], top);
                if (U < kGroups) {
                    const uint32_t low = __reduce_min_sync(0xffffffffu, here ? __float_as_uint(fmaxf(__low2float(a), __high2float(a))) : 0x7f800000u);
                    if (lane == 0) atomicMin(&smallest[U], low);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(full0 + 8 * st);
                mbar_arrive(rempty0 + 8 * rs);
            }
            return true;
        };
        if (Q8 && group < n_sub) {
            // the first tile's largest weight is 1, so the smallest scale is no more than the largest product
            ok     = expand(group) && mbar_wait_bounded(full0 + 8 * (group % kTcStages), 0);
            to_units = kUnitFirst * inverse_unit(__uint_as_float(*reinterpret_cast<volatile uint32_t *>(&smallest[group])));
        }
        for (int U = group; U < n_sub && (Q8 || ok); U += kGroups) {
            const int sb = U % kSBufs, left = n_keys - U * kSub;  // keys of this tile and after
            // (q8_0: a warp whose wait ran out stays until the barrier at the end of the tile, which the others wait at)
            if (Q8 && U + kGroups < n_sub && !expand(U + kGroups)) ok = false;
            if (!mbar_wait_bounded(bS0 + 8 * sb, (U / kSBufs) & 1) || (Q8 && !mbar_wait_bounded(full0 + 8 * (U % kTcStages), (U / kTcStages) & 1))) {
                ok = false;
                if (!Q8) break;
            }
            tc_fence_after();
            const uint32_t t_s = t_row + kSCols * sb;
            const float4 * sc  = scales[Q8 ? U % kTcStages : 0];
            uint32_t       r[kSub];
            tmem_ld64_sync(t_s, r);
            if constexpr (Q8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t x[32];
                    tmem_ld32_sync(t_s + kSub + 32 * h, x);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 d = *reinterpret_cast<const float2 *>(sc + 32 * h + i);
                        r[32 * h + i] = __float_as_uint(fmaf(__uint_as_float(x[i]), d.y, __uint_as_float(r[32 * h + i]) * d.x));
                    }
                }
            }
            if (left < kSub) {
#pragma unroll
                for (int i = 0; i < kSub; ++i)
                    if (i >= left) r[i] = 0xff800000u;
            }
            if (!Q8 && left < kSub) {
                // rows past the prefix may hold anything, and zero times a NaN is none: V's are cleared
                const int st = U % kTcStages;
                if (!mbar_wait_bounded(full0 + 8 * st, (U / kTcStages) & 1)) { ok = false; break; }
                if (row >= left && row < kSub) {
                    uint4 * v = reinterpret_cast<uint4 *>(smem_gen + (sKV - smem_base) + st * kTcStage + (kSub + row) * 128);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
            }
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < kSub; i += 4) {
                t0 = max3(t0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                t1 = max3(t1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
            }
            const float top = fmaxf(t0, t1);
            const bool first = U < kGroups;
            if (first) m = top;
            if constexpr (Q8) {
                // A product is below 2^(top - m) times a scale below 2^(e0 + 1) times less than 2^(e1 + 1).  (By exponents: what `top` is waited
                // for is a subtraction and a comparison.  With the powers themselves 256 streams under 4096 rows took 2.5 us longer.)
                auto room = [&]() {
                    const int e = (int) (*reinterpret_cast<volatile uint32_t *>(&largest[U % kTcStages]) >> 23) + (int) (__float_as_uint(to_units) >> 23) - 254;
                    return to_units < kUnitFirst * kMostInverse ? (float) (11 - e) : -INFINITY;
                };
                if (top - m > 8.0f) {
                    l *= ex2_approx(m - top);
                    to_units *= ex2_approx(top - m);  // in the accumulators' place
                    m = top;
                }
                if (__any_sync(0xffffffffu, top - m > room())) {
                    if (!first && !retired(U - kGroups)) ok = false;  // the accumulators are at rest once P.V of the group's tile before has retired
                    to_units = refit_row<8 / kGroups>(t_s, smem_u32(sc), m, first ? 0u : t_o, to_units);
                }
            } else if (!first) {
                const bool raise = top > m + 8.0f;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2_approx(m - top) : 1.0f;
                    if (raise) m = top;
                    l *= f;
                    if (!retired(U - kGroups)) { ok = false; break; }
                    rescale_row(t_o, 8 / kGroups, f);
                }
            }
            const float ref = Q8 ? m : m - kTcShift;
#pragma unroll
            for (int g = 0; g < kSub / 16; ++g) {
                if constexpr (Q8) {
                    uint32_t hi[2][8], lo[2][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float  e0 = ex2_approx(__uint_as_float(r[16 * g + 2 * i]) - ref), e1 = ex2_approx(__uint_as_float(r[16 * g + 2 * i + 1]) - ref);
                        const float2 d0 = *reinterpret_cast<const float2 *>(&sc[16 * g + 2 * i].z), d1 = *reinterpret_cast<const float2 *>(&sc[16 * g + 2 * i + 1].z);
                        l += e0 + e1;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const float p0 = e0 * to_units * (b ? d0.y : d0.x), p1 = e1 * to_units * (b ? d1.y : d1.x);
                            const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);
                            const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                            hi[b][i] = pack_half2(h0, h1);
                            lo[b][i] = pack_half2(p0 - h0, p1 - h1);
                        }
                    }
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        tmem_st8_nowait(t_s + kSub * b + 8 * g, hi[b]);
                        tmem_st8_nowait(t_s + kSub * b + kSub / 2 + 8 * g, lo[b]);
                    }
                    continue;
                }
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p0 = ex2_approx(__uint_as_float(r[16 * g + 2 * i]) - ref);
                    const float p1 = ex2_approx(__uint_as_float(r[16 * g + 2 * i + 1]) - ref);
                    const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);
                    const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                    hi[i] = pack_half2(h0, h1);
                    lo[i] = pack_half2(p0 - h0, p1 - h1);
                    l += p0 + p1;
                }
                tmem_st8_nowait(t_s + 8 * g, hi);
                tmem_st8_nowait(t_s + kSub / 2 + 8 * g, lo);
            }
            tmem_wait_st();
            tc_fence_before();
            if (Q8 && !named_bar_all(2 + group, 128, ok)) { ok = false; break; }  // every warp of the group is done with the tile's scales
            if (Q8 && row == 0) largest[U % kTcStages] = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(bP0 + 8 * sb);
        }
        if (ok && n_sub > 0 && !mbar_wait_bounded(bO, 0)) ok = false;
        if (!ok) give_up();
        all_ok = named_bar_all(1, 128 * kGroups, ok && !aborted());  // every copy and every score has been used: the memory is free
        if (all_ok && n_sub > 0) {
            tc_fence_after();
            float4 * const part  = reinterpret_cast<float4 *>(smem_gen) + (group * kRows + row) * kPartPitch;
            const float    f     = Q8 ? 1.0f / to_units : 1.0f;
            const int      parts = group >= n_sub ? 0 : kGroups == 2 || n_sub == 1 ? 2 : 4;  // accumulators with something in them
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t r[32], x[32];
                tmem_ld32_sync(t_o + 32 * h, r);
                if (parts == 0) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) r[c] = 0u;
                }
#pragma unroll 1
                for (int o = 1; o < parts; ++o) {
                    tmem_ld32_sync(t_o + kHeadDim * o + 32 * h, x);
#pragma unroll
                    for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) + __uint_as_float(x[c]));
                }
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    part[8 * h + c] = make_float4(__uint_as_float(r[4 * c]) * f, __uint_as_float(r[4 * c + 1]) * f, __uint_as_float(r[4 * c + 2]) * f,
                                                  __uint_as_float(r[4 * c + 3]) * f);
            }
            ml[group * kRows + row] = make_float2(Q8 ? m : m - kTcShift, l);
        }
        if (kGroups == 2) named_bar_sync(1, 128 * kGroups);  // the first group joins both
    }
    // Every role has left its loop and the results are in shared memory.  TMEM goes back before the cluster meets: two CTAs of this
    // kernel fit an SM (those of two calls, or of one where the decode kernel leaves room), an allocation waits for the other's release,
    // and two clusters that each held some SMs' TMEM while they waited for their other CTAs would wait for good.  (After a wait that
    // ran out products may still be on their way: then at the end.)
    tc_fence_before();
    __syncthreads();
    const bool late = aborted();
    if (warp == kScoreWarp && !late) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    float4 * const part = reinterpret_cast<float4 *>(smem_gen);
    join_and_write(p, w, part, ml, joined, rows_at, part + kRows * kPartPitch, kGroups, kRows, all_ok, tid);
    if (late) {
        __syncthreads();
        if (warp == kScoreWarp) {
            tc_fence_after();
            tmem_dealloc(tmem, 512);
        }
    }
}

// CTAs per (row tile, kv head): as many as fill the SMs once, eight at most.  A second, thinner wave costs more than SMs left
// idle.  No more than the prefix has tiles of keys, but four where row tiles are full: the CTAs also share out the rows.
int cluster_size(int sms, int n_tiles, int n_kv_heads, int n_keys, bool full) {
    const int useful = std::max((n_keys + kKeys - 1) / kKeys, full ? 4 : 1);
    return std::max(1, std::min(std::min(kMaxCluster, sms / std::max(1, n_tiles * n_kv_heads)), useful));
}

// The arrangement for the mma.sync kernel: the smallest row tiles whose CTAs still fit the SMs once with the keys cut as
// finely as can be.  A warp works on 16 rows, so smaller tiles leave every warp fewer keys.
int small_arrangement(const vox_prefix_plan * pl, int sms, int n_kv_heads, int n_keys) {
    const int finest = std::min(kMaxCluster, (n_keys + kKeys - 1) / kKeys);
    for (int k = kArrangements - 1; k > 1; --k)
        if (pl->n_tiles[k] * n_kv_heads * finest <= sms) return k;
    return 1;
}

size_t aligned(size_t n) { return (n + 255) & ~(size_t) 255; }

// Arranges the streams by prefix: a counting sort, then row tiles of one prefix each.  An entry out of range is refused
// before anything of the plan changes.
int arrange(vox_prefix_plan * pl, const int32_t * prefix_of) {
    for (int s = 0; s < pl->n_streams; ++s)
        VOX_REQUIRE(prefix_of[s] >= -1 && prefix_of[s] < pl->n_prefixes, VOX_ATTN_INVALID_ARGUMENT,
                    "prefix_of[%d] = %d: not a prefix in [0, %d), nor -1", s, prefix_of[s], pl->n_prefixes);
    std::vector<int32_t> start, count;
    try {
        start.assign((size_t) pl->n_prefixes, 0);
        count.assign((size_t) pl->n_prefixes, 0);
        pl->next.assign((size_t) pl->n_prefixes, 0);
        pl->host.assign(pl->words(), 0);
    } catch (const std::exception &) {
        set_error("out of host memory");
        return VOX_ATTN_OUT_OF_MEMORY;
    }
    pl->first = pl->n_prefixes;
    for (int s = 0; s < pl->n_streams; ++s)
        if (prefix_of[s] >= 0) {
            count[prefix_of[s]] += 1;
            pl->first = std::min(pl->first, prefix_of[s]);
        }
    for (int k = 0; k < kArrangements; ++k) {
        const int per_tile = pl->per_tile(k);
        int32_t * tiles = pl->host.data() + pl->at[k], * members = pl->host.data() + pl->members_at(k);
        int       placed = 0, n_tiles = 0;
        for (int g = 0; g < pl->n_prefixes; ++g) {
            start[g]    = n_tiles;
            pl->next[g] = 0;
            for (int left = count[g]; left > 0; left -= per_tile, ++n_tiles) {
                tiles[2 * (size_t) n_tiles]     = g;
                tiles[2 * (size_t) n_tiles + 1] = std::min(left, per_tile);
            }
            placed += count[g];
        }
        for (int s = 0; s < pl->n_streams; ++s) {
            const int g = prefix_of[s];
            if (g < 0) continue;
            const int j = pl->next[g]++;
            members[(size_t) (start[g] + j / per_tile) * per_tile + j % per_tile] = s;
        }
        pl->n_tiles[k] = n_tiles;
        if (k == 0) pl->full = 2 * placed > n_tiles * per_tile;
    }
    return VOX_ATTN_OK;
}

int check_shared(const vox_engine * e, const vox_decode_shared_args * a) {
    VOX_REQUIRE(e && a, VOX_ATTN_INVALID_ARGUMENT, "vox_attn_decode_shared: null argument");
    const int rc = check_decode(e, &a->own, "vox_attn_decode_shared");
    if (rc != VOX_ATTN_OK) return rc;
    const vox_kv_cache * c = a->own.cache;
    VOX_REQUIRE(a->own.stream_order == nullptr, VOX_ATTN_UNSUPPORTED, "vox_attn_decode_shared takes no stream_order");
    VOX_REQUIRE((reinterpret_cast<uintptr_t>(a->lse) & 3) == 0, VOX_ATTN_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    if (a->prefix == nullptr && a->plan == nullptr) {  // own rows only: nothing of a prefix may be given
        VOX_REQUIRE(a->prefix_len == nullptr && a->prefix_bound == 0, VOX_ATTN_INVALID_ARGUMENT, "prefix, plan and prefix_len must be given together");
        return VOX_ATTN_OK;
    }
    {
        // the prefix kernel reads the queries while the decode kernel writes its results: they must not share memory
        const uintptr_t q0 = reinterpret_cast<uintptr_t>(a->own.q), d0 = reinterpret_cast<uintptr_t>(a->own.dst);
        const size_t    q_bytes = (size_t) (a->own.n_streams - 1) * a->own.q_nb_stream + (size_t) (a->own.n_heads - 1) * a->own.q_nb_head + kHeadDim * sizeof(float);
        const size_t    d_bytes = (size_t) a->own.n_streams * a->own.n_heads * kHeadDim * sizeof(float);
        VOX_REQUIRE(q0 + q_bytes <= d0 || d0 + d_bytes <= q0, VOX_ATTN_INVALID_ARGUMENT, "dst and q must not overlap");
    }
    VOX_REQUIRE(a->prefix && a->plan && a->prefix_len, VOX_ATTN_INVALID_ARGUMENT, "prefix, plan and prefix_len must be given together");
    VOX_REQUIRE(a->prefix->e == e && a->plan->e == e, VOX_ATTN_INVALID_ARGUMENT, "the prefix cache or the plan belongs to another engine");
    const vox_kv_config & pc = a->prefix->cfg;
    VOX_REQUIRE(pc.type == c->cfg.type && pc.n_kv_heads == c->cfg.n_kv_heads, VOX_ATTN_INVALID_ARGUMENT,
                "the prefix cache differs from the streams' cache in type or heads");
    VOX_REQUIRE(a->own.layer < pc.n_layers, VOX_ATTN_INVALID_ARGUMENT, "layer %d out of range (the prefix cache holds %d)", a->own.layer, pc.n_layers);
    VOX_REQUIRE(a->prefix_bound >= 0 && a->prefix_bound <= pc.max_len, VOX_ATTN_INVALID_ARGUMENT,
                "prefix_bound %d exceeds the prefix cache's capacity %d", a->prefix_bound, pc.max_len);
    VOX_REQUIRE(a->plan->n_streams == a->own.n_streams, VOX_ATTN_INVALID_ARGUMENT, "the plan arranges %d streams, the call has %d",
                a->plan->n_streams, a->own.n_streams);
    VOX_REQUIRE(a->plan->n_prefixes <= pc.n_streams, VOX_ATTN_INVALID_ARGUMENT, "the plan names %d prefixes, the prefix cache holds %d",
                a->plan->n_prefixes, pc.n_streams);
    // the arriving rows are stored while the prefixes are read, in no order
    VOX_REQUIRE(a->prefix != c || a->own.k_new == nullptr || a->plan->first >= a->own.n_streams, VOX_ATTN_INVALID_ARGUMENT,
                "stream %d of the cache is a prefix and one of the %d that the call appends to", a->plan->first, a->own.n_streams);
    VOX_REQUIRE(a->plan->gqa * c->cfg.n_kv_heads == a->own.n_heads, VOX_ATTN_INVALID_ARGUMENT, "the plan was made for %d heads per kv head",
                a->plan->gqa);
    return VOX_ATTN_OK;
}

}  // namespace

extern "C" {

int vox_prefix_plan_create(vox_engine * e, int n_streams, int n_prefixes, int n_heads, int n_kv_heads, const int32_t * prefix_of,
                           vox_prefix_plan ** out) {
    VOX_REQUIRE(e && out && prefix_of, VOX_ATTN_INVALID_ARGUMENT, "vox_prefix_plan_create: null argument");
    *out = nullptr;
    VOX_REQUIRE(n_streams > 0 && n_streams <= (1 << 20) && n_prefixes > 0 && n_prefixes <= (1 << 20), VOX_ATTN_INVALID_ARGUMENT,
                "%d streams, %d prefixes: both must be in [1, 2^20]", n_streams, n_prefixes);
    VOX_REQUIRE(n_kv_heads > 0 && n_heads > 0 && n_heads % n_kv_heads == 0, VOX_ATTN_INVALID_ARGUMENT,
                "n_heads %d is not a multiple of n_kv_heads %d", n_heads, n_kv_heads);
    VOX_REQUIRE(n_heads / n_kv_heads <= 8, VOX_ATTN_UNSUPPORTED, "GQA ratio above 8 is not supported");
    VOX_CUDA_TRY(cudaSetDevice(e->device));
    vox_prefix_plan * pl = new (std::nothrow) vox_prefix_plan();
    VOX_REQUIRE(pl != nullptr, VOX_ATTN_OUT_OF_MEMORY, "out of host memory");
    pl->e = e; pl->n_streams = n_streams; pl->n_prefixes = n_prefixes; pl->gqa = n_heads / n_kv_heads;
    // full tiles, and one that is not full for every prefix in use
    for (int k = 0; k < kArrangements; ++k) {
        pl->max_tiles[k] = n_streams / pl->per_tile(k) + std::min(n_streams, n_prefixes);
        pl->at[k + 1] = (pl->members_at(k) + (size_t) pl->max_tiles[k] * pl->per_tile(k) + 1) & ~(size_t) 1;  // 8-byte pairs
    }
    int rc = arrange(pl, prefix_of);
    if (rc == VOX_ATTN_OK) {
        cudaError_t err = cudaMalloc(reinterpret_cast<void **>(&pl->dev), pl->words() * sizeof(int32_t));
        if (err == cudaSuccess) err = cudaMemcpy(pl->dev, pl->host.data(), pl->words() * sizeof(int32_t), cudaMemcpyHostToDevice);
        if (err != cudaSuccess) {
            set_error("allocating the prefix plan failed: %s", cudaGetErrorString(err));
            cudaGetLastError();
            rc = VOX_ATTN_OUT_OF_MEMORY;
        }
    }
    if (rc != VOX_ATTN_OK) {
        if (pl->dev) cudaFree(pl->dev);
        delete pl;
        return rc;
    }
    *out = pl;
    return VOX_ATTN_OK;
}

void vox_prefix_plan_destroy(vox_prefix_plan * pl) {
    if (!pl) return;
    cudaSetDevice(pl->e->device);
    if (pl->dev) cudaFree(pl->dev);
    delete pl;
}

int vox_prefix_plan_set(vox_prefix_plan * pl, const int32_t * prefix_of, void * stream) {
    VOX_REQUIRE(pl && prefix_of, VOX_ATTN_INVALID_ARGUMENT, "vox_prefix_plan_set: null argument");
    int current = -1;  // as the calls that read the plan: a stream of another device would not order the copy with them
    VOX_CUDA_TRY(cudaGetDevice(&current));
    VOX_REQUIRE(current == pl->e->device, VOX_ATTN_INVALID_ARGUMENT, "the engine's device %d must be the current device (current is %d)", pl->e->device, current);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    VOX_CUDA_TRY(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture));
    VOX_REQUIRE(capture == cudaStreamCaptureStatusNone, VOX_ATTN_UNSUPPORTED, "vox_prefix_plan_set copies from the host: call it outside a capture");
    const int rc = arrange(pl, prefix_of);
    if (rc != VOX_ATTN_OK) return rc;
    // from pageable memory: the copy has taken its source when the call returns
    VOX_CUDA_TRY(cudaMemcpyAsync(pl->dev, pl->host.data(), pl->words() * sizeof(int32_t), cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream)));
    return VOX_ATTN_OK;
}

size_t vox_attn_decode_shared_workspace_bytes(const vox_decode_shared_args * a) {
    if (a == nullptr || a->own.cache == nullptr || a->own.n_streams <= 0 || a->own.n_heads <= 0) return 0;
    const size_t own = decode_shared_workspace_bytes(a->own.n_streams, a->own.n_heads, a->own.cache->cfg.n_kv_heads, a->own.kv_bound);
    return aligned(own) + (a->plan != nullptr ? (size_t) a->own.n_streams * a->own.n_heads * sizeof(float2) : 0);
}

int vox_attn_decode_shared(vox_engine * e, const vox_decode_shared_args * a, void * workspace, size_t workspace_bytes, void * stream) {
    int rc = check_shared(e, a);
    if (rc != VOX_ATTN_OK) return rc;
    int current = -1;
    VOX_CUDA_TRY(cudaGetDevice(&current));
    VOX_REQUIRE(current == e->device, VOX_ATTN_INVALID_ARGUMENT, "the engine's device %d must be the current device (current is %d)", e->device, current);
    const size_t need = vox_attn_decode_shared_workspace_bytes(a);
    VOX_REQUIRE(workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
                VOX_ATTN_WORKSPACE_TOO_SMALL, "vox_attn_decode_shared needs %zu workspace bytes (16-byte aligned), got %zu", need, workspace_bytes);
    cudaStream_t            st  = static_cast<cudaStream_t>(stream);
    const vox_prefix_plan * pl  = a->plan;
    const int               HK  = a->own.cache->cfg.n_kv_heads;
    const size_t            own = aligned(decode_shared_workspace_bytes(a->own.n_streams, a->own.n_heads, HK, a->own.kv_bound));
    const bool              shares = pl != nullptr && a->prefix_bound > 0;
    float2 * const          ml  = shares ? reinterpret_cast<float2 *>(static_cast<uint8_t *>(workspace) + own) : nullptr;
    const vox_kv_cache *    pc  = a->prefix;
    const bool              q8  = a->own.cache->cfg.type == VOX_TYPE_Q8_0, tc = shares && pl->full;
    const int               sms = std::min(kDecodeMaxSms, e->sm_count), k = !shares || tc ? 0 : small_arrangement(pl, sms, HK, a->prefix_bound);
    const int               cluster = shares ? cluster_size(sms, pl->n_tiles[k], HK, a->prefix_bound, tc) : 1;
    // Two softmax groups, beside one decode CTA per SM, where the streams' own 64-row tiles per SM are few against the tiles that a
    // CTA of the prefix kernel walks: then the prefix kernel is what the call waits for.  256 streams under two prompts of 4096
    // rows, own rows 1 / 128 / 512 / 1024 / 2048: f16 28 / 25 / 36 / 47 / 68 us against 29 / 30 / 32 / 38 / 49 us with one group;
    // q8_0, whose scores cost more, 44 / 44 / 50 / 57 / 75 against 55 / 56 / 61 / 63 / 71 us.
    const long long own_tiles = (long long) a->own.n_streams * HK * ((a->own.kv_bound + kKvTile - 1) / kKvTile) / sms;
    const bool      wide = tc && 4 * own_tiles <= (q8 ? 20LL : 5LL) * ((a->prefix_bound + kSub - 1) / kSub) / cluster;
    rc = launch_decode_shared(e, &a->own, OwnRows{a->lse, ml, !shares ? 0 : wide ? 1 : 2}, workspace, own, st);
    if (rc != VOX_ATTN_OK || !shares) return rc;
    SharedParams         p;
    p.q = reinterpret_cast<const uint8_t *>(a->own.q);
    p.q_nb_head = a->own.q_nb_head; p.q_nb_stream = a->own.q_nb_stream;
    p.rope    = reinterpret_cast<const float2 *>(a->own.rope_table);
    p.tiles   = reinterpret_cast<const int2 *>(pl->dev + pl->at[k]);
    p.members = pl->dev + pl->members_at(k);
    p.len     = a->prefix_len;
    p.per_tile = pl->per_tile(k); p.n_kv_heads = HK; p.n_heads = a->own.n_heads; p.gqa = pl->gqa; p.layer = a->own.layer; p.max_len = pc->cfg.max_len;
    p.cluster    = cluster;
    p.scale_log2 = a->own.scale * 1.4426950408889634f;
    p.q8_tiles   = pc->k_data + (size_t) a->own.layer * pc->nb_layer;
    p.q8_nb_head = pc->nb_head; p.q8_nb_stream = pc->nb_stream;
    p.dst = a->own.dst; p.ml = ml; p.lse = a->lse;
    p.status = e->status_dev;
    auto     kernel  = q8 ? shared_rows_kernel<true> : shared_rows_kernel<false>;
    int      smem    = q8 ? Ring<true>::kSmemBytes : Ring<false>::kSmemBytes, threads = kThreads;
    uint32_t bit     = 1u << (q8 ? 19 : 18);
    if (wide) {
        kernel  = q8 ? shared_rows_tc_kernel<true, 2> : shared_rows_tc_kernel<false, 2>;
        smem    = q8 ? Tc<true, 2>::kSmem : Tc<false, 2>::kSmem;
        threads = Tc<false, 2>::kThreads;
        bit     = 1u << (q8 ? 30 : 29);
    } else if (tc) {
        kernel  = q8 ? shared_rows_tc_kernel<true, 1> : shared_rows_tc_kernel<false, 1>;
        smem    = q8 ? Tc<true, 1>::kSmem : Tc<false, 1>::kSmem;
        threads = Tc<false, 1>::kThreads;
        bit     = 1u << (q8 ? 28 : 21);
    }
    if (!(e->attr_mask & bit)) {
        VOX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        // all of the SM's memory as shared memory, so that a CTA fits beside one of the decode kernel's
        VOX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        e->attr_mask |= bit;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (pl->max_tiles[k] * HK * p.cluster)); cfg.blockDim = dim3((unsigned) threads);
    cfg.dynamicSmemBytes = (size_t) smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) p.cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, pc->map_k, pc->map_v, p);
    return check_launch(e, tc ? (q8 ? "shared_rows_tc_kernel<q8_0>" : "shared_rows_tc_kernel<f16>") : q8 ? "shared_rows_kernel<q8_0>" : "shared_rows_kernel<f16>");
}

}  // extern "C"
