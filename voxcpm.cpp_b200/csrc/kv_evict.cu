// Eviction from the cache by accumulated attention weight (vox_kv_evict).
//
// Per (layer, stream, kv head) with more rows than the budget: the `budget` largest keys stay (a key orders the rows as the
// contract does: protected rows above every score, scores as numbers, NaN below; equal keys by index), then the i-th kept
// row at or above the budget moves to the i-th place below it whose row goes.  Sources and destinations never overlap, so
// rows move in place and in any order.
//
// One CTA per row list, keys in shared memory.  The border between what stays and what goes is found by a histogram of the
// keys' top 11 bits (sign, exponent and two bits of the mantissa: a bin is a quarter of an octave) and, as a rule, by ranking the
// keys of the bin it falls in against one another; only a bin with more keys than threads (many equal scores) is cut further, 11 and
// 10 bits at a time.  Lists are few when one stream is cut: then a cluster of CTAs takes each, every CTA
// selecting for itself (the scores are in L2) and moving a share of the rows.
// 1440 lists of up to 2048 f16 rows cut to 512 (194 MB read and written): 46 us, 4.2 TB/s.  The rows move at HBM's rate (29 us); what
// comes before is a chain of short phases (keys 8, border 5, places 4 us, over one round of CTAs and a part); q8_0 rows 40 us (17 at HBM's
// rate).  128, 192 and 512 threads,
// and fewer CTAs with more loads in flight, came out equal or slower.  Six lists of 300 rows: 5 us, latency (10 us when a bin of more than
// 96 keys took another histogram and the others were ranked a key at a time).
#include "kv_cache.cuh"
#include "row_lists.h"

#include <algorithm>

using namespace vox;

namespace {

constexpr int kThreads   = 256;
constexpr int kWarps     = kThreads / 32;
constexpr int kBits      = 11;
constexpr int kBins      = 1 << kBits;
constexpr int kRanked    = kThreads; // keys of a bin that are ranked against one another, one of a thread
constexpr int kMaxRows   = 49152;    // rows are numbered in 16 bits in the lists of moving rows
constexpr size_t kSmemMost = 200 * 1024;  // keys that fit stay in shared memory; those of longer row lists are made again
constexpr int kMaxCluster = 8;

struct EvictParams {
    uint8_t * k_data;
    uint8_t * v_data;
    size_t    c_nb_head, c_nb_stream, c_nb_layer;
    int       q8, layer0, n_kv_heads, n_streams, kv_bound, budget, n_sink, n_recent, n_list, keys_kept, cluster;
    const int32_t * kv_len;
    const int32_t * n_seen;
    uint8_t * score;
    uint8_t * row_pos;
    size_t    nb_head, nb_stream, nb_layer;
    int32_t * new_len;
    int32_t * kept;
    int *     status;
};

// f32 -> unsigned in the order of the numbers: -0 as 0, NaN lowest (0), every number between 1 and 2^32 - 2
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return isnan(x) ? 0u : b ^ ((uint32_t) ((int32_t) b >> 31) | 0x80000000u);
}
// The positions that are not protected: n_sink and `free_rows(..)` from there on, so that one comparison tells.
__device__ __forceinline__ uint32_t free_rows(int n_seen, int n_sink, int n_recent) {
    return (uint32_t) max(0LL, (long long) n_seen - n_recent - n_sink);
}
__device__ __forceinline__ uint32_t key_of_row(int pos, float score, int n_sink, uint32_t n_free) {
    return (uint32_t) pos - (uint32_t) n_sink < n_free ? ordered(score) : 0xffffffffu;
}
// four rows of scores and positions, wherever they lie; both come in vectors if every fourth row starts on 16 bytes
__device__ __forceinline__ bool in_vectors(const float * score, const int32_t * pos) {
    return ((reinterpret_cast<uintptr_t>(score) | reinterpret_cast<uintptr_t>(pos)) & 15) == 0;
}

// one of the eight 16-byte pieces of a q8_0 row: four of K, four of V; the first of either also takes its two scales
struct Q8Piece { uint4 bytes; uint32_t scales; };
__device__ __forceinline__ Q8Piece load_q8_piece(const uint8_t * pair, int row, int piece) {
    const uint8_t * a = pair + q8_tile_off(row);
    Q8Piece         x;
    x.bytes  = *reinterpret_cast<const uint4 *>(a + (piece & 4 ? kQ8VBytesOff : 0) + q8_byte_off(row, 16 * (piece & 3)));
    x.scales = (piece & 3) == 0 ? *reinterpret_cast<const uint32_t *>(a + (piece & 4 ? kQ8VScaleOff : kQ8KScaleOff) + q8_scale_off(row, 0)) : 0u;
    return x;
}
__device__ __forceinline__ void store_q8_piece(uint8_t * pair, int row, int piece, const Q8Piece & x) {
    uint8_t * b = pair + q8_tile_off(row);
    *reinterpret_cast<uint4 *>(b + (piece & 4 ? kQ8VBytesOff : 0) + q8_byte_off(row, 16 * (piece & 3))) = x.bytes;
    if ((piece & 3) == 0) *reinterpret_cast<uint32_t *>(b + (piece & 4 ? kQ8VScaleOff : kQ8KScaleOff) + q8_scale_off(row, 0)) = x.scales;
}

// Exclusive prefix sums over the block, and their total.  Two buffers of warp sums in turn, so that one barrier is enough.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t (*warp_sums)[kWarps], int & turn, uint32_t & total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t  incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    turn ^= 1;
    if (lane == 31) warp_sums[turn][warp] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const uint32_t s = warp_sums[turn][w];
        if (w < warp) before += s;
        all += s;
    }
    total = all;
    return before + incl - x;
}

__global__ void __launch_bounds__(kThreads, 7) evict_kernel(const EvictParams p) {
    extern __shared__ __align__(16) uint32_t smem[];  // keys (if they are kept), then sources and destinations of the rows that move
    __shared__ __align__(16) uint32_t hist[kBins];
    __shared__ uint32_t warp_sums[2][kWarps], found[3];
    uint32_t * const keys = smem;
    uint16_t * const src  = reinterpret_cast<uint16_t *>(smem + (p.keys_kept ? (p.kv_bound + 3) / 4 * 4 : 0)), * const dst = src + p.n_list;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int turn = 0, rank = 0, list = blockIdx.x;
    if (p.cluster > 1) {
        list = blockIdx.x / p.cluster;
        rank = blockIdx.x - list * p.cluster;
    }
    const int kvh = list % p.n_kv_heads, stream = (list / p.n_kv_heads) % p.n_streams, layer = list / (p.n_kv_heads * p.n_streams);
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int len = max(0, p.kv_len[stream]);
    const bool first = kvh == 0 && layer == 0 && rank == 0 && tid == 0;
    if (len > p.kv_bound) {
        if (first) { atomicOr(p.status, kStatusBadState); p.new_len[stream] = len; }
        return;
    }
    if (first) p.new_len[stream] = min(len, p.budget);
    int32_t * const kept = p.kept ? p.kept + (((size_t) layer * p.n_streams + stream) * p.n_kv_heads + kvh) * p.budget : nullptr;
    if (len <= p.budget) {
        if (kept && rank == 0) for (int j = tid; j < len; j += kThreads) kept[j] = j;
        return;
    }
    const size_t at = (size_t) layer * p.nb_layer + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head;
    float *   const score = reinterpret_cast<float *>(p.score + at);
    int32_t * const pos   = reinterpret_cast<int32_t *>(p.row_pos + at);
    const uint32_t n_free = free_rows(p.n_seen ? p.n_seen[stream] : len, p.n_sink, p.n_recent);
    auto make_key = [&](int j) { return key_of_row(pos[j], score[j], p.n_sink, n_free); };
    auto key_of = [&](int j) { return p.keys_kept ? keys[j] : make_key(j); };
    __syncthreads();
    int done = 0;
    if (p.keys_kept && in_vectors(score, pos)) {
        done = len & ~3;
#pragma unroll 2
        for (int j = 4 * tid; j < done; j += 4 * kThreads) {
            const int4   q = *reinterpret_cast<const int4 *>(pos + j);
            const float4 w = *reinterpret_cast<const float4 *>(score + j);
            const uint4  k = make_uint4(key_of_row(q.x, w.x, p.n_sink, n_free), key_of_row(q.y, w.y, p.n_sink, n_free),
                                        key_of_row(q.z, w.z, p.n_sink, n_free), key_of_row(q.w, w.w, p.n_sink, n_free));
            *reinterpret_cast<uint4 *>(keys + j) = k;
            atomicAdd(&hist[k.x >> (32 - kBits)], 1u);
            atomicAdd(&hist[k.y >> (32 - kBits)], 1u);
            atomicAdd(&hist[k.z >> (32 - kBits)], 1u);
            atomicAdd(&hist[k.w >> (32 - kBits)], 1u);
        }
    }
#pragma unroll 4
    for (int j = done + tid; j < len; j += kThreads) {
        const uint32_t k = make_key(j);
        if (p.keys_kept) keys[j] = k;
        atomicAdd(&hist[k >> (32 - kBits)], 1u);
    }
    __syncthreads();

    // The border: keys above `edge` stay, and of those equal to it the ones up to index `last`.
    uint32_t edge = 0, mask = 0;
    int      last = len, need = p.budget;
    for (int shift = 32 - kBits;;) {
        // the bin, from the top, in which the count reaches `need`
        constexpr int kPer = kBins / kThreads;  // (fewer bins: the others are zeros)
        static_assert(kPer == 8, "two vectors of a thread");
        const int bits = min(kBits, 32 - __popc(mask)), bins = 1 << bits, top = kBins - 1 - tid * kPer;
        const uint4 b0 = *reinterpret_cast<const uint4 *>(hist + top - 7), b1 = *reinterpret_cast<const uint4 *>(hist + top - 3);
        uint32_t  mine = (b0.x + b0.y) + (b0.z + b0.w) + (b1.x + b1.y) + (b1.z + b1.w), total;
        uint32_t before = block_scan(mine, warp_sums, turn, total);
        if (before < (uint32_t) need && before + mine >= (uint32_t) need) {
            int bin = top;
            while (before + hist[bin] < (uint32_t) need) before += hist[bin--];
            found[0] = (uint32_t) bin;
            found[1] = before;
            found[2] = hist[bin];
        }
        __syncthreads();
        edge |= found[0] << shift;
        mask |= (uint32_t) (bins - 1) << shift;
        need -= (int) found[1];
        const int n_bin = (int) found[2];
        if (shift == 0) {
            if (n_bin > need) {  // equal keys on both sides of the border: the first `need` of them stay
                __syncthreads();
                for (int j0 = 0, seen = 0; j0 < len && seen < need; j0 += 4 * kThreads) {
                    uint32_t count = 0, n;
#pragma unroll
                    for (int e = 0; e < 4; ++e) count += j0 + 4 * tid + e < len && key_of(j0 + 4 * tid + e) == edge ? 1u : 0u;
                    uint32_t r = seen + block_scan(count, warp_sums, turn, n);
                    if (r < (uint32_t) need && r + count >= (uint32_t) need) {
                        int j = j0 + 4 * tid;
                        for (;; ++j)
                            if (key_of(j) == edge && ++r == (uint32_t) need) break;
                        found[0] = (uint32_t) j;
                    }
                    seen += (int) n;
                }
                __syncthreads();
                last = (int) found[0];
            }
            break;
        }
        __syncthreads();
        if (n_bin <= kRanked) {  // rank the keys of the bin against one another; the histogram's memory holds them
            // a key, and of equal ones the lower index first, as one number; none is 0, which fills the last pair
            unsigned long long * const of_bin = reinterpret_cast<unsigned long long *>(hist);
            if (tid == 0) {
                found[2] = 0;
                of_bin[n_bin] = 0;
            }
            __syncthreads();
            for (int j = tid; j < len; j += kThreads) {
                const uint32_t k = key_of(j);
                if ((k & mask) == edge) {
                    const uint32_t i = atomicAdd(&found[2], 1u);
                    of_bin[i] = (unsigned long long) k << 32 | (0xffffffffu - (uint32_t) j);
                }
            }
            __syncthreads();
            if (tid < n_bin) {
                const unsigned long long own = of_bin[tid];
                int                      above = 0;
#pragma unroll 4
                for (int o = 0; o < n_bin; o += 2) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(of_bin + o);
                    above += (x.x > own) + (x.y > own);
                }
                if (above == need - 1) {  // the last one that stays
                    found[0] = (uint32_t) (own >> 32);
                    found[1] = 0xffffffffu - (uint32_t) own;
                }
            }
            __syncthreads();
            edge = found[0];
            last = (int) found[1];
            break;
        }
        const int next = max(0, shift - kBits), width = shift - next;
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += kThreads) {
            const uint32_t k = key_of(j);
            if ((k & mask) == edge) atomicAdd(&hist[(k >> next) & ((1u << width) - 1u)], 1u);
        }
        __syncthreads();
        shift = next;
    }

    // In index order: the places below the budget whose rows go, the rows above it that stay.  Four rows per thread.
    uint32_t marks = 0;  // places in the low half, rows in the high half
    for (int j0 = 0; j0 < len; j0 += 4 * kThreads) {
        const int j = j0 + 4 * tid;
        uint32_t  flags = 0, count = 0, n, four[4];
        if (p.keys_kept && j < len) {
            const uint4 x = *reinterpret_cast<const uint4 *>(keys + j);
            four[0] = x.x; four[1] = x.y; four[2] = x.z; four[3] = x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e >= len) continue;
            const uint32_t k = p.keys_kept ? four[e] : make_key(j + e);
            const bool     stays = k > edge || (k == edge && j + e <= last), low = j + e < p.budget;
            if (stays != low) {
                flags |= 1u << e;
                count += low ? 1u : 0x10000u;
            }
            if (kept && low && stays && rank == 0) kept[j + e] = j + e;
        }
        uint32_t mark = marks + block_scan(count, warp_sums, turn, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!(flags >> e & 1u)) continue;
            if (j + e < p.budget) {
                dst[mark & 0xffffu] = (uint16_t) (j + e);
                mark += 1u;
            } else {
                src[mark >> 16] = (uint16_t) (j + e);
                mark += 0x10000u;
            }
        }
        marks += n;
    }
    __syncthreads();
    if (p.cluster > 1) {  // every CTA of the cluster has read the scores and positions that are about to change
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    const int n_move = (int) (marks & 0xffffu);
    for (int i = rank * kThreads + tid; i < n_move; i += p.cluster * kThreads) {
        const int a = src[i], b = dst[i];
        score[b] = score[a];
        pos[b]   = pos[a];
        if (kept) kept[b] = a;
    }
    const size_t pair = (size_t) (p.layer0 + layer) * p.c_nb_layer + (size_t) stream * p.c_nb_stream + (size_t) kvh * p.c_nb_head;
    if (!p.q8) {  // 16 lanes a row: 8 x 16 bytes of K, 8 of V; four rows of a lane in flight
        uint8_t * const base = (lane & 8 ? p.v_data : p.k_data) + pair + (lane & 7) * 16;
        const int       pace = 2 * kWarps * p.cluster;
        constexpr int   U = 4;
        for (int i = 2 * (rank * kWarps + warp) + (lane >> 4); i < n_move; i += U * pace) {
            uint4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * pace < n_move) x[u] = *reinterpret_cast<const uint4 *>(base + (size_t) src[i + u * pace] * 128);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * pace < n_move) *reinterpret_cast<uint4 *>(base + (size_t) dst[i + u * pace] * 128) = x[u];
        }
    } else {      // 8 lanes a row
#pragma unroll 2
        for (int i = 4 * (rank * kWarps + warp) + (lane >> 3); i < n_move; i += 4 * kWarps * p.cluster) store_q8_piece(p.k_data + pair, dst[i], lane & 7, load_q8_piece(p.k_data + pair, src[i], lane & 7));
    }
}

// Few rows to give up (a stream that gains a row a step gives one up a step): no border is looked for, the rows that go are,
// one after the other, by reductions over the block.  They go in the order of their keys, of equal ones the highest
// index first, so the next is the least of those after the last.  1920 lists that give up one row of 1025: 10 us for 16.4 MB, bound by
// instructions and by the chain from the length to the row that moves (12 us before vectors and one comparison for protection).
constexpr int kFew        = 4;
constexpr int kFewThreads = 128;
static_assert(kFewThreads / 32 >= kFew, "a warp for each row behind the budget");
__global__ void __launch_bounds__(kFewThreads, 16) evict_few_kernel(const EvictParams p) {
    __shared__ uint32_t least_key[2][kFewThreads / 32];
    __shared__ int      least_row[2][kFewThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, list = blockIdx.x;
    const int kvh = list % p.n_kv_heads, stream = (list / p.n_kv_heads) % p.n_streams, layer = list / (p.n_kv_heads * p.n_streams);
    pdl_wait();
    pdl_launch_dependents();
    const int len = max(0, p.kv_len[stream]);
    const bool first = kvh == 0 && layer == 0 && tid == 0;
    if (len > p.kv_bound) {
        if (first) { atomicOr(p.status, kStatusBadState); p.new_len[stream] = len; }
        return;
    }
    if (first) p.new_len[stream] = min(len, p.budget);
    int32_t * const kept = p.kept ? p.kept + (((size_t) layer * p.n_streams + stream) * p.n_kv_heads + kvh) * p.budget : nullptr;
    const size_t at = (size_t) layer * p.nb_layer + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head;
    float *   const score = reinterpret_cast<float *>(p.score + at);
    int32_t * const pos   = reinterpret_cast<int32_t *>(p.row_pos + at);
    const uint32_t n_free = free_rows(p.n_seen ? p.n_seen[stream] : len, p.n_sink, p.n_recent);
    const int      n_go = len - p.budget;
    if (n_go <= 0) {
        if (kept) for (int j = tid; j < len; j += kFewThreads) kept[j] = j;
        return;
    }
    // the rows behind the budget are at most kFew: a warp asks for each, wherever it may have to go
    const size_t    pair = (size_t) (p.layer0 + layer) * p.c_nb_layer + (size_t) stream * p.c_nb_stream + (size_t) kvh * p.c_nb_head;
    uint8_t * const base = (lane & 8 ? p.v_data : p.k_data) + pair + (lane & 7) * 16;
    const int       from = p.budget + warp;
    Q8Piece         row = {};
    float           row_score = 0.0f;
    int             row_at = 0;
    if (warp < n_go) {
        if (lane == 31) {
            row_score = score[from];
            row_at    = pos[from];
        } else if (!p.q8 && lane < 16) {
            row.bytes = *reinterpret_cast<const uint4 *>(base + (size_t) from * 128);
        } else if (p.q8 && lane < 8) {
            row = load_q8_piece(p.k_data + pair, from, lane);
        }
    }
    const bool vectors = in_vectors(score, pos);
    int      gone[kFew];
    uint32_t last_key = 0;
    int      last_row = 0x7fffffff;
#pragma unroll
    for (int g = 0; g < kFew; ++g) {
        gone[g] = 0x7fffffff;
        if (g >= n_go) continue;
        uint32_t key = 0xffffffffu;
        int      at = -1;
        auto look = [&](int j, int q, float w) {  // of equal keys the last
            const uint32_t k = key_of_row(q, w, p.n_sink, n_free);
            const bool     later = g == 0 || k > last_key || (k == last_key && j < last_row);
            if (later && k <= key) { key = k; at = j; }
        };
        int done = 0;
        if (vectors) {
            done = len & ~3;
#pragma unroll 2
            for (int j = 4 * tid; j < done; j += 4 * kFewThreads) {
                const int4   q = *reinterpret_cast<const int4 *>(pos + j);
                const float4 w = *reinterpret_cast<const float4 *>(score + j);
                look(j, q.x, w.x);
                look(j + 1, q.y, w.y);
                look(j + 2, q.z, w.z);
                look(j + 3, q.w, w.w);
            }
        }
#pragma unroll 8
        for (int j = done + tid; j < len; j += kFewThreads) look(j, pos[j], score[j]);
        const uint32_t least = __reduce_min_sync(0xffffffffu, key);
        at = __reduce_max_sync(0xffffffffu, key == least ? at : -1);
        if (lane == 0) { least_key[g & 1][warp] = least; least_row[g & 1][warp] = at; }
        __syncthreads();
        key = least_key[g & 1][0];
        at  = least_row[g & 1][0];
#pragma unroll
        for (int o = 1; o < kFewThreads / 32; ++o) {
            const uint32_t k = least_key[g & 1][o];
            const int      r = least_row[g & 1][o];
            if (k < key || (k == key && r > at)) { key = k; at = r; }
        }
        last_key = key;
        last_row = at;
        gone[g]  = at;
    }
#pragma unroll
    for (int a = 0; a + 1 < kFew; ++a)  // by index
#pragma unroll
        for (int b = 0; b + 1 < kFew - a; ++b) {
            const int lo = min(gone[b], gone[b + 1]), hi = max(gone[b], gone[b + 1]);
            gone[b] = lo;
            gone[b + 1] = hi;
        }
    if (kept)
        for (int j = tid; j < p.budget; j += kFewThreads) kept[j] = j;
    __syncthreads();  // every thread has read the scores; and the rows that go are written over in `kept`
    if (warp >= n_go) return;
    // the i-th row behind the budget that stays moves to the i-th place below it whose row goes
    int nth = 0, to = p.budget;
#pragma unroll
    for (int i = 0; i < kFew; ++i) {
        if (gone[i] == from) return;
        if (p.budget + i < from) ++nth;
    }
#pragma unroll
    for (int i = 0; i < kFew; ++i)
        if (gone[i] >= p.budget && gone[i] < from) --nth;
#pragma unroll
    for (int i = 0; i < kFew; ++i)
        if (i == nth) to = gone[i];
    if (lane == 31) {
        score[to] = row_score;
        pos[to]   = row_at;
        if (kept) kept[to] = from;
    } else if (!p.q8 && lane < 16) {
        *reinterpret_cast<uint4 *>(base + (size_t) to * 128) = row.bytes;
    } else if (p.q8 && lane < 8) {
        store_q8_piece(p.k_data + pair, to, lane, row);
    }
}

int check_evict(const vox_engine * e, const vox_kv_evict_args * a) {
    VOX_REQUIRE(e && a && a->cache && a->score && a->row_pos && a->kv_len && a->new_len, VOX_ATTN_INVALID_ARGUMENT, "vox_kv_evict: null argument");
    const vox_kv_cache * c = a->cache;
    VOX_REQUIRE(c->e == e, VOX_ATTN_INVALID_ARGUMENT, "cache belongs to another engine");
    VOX_REQUIRE(a->n_layers > 0 && a->layer0 >= 0 && a->layer0 <= c->cfg.n_layers - a->n_layers, VOX_ATTN_INVALID_ARGUMENT,
                "layers %d .. %d out of range (cache holds %d)", a->layer0, a->layer0 + a->n_layers - 1, c->cfg.n_layers);
    VOX_REQUIRE(a->n_streams > 0 && a->n_streams <= c->cfg.n_streams, VOX_ATTN_INVALID_ARGUMENT, "n_streams %d out of range (cache holds %d)",
                a->n_streams, c->cfg.n_streams);
    VOX_REQUIRE(a->kv_bound >= 0 && a->kv_bound <= c->cfg.max_len, VOX_ATTN_INVALID_ARGUMENT, "kv_bound %d exceeds the cache capacity %d",
                a->kv_bound, c->cfg.max_len);
    VOX_REQUIRE(a->budget >= 1 && a->n_sink >= 0 && a->n_recent >= 0 && a->n_sink <= a->budget - a->n_recent, VOX_ATTN_INVALID_ARGUMENT,
                "budget %d must be positive and hold n_sink %d + n_recent %d", a->budget, a->n_sink, a->n_recent);
    for (const int32_t * in : {a->kv_len, a->n_seen})  // read by every CTA of the launch, while one of them writes new_len
        VOX_REQUIRE(in == nullptr || a->new_len + a->n_streams <= in || in + a->n_streams <= a->new_len, VOX_ATTN_INVALID_ARGUMENT,
                    "new_len must not overlap kv_len or n_seen");
    VOX_REQUIRE(a->kv_bound <= kMaxRows, VOX_ATTN_UNSUPPORTED, "kv_bound %d: at most %d rows a stream", a->kv_bound, kMaxRows);
    VOX_REQUIRE(((reinterpret_cast<uintptr_t>(a->score) | reinterpret_cast<uintptr_t>(a->row_pos) | reinterpret_cast<uintptr_t>(a->new_len) |
                  reinterpret_cast<uintptr_t>(a->kept)) & 3) == 0 && a->nb_head % 4 == 0 && a->nb_stream % 4 == 0 && a->nb_layer % 4 == 0,
                VOX_ATTN_INVALID_ARGUMENT, "score, row_pos, new_len and kept must be 4-byte aligned");
    const size_t row_bytes = (size_t) a->kv_bound * sizeof(float);
    const RowLists lists(a->score, row_bytes, {{c->cfg.n_kv_heads, a->nb_head}, {a->n_streams, a->nb_stream}, {a->n_layers, a->nb_layer}});
    VOX_REQUIRE(!lists.overlap(), VOX_ATTN_INVALID_ARGUMENT, "the scores of %d rows overlap (strides %zu, %zu, %zu bytes)", a->kv_bound, a->nb_head,
                a->nb_stream, a->nb_layer);
    VOX_REQUIRE(!lists.overlap_shifted(a->row_pos), VOX_ATTN_INVALID_ARGUMENT, "score and row_pos overlap");
    const RowLists positions(a->row_pos, row_bytes, {{c->cfg.n_kv_heads, a->nb_head}, {a->n_streams, a->nb_stream}, {a->n_layers, a->nb_layer}});
    const size_t lens_bytes = (size_t) a->n_streams * sizeof(int32_t);
    const size_t kept_bytes = a->kept ? (size_t) a->n_layers * a->n_streams * c->cfg.n_kv_heads * a->budget * sizeof(int32_t) : 0;
    for (const int32_t * x : {a->kv_len, a->n_seen, static_cast<const int32_t *>(a->new_len)}) {
        VOX_REQUIRE(!lists.meets(x, lens_bytes) && !positions.meets(x, lens_bytes), VOX_ATTN_INVALID_ARGUMENT,
                    "score and row_pos must not overlap kv_len, n_seen or new_len");
        VOX_REQUIRE(!ranges_meet(x, lens_bytes, a->kept, kept_bytes), VOX_ATTN_INVALID_ARGUMENT, "kept must not overlap kv_len, n_seen or new_len");
    }
    VOX_REQUIRE(!lists.meets(a->kept, kept_bytes) && !positions.meets(a->kept, kept_bytes), VOX_ATTN_INVALID_ARGUMENT,
                "kept must not overlap score or row_pos");
    VOX_REQUIRE((long long) a->n_layers * a->n_streams * c->cfg.n_kv_heads < (1LL << 31), VOX_ATTN_UNSUPPORTED, "more than 2^31 row lists in one call");
    return VOX_ATTN_OK;
}

}  // namespace

extern "C" int vox_kv_evict(vox_engine * e, const vox_kv_evict_args * a, void * stream) {
    const int rc = check_evict(e, a);
    if (rc != VOX_ATTN_OK) return rc;
    int current = -1;
    VOX_CUDA_TRY(cudaGetDevice(&current));
    VOX_REQUIRE(current == e->device, VOX_ATTN_INVALID_ARGUMENT, "the engine's device %d must be the current device (current is %d)", e->device, current);
    vox_kv_cache * c = a->cache;
    EvictParams    p;
    p.k_data = c->k_data; p.v_data = c->v_data;
    p.c_nb_head = c->nb_head; p.c_nb_stream = c->nb_stream; p.c_nb_layer = c->nb_layer;
    p.q8 = c->cfg.type == VOX_TYPE_Q8_0;
    p.layer0 = a->layer0; p.n_kv_heads = c->cfg.n_kv_heads; p.n_streams = a->n_streams;
    p.kv_bound = a->kv_bound; p.budget = a->budget; p.n_sink = a->n_sink; p.n_recent = a->n_recent;
    p.n_list = std::max(1, std::min(a->budget, a->kv_bound - a->budget));  // rows that can move
    p.kv_len = a->kv_len; p.n_seen = a->n_seen;
    p.score = reinterpret_cast<uint8_t *>(a->score); p.row_pos = reinterpret_cast<uint8_t *>(a->row_pos);
    p.nb_head = a->nb_head; p.nb_stream = a->nb_stream; p.nb_layer = a->nb_layer;
    p.new_len = a->new_len; p.kept = a->kept; p.status = e->status_dev;
    if (a->kv_bound - a->budget <= kFew) {
        launch_pdl(evict_few_kernel, dim3((unsigned) (a->n_layers * a->n_streams * p.n_kv_heads)), dim3(kFewThreads), 0, static_cast<cudaStream_t>(stream), p);
        return check_launch(e, "evict_few_kernel");
    }
    const size_t    key_bytes = (size_t) (a->kv_bound + 3) / 4 * 16, list_bytes = (size_t) 2 * p.n_list * sizeof(uint16_t);
    p.keys_kept = key_bytes + list_bytes <= kSmemMost;
    const size_t    smem  = (p.keys_kept ? key_bytes : 0) + list_bytes;
    const long long lists = (long long) a->n_layers * a->n_streams * p.n_kv_heads;
    // few lists: as many CTAs to a list as give every SM two, if the rows that may move are enough to share
    p.cluster = (int) std::max(1LL, std::min<long long>(std::min<long long>(kMaxCluster, 2LL * e->sm_count / lists), p.n_list / 64));
    const uint32_t bit = 1u << 20;
    if (!(e->attr_mask & bit)) {
        VOX_CUDA_TRY(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) kSmemMost));
        e->attr_mask |= bit;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (lists * p.cluster)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned) p.cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, evict_kernel, p);
    return check_launch(e, "evict_kernel");
}
