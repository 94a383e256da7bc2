// Eviction from the cache by accumulated attention weight (vox_kv_evict).
//
// Per (layer, stream, kv head) with more rows than the budget: the `budget` largest keys stay (a key orders the rows as the
// contract does: protected rows above every score, scores as numbers, NaN below), found by a radix select over the keys;
// then the i-th kept row at or above the budget moves to the i-th place below it whose row goes.  Sources and
// destinations never overlap, so rows move in place and in any order.
#include "kv_cache.cuh"

#include <algorithm>

using namespace vox;

namespace {

constexpr int kThreads  = 512;
constexpr int kMaxRows  = 49152;   // the two lists of moving rows fit shared memory up to here

struct EvictParams {
    uint8_t * k_data;
    uint8_t * v_data;
    size_t    c_nb_head, c_nb_stream, c_nb_layer;
    int       q8, layer0, n_kv_heads, n_streams, kv_bound, budget, n_sink, n_recent, n_list;
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
    if (isnan(x)) return 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// exclusive prefix sums over the block of two counts packed in one word, and their total
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t * warp_sums, uint32_t & total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t  incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        const uint32_t s = warp_sums[w];
        if (w < warp) before += s;
        all += s;
    }
    total = all;
    return before + incl - x;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(const EvictParams p) {
    extern __shared__ int32_t lists[];  // sources, then destinations
    __shared__ uint32_t hist[256], warp_sums[kThreads / 32], chosen[2];
    int32_t * const src = lists, * const dst = lists + p.n_list;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.x % p.n_kv_heads, stream = (blockIdx.x / p.n_kv_heads) % p.n_streams, layer = blockIdx.x / (p.n_kv_heads * p.n_streams);
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
    if (len <= p.budget) {
        if (kept) for (int j = tid; j < len; j += kThreads) kept[j] = j;
        return;
    }
    const size_t at = (size_t) layer * p.nb_layer + (size_t) stream * p.nb_stream + (size_t) kvh * p.nb_head;
    float *   const score = reinterpret_cast<float *>(p.score + at);
    int32_t * const pos   = reinterpret_cast<int32_t *>(p.row_pos + at);
    const int recent = (p.n_seen ? p.n_seen[stream] : len) - p.n_recent;
    auto key_of = [&](int j) {
        const int q = pos[j];
        return q < p.n_sink || q >= recent ? 0xffffffffu : ordered(score[j]);
    };
    // radix select: the largest keys' common byte prefix, a byte per pass; `need` of the keys that match it so far stay
    uint32_t prefix = 0, mask = 0;
    int      need   = p.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += kThreads) {
            const uint32_t k = key_of(j);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (warp == 0) {  // the bin, from the top, in which the count reaches `need`
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine += hist[255 - 8 * lane - i];
            uint32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            uint32_t before = incl - mine;
            if (before < (uint32_t) need && incl >= (uint32_t) need) {
                int bin = 255 - 8 * lane;
                while (before + hist[bin] < (uint32_t) need) before += hist[bin--];
                chosen[0] = (uint32_t) bin;
                chosen[1] = before;
            }
        }
        __syncthreads();
        prefix |= chosen[0] << shift;
        mask   |= 0xffu << shift;
        need   -= (int) chosen[1];
        __syncthreads();
    }
    // rows above the key `prefix` stay, and the first `need` that have it.  In index order: the places below the budget
    // whose rows go, the rows above it that stay
    uint32_t ties = 0, lists_n = 0;  // lists_n: holes in the low half, movers in the high half (both below 2^16)
    for (int j0 = 0; j0 < len; j0 += kThreads) {
        const int      j = j0 + tid;
        const uint32_t k = j < len ? key_of(j) : 0u;
        const bool     tie = j < len && k == prefix;
        uint32_t       n_tie, n_list;
        const uint32_t rank = ties + block_scan(tie ? 1u : 0u, warp_sums, n_tie);
        const bool     keep = j < len && (k > prefix || (tie && rank < (uint32_t) need));
        const bool     hole = j < p.budget && !keep, mover = j >= p.budget && keep;
        const uint32_t mark = lists_n + block_scan((hole ? 1u : 0u) | (mover ? 0x10000u : 0u), warp_sums, n_list);
        if (hole) dst[mark & 0xffffu] = j;
        if (mover) src[mark >> 16] = j;
        if (kept && j < p.budget && keep) kept[j] = j;
        ties += n_tie;
        lists_n += n_list;
    }
    __syncthreads();
    const int n_move = (int) (lists_n & 0xffffu);
    for (int i = tid; i < n_move; i += kThreads) {
        const int a = src[i], b = dst[i];
        score[b] = score[a];
        pos[b]   = pos[a];
        if (kept) kept[b] = a;
    }
    const size_t pair = (size_t) (p.layer0 + layer) * p.c_nb_layer + (size_t) stream * p.c_nb_stream + (size_t) kvh * p.c_nb_head;
    if (!p.q8) {  // 16 lanes a row: 8 x 16 bytes of K, 8 of V
        uint8_t * const base = (lane & 8 ? p.v_data : p.k_data) + pair + (lane & 7) * 16;
        for (int i = 2 * warp + (lane >> 4); i < n_move; i += 2 * (kThreads / 32))
            *reinterpret_cast<uint4 *>(base + (size_t) dst[i] * 128) = *reinterpret_cast<const uint4 *>(base + (size_t) src[i] * 128);
    } else {      // 8 lanes a row: 4 x 16 bytes of K, 4 of V; the first of either also takes its two scales
        const int      piece = lane & 3;
        const uint32_t bytes = lane & 4 ? kQ8VBytesOff : 0, scales = lane & 4 ? kQ8VScaleOff : kQ8KScaleOff;
        for (int i = 4 * warp + (lane >> 3); i < n_move; i += 4 * (kThreads / 32)) {
            const uint8_t * a = p.k_data + pair + q8_tile_off(src[i]);
            uint8_t *       b = p.k_data + pair + q8_tile_off(dst[i]);
            *reinterpret_cast<uint4 *>(b + bytes + q8_byte_off(dst[i], 16 * piece)) =
                *reinterpret_cast<const uint4 *>(a + bytes + q8_byte_off(src[i], 16 * piece));
            if (piece == 0)
                *reinterpret_cast<uint32_t *>(b + scales + q8_scale_off(dst[i], 0)) = *reinterpret_cast<const uint32_t *>(a + scales + q8_scale_off(src[i], 0));
        }
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
    VOX_REQUIRE(a->new_len != a->kv_len, VOX_ATTN_INVALID_ARGUMENT, "new_len must not be kv_len itself");
    VOX_REQUIRE(a->kv_bound <= kMaxRows, VOX_ATTN_UNSUPPORTED, "kv_bound %d: at most %d rows a stream", a->kv_bound, kMaxRows);
    VOX_REQUIRE(((reinterpret_cast<uintptr_t>(a->score) | reinterpret_cast<uintptr_t>(a->row_pos) | reinterpret_cast<uintptr_t>(a->new_len) |
                  reinterpret_cast<uintptr_t>(a->kept)) & 3) == 0 && a->nb_head % 4 == 0 && a->nb_stream % 4 == 0 && a->nb_layer % 4 == 0,
                VOX_ATTN_INVALID_ARGUMENT, "score, row_pos, new_len and kept must be 4-byte aligned");
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
    const size_t   smem = (size_t) 2 * p.n_list * sizeof(int32_t);
    const uint32_t bit  = 1u << 20;
    if (!(e->attr_mask & bit)) {
        VOX_CUDA_TRY(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxRows / 2) * 2 * (int) sizeof(int32_t)));
        e->attr_mask |= bit;
    }
    launch_pdl(evict_kernel, dim3((unsigned) (a->n_layers * a->n_streams * p.n_kv_heads)), dim3(kThreads), smem, static_cast<cudaStream_t>(stream), p);
    return check_launch(e, "evict_kernel");
}
