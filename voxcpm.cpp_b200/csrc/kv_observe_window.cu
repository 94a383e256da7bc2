// The attention weight that every cache row receives from a window of queries (vox_kv_observe with n_q > 1), on the
// 5th-generation tensor cores.
//
//   score[j] += sum over rows r = (query, head) of 2^(s[r][j] - M[r]) / L[r],    s = scale * log2 e * q.k
//
// Two launches over the same cut of the work: the first finds every row's (max, sum) over a part of the keys, the second joins
// them over the parts and adds up the weights.  A score is needed in both, and making it again (2 * 64 products) costs less than
// 4 bytes through HBM and back would.  No P.V follows, so the tensor core's share is small and what bounds both launches is the
// exponentials: one per score and launch, 16 per clock and SM.
//   - the first launch takes the queries as rows (a thread per query row and 64 keys at a time: maximum and sum stay in the
//     thread), the second the keys (a thread per key and 64 query rows at a time: the sum over rows stays in the thread), so
//     neither reduces anything across threads; the operands are the same tiles in shared memory, A and B exchanged;
//   - the queries of a pair (at most 64 x 8 rows) are turned into two f16 tiles, value and remainder, once per CTA;
//   - q8_0 rows become f16 numbers q (exact) by two warps of their own; either 32-value block has its own accumulator and the
//     scales are applied in f32.
// 8 streams of up to 8192 rows, 64 queries: 45.7 us, of which the exponentials alone are 18.7 us (2 x 42 M) and the two launches'
// prologues (dependency wait, cut, queries, first tiles) about 6 us each; two groups of warps instead of four, 50.0 us.  16 q8_0
// streams of 2000 rows, 32 queries: 28.7 us.  (A part of the exponentials by a polynomial on the FMA units changed nothing or cost
// time: 44.9 / 45.8 / 48.8 us for a sixteenth / an eighth / a quarter of them.)
// The work is cut on the device from the lengths as they are: every (stream, kv head) into nearly equal parts of at most r
// 128-key tiles, r the smallest for which the parts are no more than the CTAs.  No atomics, every sum in one fixed order.
#include "kv_observe.cuh"
#include "tcgen05.cuh"

using namespace vox;

namespace {

constexpr int kKeys     = 128;                  // keys of a tile
constexpr int kSub      = 64;                   // columns of a score tile
constexpr int kMaxRows  = kObserveMaxQ * 8;
constexpr int kQTile    = kMaxRows * 128;       // the queries' f16 values; their remainders behind
constexpr int kKTile    = kKeys * 128;
constexpr int kRawStage = 2 * (kKvTile * 64 + kKvTile * 4);  // q8_0: bytes and scales of 128 rows of K
constexpr int kRawStages = 4;
constexpr int kGroups   = 4;                    // groups of four warps that take score tiles
constexpr int kTakers   = kGroups * 128;
static_assert(kMaxRows == kTakers, "a thread joins the statistics of one row");
template <bool Q8> struct Shape {
    static constexpr int kStages  = Q8 ? 2 : 4;    // f16 tiles of K
    static constexpr int kThreads = kTakers + (Q8 ? 4 : 2) * 32;
    static constexpr int kCols    = Q8 ? 2 * kSub : kSub;  // TMEM columns of a score tile: q8_0 has an accumulator per block
    static constexpr int kBufs    = 512 / kCols;
    static constexpr int kSmem    = 2 * kQTile + kStages * kKTile + (Q8 ? kRawStages * kRawStage : 0) + 1024;
};

struct Part {
    int stream, kvh, len, tile0, tiles, first_slot, slots;  // tiles of this part; the slots of the pair's statistics
    int parts;                                              // of the whole cut
};

// Part `b` of the cut, by one warp (each lane holds the tile counts of every 32nd stream); false past the last part.
__device__ __forceinline__ int tiles_of(const ObserveParams & p, int s) {
    const int len = p.kv_len[s];
    return len > p.kv_bound || len <= 0 ? 0 : (len + kKeys - 1) / kKeys;
}
__device__ bool find_part(const ObserveParams & p, int b, int n_ctas, Part & w) {
    const int lane = threadIdx.x & 31, n = p.n_streams, HK = p.n_kv_heads, rounds = (n + 31) / 32;
    int total = 0, live = 0, most = 0;
    for (int i = 0; i < rounds; ++i) {
        const int t = 32 * i + lane < n ? tiles_of(p, 32 * i + lane) : 0;
        total += t;
        live += t > 0;
        most = max(most, t);
    }
    total = __reduce_add_sync(0xffffffffu, total) * HK;
    live  = __reduce_add_sync(0xffffffffu, live) * HK;
    most  = __reduce_max_sync(0xffffffffu, most);
    if (total == 0) return false;
    int r = live >= n_ctas ? most : (total + n_ctas - 1) / n_ctas;
    w.parts = live;  // r == most
    for (; r < most; ++r) {
        int parts = 0;
        for (int i = 0; i < rounds; ++i) parts += 32 * i + lane < n ? (tiles_of(p, 32 * i + lane) + r - 1) / r : 0;
        parts = __reduce_add_sync(0xffffffffu, parts) * HK;
        if (parts <= n_ctas) { w.parts = parts; break; }
    }
    int before = 0;  // parts of the streams before this round's
    for (int i = 0; i < rounds; ++i) {
        const int s = 32 * i + lane, t = s < n ? tiles_of(p, s) : 0, np = (t + r - 1) / r;
        int       incl = np;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const int      lo = (before + incl - np) * HK, hi = (before + incl) * HK;
        const unsigned owner = __ballot_sync(0xffffffffu, b >= lo && b < hi);
        if (owner != 0) {
            const int src = __ffs(owner) - 1;
            const int s0 = __shfl_sync(0xffffffffu, s, src), t0 = __shfl_sync(0xffffffffu, t, src), n0 = __shfl_sync(0xffffffffu, np, src),
                      lo0 = __shfl_sync(0xffffffffu, lo, src);
            const int j = (b - lo0) % n0;
            w.stream = s0;
            w.kvh    = (b - lo0) / n0;
            w.len    = p.kv_len[s0];
            w.tile0  = j * t0 / n0;
            w.tiles  = (j + 1) * t0 / n0 - w.tile0;
            w.first_slot = b - j;
            w.slots  = n0;
            return true;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

template <bool Q8, bool kWeights>
__global__ void __launch_bounds__(Shape<Q8>::kThreads, 1)
observe_window_kernel(const __grid_constant__ CUtensorMap map_k, const ObserveParams p) {
    using Z = Shape<Q8>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * Z::kStages + 2 * kRawStages + 2 * Z::kBufs];
    __shared__ uint32_t tmem_slot;
    __shared__ int      abort_flag, have_part;
    __shared__ Part     part;
    __shared__ __align__(16) float2 row_stat[kMaxRows];         // kWeights: (max, 1 / sum); otherwise what the second group found
    __shared__ float2   scales[Z::kStages][kKeys];  // q8_0: of the f16 tile of a stage
    __shared__ float    group_sum[2][kGroups][kKeys];  // kWeights: the groups' sums of a key tile (two buffers in turn)
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *      smem_gen  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t sQ = smem_base, sK = sQ + 2 * kQTile, sRaw = sK + Z::kStages * kKTile;
    const int      tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int  kCopyWarp = kTakers / 32, kIssueWarp = kCopyWarp + 1;  // behind them the converting warps
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = full0 + 8 * Z::kStages, rfull0 = empty0 + 8 * Z::kStages, rempty0 = rfull0 + 8 * kRawStages,
                   bS0 = rempty0 + 8 * kRawStages, bE0 = bS0 + 8 * Z::kBufs;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < Z::kStages; ++s) {
            mbar_init(full0 + 8 * s, Q8 ? 2 : 1);  // the converting warps, or the copy
            mbar_init(empty0 + 8 * s, Q8 ? 1 + kTakers / 32 : 1);  // the products have retired (and the warps that read the scales are done)
        }
        for (int s = 0; s < kRawStages; ++s) {
            mbar_init(rfull0 + 8 * s, 1);
            mbar_init(rempty0 + 8 * s, 2);
        }
        for (int s = 0; s < Z::kBufs; ++s) {
            mbar_init(bS0 + 8 * s, 1);
            mbar_init(bE0 + 8 * s, 4);  // the four warps that take the score tile
        }
        fence_mbar_init();
    }
    if (warp == kIssueWarp) tmem_alloc(smem_u32(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // The second launch reads one thing that the first has written, the statistics: it waits for it when its queries are ready.
    // (All else it reads was there before the first launch began, and that one has begun.)
    bool waits = kWeights;
    if (!kWeights) {
        pdl_wait();
        pdl_launch_dependents();
    }
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_slot);
    // A group of warps takes every fourth score tile or more (q8_0, first launch: three blocks of 128 rows count as four): a tile's wait
    // tells it from the one before it in the same buffer only if the group has taken one of the kBufs tiles in between.
    const int rows = p.n_q * p.gqa, n_b = (rows + kSub - 1) / kSub, blocks = (rows + 127) / 128;
    const int n_m = Q8 && !kWeights && blocks == 3 ? 4 : blocks;
    static_assert(Z::kBufs >= kGroups && (Q8 || Z::kBufs >= 2 * kMaxRows / 128), "see above");
    const int per_tile = kWeights ? n_b : 2 * n_m;  // score tiles per key tile
    auto give_up = [&]() {
        atomicOr(p.status, kStatusTimeout);
        atomicExch(&abort_flag, 1);
    };
    auto aborted   = [&]() { return *reinterpret_cast<volatile int *>(&abort_flag) != 0; };
    auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity)) != 0; };
    if (!kWeights && blockIdx.x == 0 && warp == 1)  // a stream longer than the call said is left alone
        for (int s = lane; s < p.n_streams; s += 32)
            if (p.kv_len[s] > p.kv_bound) atomicOr(p.status, kStatusBadState);
    int issued = 0;    // copies of key tiles, by the warp that issues them
    int T = 0, U = 0;  // key tiles and score tiles so far, over all parts of this CTA: they fix the phase of every barrier

    for (int b = blockIdx.x, n_parts = 0x7fffffff; b < n_parts; b += gridDim.x) {
        if (warp == 0) {
            Part      w{};
            const bool have = find_part(p, b, gridDim.x, w);
            if (lane == 0) { part = w; have_part = have && !aborted(); }
        }
        __syncthreads();
        if (!have_part) break;
        const Part w = part;
        n_parts = w.parts;

        auto copy_tile = [&](int t) {  // one lane
            const int n = T + t, key = (w.tile0 + t) * kKeys, boxes = w.len - key > kKvTile ? 2 : 1;
            if constexpr (Q8) {
                const int st = n % kRawStages;
                issued = n;
                if (n >= kRawStages && !mbar_wait_bounded(rempty0 + 8 * st, ((n / kRawStages) - 1) & 1)) return false;
                const uint32_t bar = rfull0 + 8 * st, dst = sRaw + st * kRawStage;
                mbar_expect_tx(bar, boxes * (kRawStage / 2));
                for (int x = 0; x < boxes; ++x) {
                    const uint8_t * src = p.k + (size_t) w.stream * p.k_nb_stream + (size_t) w.kvh * p.k_nb_head + q8_tile_off(key + x * kKvTile);
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst + x * kKvTile * 64),
                                 "l"(src), "r"(kKvTile * 64), "r"(bar)
                                 : "memory");
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst + 2 * kKvTile * 64 + x * kKvTile * 4),
                                 "l"(src + kQ8KScaleOff), "r"(kKvTile * 4), "r"(bar)
                                 : "memory");
                }
            } else {
                const int st = n % Z::kStages;
                issued = n;
                if (n >= Z::kStages && !mbar_wait_bounded(empty0 + 8 * st, ((n / Z::kStages) - 1) & 1)) return false;
                const uint32_t bar = full0 + 8 * st, dst = sK + st * kKTile;
                mbar_expect_tx(bar, boxes * kKvTile * 128);
                for (int x = 0; x < boxes; ++x) tma_load_5d(dst + x * kKvTile * 128, &map_k, bar, 0, key + x * kKvTile, w.kvh, w.stream, p.layer);
            }
            return true;
        };
        bool first_ok = true;
        if (warp == kCopyWarp && lane == 0)  // the first two while the queries are made ready
            for (int t = 0; t < min(w.tiles, 2) && first_ok; ++t) first_ok = copy_tile(t);

        // ---- the queries of the pair, by the warps that will take score tiles; in the second launch their statistics too
        if (warp < kCopyWarp) {
            const int       c = lane & 15, n_rows = n_m * 128;
            const uint8_t * q_base = p.q + (size_t) w.stream * p.q_nb_stream + (size_t) (w.kvh * p.gqa) * p.q_nb_head + 16 * c;
            constexpr int kLoads = 8;  // rows of a lane in flight
#pragma unroll 1
            for (int r0 = 2 * warp * kLoads; r0 < n_rows; r0 += kTakers / 16 * kLoads) {
                float4 x[kLoads];
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const uint32_t row = r0 + 2 * i + (lane >> 4), at = min(row, (uint32_t) rows - 1), q = at * p.gqa_magic >> 16;  // at / gqa
                    const uint8_t * src = q_base + q * p.q_nb_tok + (at - q * p.gqa) * p.q_nb_head;
                    const float2 lo = *reinterpret_cast<const float2 *>(src), hi = *reinterpret_cast<const float2 *>(src + 8);
                    x[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int     row = r0 + 2 * i + (lane >> 4);
                    const float   mul = p.scale_log2;
                    const __half2 h0 = __floats2half2_rn(x[i].x * mul, x[i].y * mul), h1 = __floats2half2_rn(x[i].z * mul, x[i].w * mul);
                    const float2  f0 = __half22float2(h0), f1 = __half22float2(h1);
                    uint2 hi = make_uint2(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1));
                    uint2 lo = make_uint2(pack_half2(x[i].x * mul - f0.x, x[i].y * mul - f0.y), pack_half2(x[i].z * mul - f1.x, x[i].w * mul - f1.y));
                    if (row >= rows) hi = lo = make_uint2(0u, 0u);
                    uint8_t * dst = smem_gen + row * 128 + (((c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8;
                    *reinterpret_cast<uint2 *>(dst)          = hi;
                    *reinterpret_cast<uint2 *>(dst + kQTile) = lo;
                }
            }
            fence_proxy_async_smem();
        }
        if (kWeights) {
            if (waits) {
                pdl_wait();
                pdl_launch_dependents();
                waits = false;
            }
            if (warp < kCopyWarp) {  // the rows' statistics: a row of a thread, eight parts in flight
                constexpr int  kParts = 8;
                const float2 * all = p.stats + (size_t) w.first_slot * rows + tid;
                float          M = -INFINITY, L = 0.0f;
                if (tid < rows)
                    for (int s0 = 0; s0 < w.slots; s0 += kParts) {
                        float2 x[kParts];
#pragma unroll
                        for (int s = 0; s < kParts; ++s) x[s] = s0 + s < w.slots ? __ldcg(all + (size_t) (s0 + s) * rows) : make_float2(-INFINITY, 0.0f);
                        float most = M;
#pragma unroll
                        for (int s = 0; s < kParts; ++s) most = fmaxf(most, x[s].x);
                        if (M != -INFINITY) L *= exp2f(M - most);
                        M = most;
#pragma unroll
                        for (int s = 0; s < kParts; ++s) L = fmaf(x[s].y, x[s].x == -INFINITY ? (x[s].y == 0.0f ? 0.0f : 1.0f) : exp2f(x[s].x - most), L);
                    }
                row_stat[tid] = L == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(M, 1.0f / L);  // a row that sees nothing adds nothing
            }
        }
        __syncthreads();

        if (warp == kCopyWarp) {
            // ------------------------------------------------------------------ copies
            if (lane == 0) {
                bool ok = first_ok;
                for (int t = min(w.tiles, 2); t < w.tiles && ok; ++t) ok = copy_tile(t);
                if (ok) issued = T + w.tiles;
                else    give_up();
            }
            __syncwarp();
        } else if (warp == kIssueWarp) {
            // ------------------------------------------------------------------ products (all lanes in the loop, one issues)
            constexpr uint32_t idesc = idesc_f16(kSub, false);
            const uint64_t     dQ = smem_desc_sw128(sQ), dK = smem_desc_sw128(sK);
            constexpr uint64_t kLo = kQTile >> 4;
            const bool         leader = elect_one();
            bool               ok = true;
            int                u = U;
            for (int t = 0; t < w.tiles && ok; ++t) {
                const int n = T + t, st = n % Z::kStages;
                if (!warp_wait(full0 + 8 * st, (n / Z::kStages) & 1)) { ok = false; break; }
                const uint64_t k0 = dK + (uint64_t) (st * (kKTile >> 4));
                for (int i = 0; i < per_tile; ++i, ++u) {
                    const int sb = u % Z::kBufs;
                    if (u >= Z::kBufs && !warp_wait(bE0 + 8 * sb, ((u / Z::kBufs) - 1) & 1)) { ok = false; break; }
                    tc_fence_after();
                    if (leader) {
                        const uint32_t dS = tmem + Z::kCols * sb;
                        // first launch: A = 128 query rows (i / 2), B = 64 keys (i % 2); second: A = 128 keys, B = 64 query rows (i)
                        const uint64_t q0 = dQ + (uint64_t) (kWeights ? i * ((kSub * 128) >> 4) : (i >> 1) * ((128 * 128) >> 4));
                        const uint64_t kh = kWeights ? k0 : k0 + (uint64_t) ((i & 1) * ((kSub * 128) >> 4));
#pragma unroll
                        for (int part_q = 1; part_q >= 0; --part_q)  // the remainders' products first: the accumulator truncates
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint64_t q = q0 + part_q * kLo + k * 2, x = kh + k * 2;
                                const uint32_t d = Q8 ? dS + (k >> 1) * kSub : dS;
                                tc_mma_f16(d, kWeights ? x : q, kWeights ? q : x, idesc, part_q == 0 || (Q8 ? (k & 1) : k) != 0);
                            }
                        tc_commit(bS0 + 8 * sb);
                        if (i == per_tile - 1) tc_commit(empty0 + 8 * st);
                    }
                    __syncwarp();
                }
            }
            if (!ok && lane == 0) give_up();
        } else if (warp < kCopyWarp) {
            // ------------------------------------------------------------------ scores out, by groups of four warps.  First launch:
            // group g has half g % 2 of a tile's keys and every other 128 query rows from g / 2 on; second: every fourth score tile.
            const int      group = warp >> 2, row = tid & 127, first_cut = w.len - p.n_q;  // first key that not every query sees
            const uint32_t t_row = tmem + ((uint32_t) (32 * (warp & 3)) << 16);
            constexpr int  kMine = kMaxRows / 256;
            bool           ok = true;
            int            u = U;
            float          m[kMine], l[kMine];
            if (!kWeights) {
#pragma unroll
                for (int i = 0; i < kMine; ++i) { m[i] = -INFINITY; l[i] = 0.0f; }
            }
            for (int t = 0; t < w.tiles && ok; ++t) {
                const int n = T + t, st = n % Z::kStages, key0 = (w.tile0 + t) * kKeys, key = key0 + row;
                float     sum = 0.0f, d0 = 1.0f, d1 = 1.0f, old = 0.0f;
                float *   score = nullptr;
                if (Q8) {  // the scales are the converting warps'
                    // (a warp whose wait ran out stays until the barrier at the end of the tile, which the others wait at)
                    if (!mbar_wait_bounded(full0 + 8 * st, (n / Z::kStages) & 1)) ok = false;
                    if (kWeights) { d0 = scales[st][row].x; d1 = scales[st][row].y; }
                }
                const bool mine = kWeights && group == (t & (kGroups - 1)) && key < w.len, fresh = key >= w.len - p.n_new;  // who writes this tile's scores
                if (mine) {
                    score = reinterpret_cast<float *>(p.score + (size_t) w.stream * p.nb_stream + (size_t) w.kvh * p.nb_head) + key;
                    if (!fresh) old = *score;
                }
                auto take = [&](int uu) {  // a score tile is there
                    if (!mbar_wait_bounded(bS0 + 8 * (uu % Z::kBufs), (uu / Z::kBufs) & 1)) return false;
                    tc_fence_after();
                    return true;
                };
                auto give_back = [&](int uu) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bE0 + 8 * (uu % Z::kBufs));
                };
                if constexpr (!kWeights) {
                    constexpr int kCols = Q8 ? 32 : kSub;  // scores at a time
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        const int mt = 2 * i + (group >> 1), uu = u + 2 * mt + (group & 1), k0 = key0 + kSub * (group & 1);
                        if (mt >= n_m || !ok) break;
                        if (!take(uu)) { ok = false; break; }
#pragma unroll
                        for (int h = 0; h < kSub; h += kCols) {
                            uint32_t r[kCols];
                            if constexpr (Q8) {
                                uint32_t x[32];
                                tmem_ld32_sync(t_row + Z::kCols * (uu % Z::kBufs) + h, r);
                                tmem_ld32_sync(t_row + Z::kCols * (uu % Z::kBufs) + kSub + h, x);
                                const float2 * ds = scales[st] + kSub * (group & 1) + h;
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const float2 d = ds[e];
                                    r[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), d.y, __uint_as_float(r[e]) * d.x));
                                }
                            } else {
                                tmem_ld64_sync(t_row + Z::kCols * (uu % Z::kBufs), r);
                            }
                            if (h + kCols == kSub) give_back(uu);
                            if (k0 + kSub > first_cut) {  // keys that this row's query does not see, and keys past the end
                                const int last = first_cut + (int) ((uint32_t) (128 * mt + row) * p.gqa_magic >> 16) - k0 - h;
#pragma unroll
                                for (int e = 0; e < kCols; ++e)
                                    if (e > last) r[e] = 0xff800000u;
                            }
                            float t0 = m[i], t1 = -INFINITY;
#pragma unroll
                            for (int e = 0; e < kCols; e += 4) {
                                t0 = max3(t0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
                                t1 = max3(t1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
                            }
                            const float mn = fmaxf(t0, t1), ref = mn == -INFINITY ? 0.0f : mn;
                            float s0 = m[i] == -INFINITY ? l[i] : l[i] * ex2_approx(m[i] - ref), s1 = 0.0f;
#pragma unroll
                            for (int e = 0; e < kCols; e += 2) {
                                s0 += ex2_approx(__uint_as_float(r[e]) - ref);
                                s1 += ex2_approx(__uint_as_float(r[e + 1]) - ref);
                            }
                            m[i] = mn;
                            l[i] = s0 + s1;
                        }
                    }
                } else {
                    const int hidden = (key - first_cut) * p.gqa;  // rows before this one do not see the key
                    float     s1 = 0.0f;
                    for (int i = (group - u) & (kGroups - 1); i < n_b && ok; i += kGroups) {
                        if (!take(u + i)) { ok = false; break; }
                        const bool cut = key0 + kKeys > first_cut;
#pragma unroll
                        for (int h = 0; h < kSub; h += 32) {
                            uint32_t r[32];
                            tmem_ld32_sync(t_row + Z::kCols * ((u + i) % Z::kBufs) + h, r);
                            if constexpr (Q8) {
                                uint32_t x[32];
                                tmem_ld32_sync(t_row + Z::kCols * ((u + i) % Z::kBufs) + kSub + h, x);
#pragma unroll
                                for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(x[e]), d1, __uint_as_float(r[e]) * d0));
                            }
                            if (h + 32 == kSub) give_back(u + i);
                            const float4 * st4 = reinterpret_cast<const float4 *>(row_stat + kSub * i + h);
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float4 q = st4[e >> 1];  // two rows' (max, 1 / sum), the same for all threads
                                float        a = ex2_approx(__uint_as_float(r[e]) - q.x), c = ex2_approx(__uint_as_float(r[e + 1]) - q.z);
                                if (cut) {  // (the sum of a row that does not see the key may be NaN)
                                    if (kSub * i + h + e < hidden) a = q.y = 0.0f;
                                    if (kSub * i + h + e + 1 < hidden) c = q.w = 0.0f;
                                }
                                sum = fmaf(a, q.y, sum);
                                s1  = fmaf(c, q.w, s1);
                            }
                        }
                    }
                    group_sum[t & 1][group][row] = sum + s1;
                    if (!named_bar_all(1, kTakers, ok)) { ok = false; break; }
                    if (mine) {
                        sum = 0.0f;
#pragma unroll
                        for (int g = 0; g < kGroups; ++g) sum += group_sum[t & 1][g][row];
                        *score = fresh ? sum : fmaf(p.decay, old, sum);
                        if (fresh && p.row_pos != nullptr)
                            *(reinterpret_cast<int32_t *>(p.row_pos + (size_t) w.stream * p.nb_stream + (size_t) w.kvh * p.nb_head) + key) =
                                (p.n_seen ? p.n_seen[w.stream] : w.len) - w.len + key;
                    }
                }
                u += per_tile;
                if (Q8) {  // the scales of this stage are no longer needed
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty0 + 8 * st);
                }
            }
            if (!ok) give_up();
            if (!kWeights) {
                // a row's two halves of the keys meet through shared memory
                if (group & 1)
#pragma unroll
                    for (int i = 0; i < kMine; ++i) row_stat[256 * i + 128 * (group >> 1) + row] = make_float2(m[i], l[i]);
                ok = named_bar_all(1, kTakers, ok && !aborted());
                if (ok && !(group & 1)) {
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        const int at = 256 * i + 128 * (group >> 1) + row;
                        if (at >= rows) break;
                        const float2 o = row_stat[at];
                        const float  M = fmaxf(m[i], o.x), fa = m[i] == -INFINITY ? 1.0f : ex2_approx(m[i] - M), fb = o.x == -INFINITY ? 1.0f : ex2_approx(o.x - M);
                        p.stats[(size_t) b * rows + at] = make_float2(M, fmaf(l[i], fa, o.y * fb));
                    }
                }
            }
        } else if (Q8) {
            // ------------------------------------------------------------------ q8_0 rows to f16: two per thread
            bool ok = true;
            for (int t = 0; t < w.tiles && ok; ++t) {
                const int n = T + t, rs = n % kRawStages, st = n % Z::kStages, left = w.len - (w.tile0 + t) * kKeys;
                if (!mbar_wait_bounded(rfull0 + 8 * rs, (n / kRawStages) & 1) ||
                    (n >= Z::kStages && !mbar_wait_bounded(empty0 + 8 * st, ((n / Z::kStages) - 1) & 1))) { ok = false; break; }
                const uint8_t * raw = smem_gen + (sRaw - smem_base) + rs * kRawStage;
#pragma unroll 1
                for (int row = tid - (kIssueWarp + 1) * 32; row < kKeys; row += 64) {
                uint8_t *  out = smem_gen + (sK - smem_base) + st * kKTile + row * 128;
                const bool here = row < left;  // rows past the end: zeros, whatever the cache holds there
#pragma unroll
                for (int c = 0; c < 4; ++c) {  // 16 bytes: two pieces of eight f16
                    const uint4 x = *reinterpret_cast<const uint4 *>(raw + (row >> 6) * kKvTile * 64 + q8_byte_off(row, 16 * c));
                    const uint32_t v[4] = {x.x, x.y, x.z, x.w};
                    uint32_t       h[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[2 * e]     = here ? s8_pair_to_half2(v[e], 0x4140) : 0u;
                        h[2 * e + 1] = here ? s8_pair_to_half2(v[e], 0x4342) : 0u;
                    }
                    *reinterpret_cast<uint4 *>(out + (((2 * c) ^ (row & 7)) << 4))     = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(out + (((2 * c + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
                }
                const uint32_t d = *reinterpret_cast<const uint32_t *>(raw + 2 * kKvTile * 64 + row * 4);
                scales[st][row] = here ? make_float2(half_lo(d), half_hi(d)) : make_float2(0.0f, 0.0f);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(full0 + 8 * st);
                    mbar_arrive(rempty0 + 8 * rs);
                }
            }
            if (!ok) give_up();
        }
        T += w.tiles;
        U += w.tiles * per_tile;
        __syncthreads();  // the queries' tiles and the part's description are free
    }
    if (kWeights && waits) pdl_wait();  // no launch of the next call ends before the first one of this call
    if (warp == kCopyWarp && lane == 0 && aborted()) {  // copies in flight land before the CTA retires
        constexpr int      n_stages = Q8 ? kRawStages : Z::kStages;
        const uint32_t     bar0 = Q8 ? rfull0 : full0;
        for (int i = max(0, issued - n_stages); i < issued; ++i) mbar_wait_bounded(bar0 + 8 * (i % n_stages), (i / n_stages) & 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <bool Q8, bool kWeights>
int launch_one(vox_engine * e, const vox_kv_cache * c, const ObserveParams & p, int ctas, cudaStream_t st) {
    const uint32_t bit = 1u << ((Q8 ? 26 : 22) + (kWeights ? 1 : 0));
    if (!(e->attr_mask & bit)) {
        VOX_CUDA_TRY(cudaFuncSetAttribute(observe_window_kernel<Q8, kWeights>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<Q8>::kSmem));
        e->attr_mask |= bit;
    }
    launch_pdl(observe_window_kernel<Q8, kWeights>, dim3((unsigned) ctas), dim3(Shape<Q8>::kThreads), (size_t) Shape<Q8>::kSmem, st, c->map_k, p);
    return check_launch(e, kWeights ? "observe_window_kernel<weights>" : "observe_window_kernel<statistics>");
}

}  // namespace

namespace vox {

int observe_window_ctas(int n_streams, int n_kv_heads, int kv_bound) {
    const long long tiles = (long long) n_streams * n_kv_heads * ((kv_bound + kKeys - 1) / kKeys);
    return (int) std::max(1LL, std::min<long long>(tiles, kDecodeMaxSms));
}

// (max, sum) of every row of a part; the parts are no more than the CTAs, or as many as there are pairs
size_t observe_window_bytes(int n_streams, int n_kv_heads, int rows, int kv_bound) {
    return (size_t) std::max(observe_window_ctas(n_streams, n_kv_heads, kv_bound), n_streams * n_kv_heads) * rows * sizeof(float2);
}

int launch_observe_window(vox_engine * e, const vox_kv_cache * c, const ObserveParams & p, cudaStream_t st) {
    const int ctas = std::min(observe_window_ctas(p.n_streams, p.n_kv_heads, p.kv_bound), e->sm_count);
    int       rc;
    if (c->cfg.type == VOX_TYPE_Q8_0) {
        rc = launch_one<true, false>(e, c, p, ctas, st);
        return rc != VOX_ATTN_OK ? rc : launch_one<true, true>(e, c, p, ctas, st);
    }
    rc = launch_one<false, false>(e, c, p, ctas, st);
    return rc != VOX_ATTN_OK ? rc : launch_one<false, true>(e, c, p, ctas, st);
}

}  // namespace vox
