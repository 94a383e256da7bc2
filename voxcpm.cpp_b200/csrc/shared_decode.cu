// Decode attention over rows that many streams share (a voice prompt), computed once for all of them.
//
//   out[s] = softmax over (prefix rows of s, own rows of s) of scale * q[s].k, times v
//
// A stream's softmax splits into the part over its prefix and the part over its own rows; each part is a (max, sum,
// unnormalised output) and two parts join as two chunks of split-KV decode do.  The own rows are the decode kernel's work
// (decode_attn.cu), bound by HBM.  The prefix rows are this kernel's: the queries of all streams that share a prefix are
// the rows of one matrix product against it, so the prefix leaves HBM once for all of them instead of once per stream.
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <exception>
#include <new>
#include <vector>

using namespace vox;

// The streams of a call, arranged by prefix.  Host copy of the arrangement and its device arrays (one allocation):
//   [0] number of row tiles, then  tiles [max_tiles][4] = prefix, first entry of order, streams, 0;  order [n_streams];
//   place [n_streams];  of [n_streams]
struct vox_prefix_plan {
    vox_engine *         e = nullptr;
    int                  n_streams = 0, n_prefixes = 0, gqa = 0, max_tiles = 0;
    bool                 full = false;  // the row tiles are more than half full on average
    std::vector<int32_t> host;
    int32_t *            dev = nullptr;
    size_t tiles_at() const { return 4; }
    size_t order_at() const { return 4 + (size_t) max_tiles * 4; }
    size_t place_at() const { return order_at() + n_streams; }
    size_t of_at() const { return place_at() + n_streams; }
    size_t words() const { return of_at() + n_streams; }
};

namespace {

constexpr int kWarps    = 8;                    // consumer warps
constexpr int kThreads  = (kWarps + 1) * 32;
constexpr int kKeys     = 128;                  // keys per ring stage
constexpr int kMergeStride = 66;

template <bool Q8> struct Ring {
    static constexpr int kStages     = Q8 ? 4 : 3;
    static constexpr int kBoxBytes   = Q8 ? 9 * 1024 : 2 * kKvTile * 128;  // 64 rows of K and V
    static constexpr int kBoxTx      = Q8 ? kQ8TileBytes : kBoxBytes;
    static constexpr int kVOff       = Q8 ? kQ8VBytesOff : kKvTile * 128;
    static constexpr int kStageBytes = 2 * kBoxBytes;
    static constexpr int kMergeBytes = (kWarps / 2) * 16 * kMergeStride * 4;
    static constexpr int kSmemBytes  = kStages * kStageBytes + kMergeBytes + 1024;
};

struct SharedParams {
    const uint8_t * q;
    size_t          q_nb_head, q_nb_stream;
    const float2 *  rope;
    const int32_t * plan;      // [0] row tiles
    const int32_t * tiles;     // [tile][4]
    const int32_t * order;
    const int32_t * len;       // [prefix]
    float2 *        ml;
    float4 *        acc;
    int             n_prefixes, n_kv_heads, gqa, layer, max_len;
    int             chunk, max_chunks;
    float           scale_log2;
    const uint8_t * q8_tiles;
    size_t          q8_nb_head, q8_nb_stream;
    int *           status;
};

struct Item {
    int prefix, first, rows, kvh, key0, key1, slot;
};
// item i of the launch: chunk fastest, then kv head, then row tile; false where there is nothing to do
__device__ __forceinline__ bool load_item(const SharedParams & p, int i, Item & w) {
    const int chunk = i % p.max_chunks, pair = i / p.max_chunks;
    w.kvh = pair % p.n_kv_heads;
    const int4 t = *reinterpret_cast<const int4 *>(p.tiles + 4 * (size_t) (pair / p.n_kv_heads));
    w.prefix = t.x; w.first = t.y; w.rows = t.z * p.gqa;
    const int len = max(0, min(p.len[w.prefix], p.max_len));
    if (chunk >= prefix_chunks(len, p.chunk, p.max_chunks)) return false;
    w.key0 = chunk * p.chunk;
    w.key1 = chunk == p.max_chunks - 1 ? len : min(len, w.key0 + p.chunk);
    w.slot = i;
    return true;
}

template <bool Q8>
__global__ void __launch_bounds__(kThreads, 1)
shared_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedParams p) {
    using R = Ring<Q8>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * R::kStages];
    __shared__ int      abort_flag;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float *        merge     = reinterpret_cast<float *>(smem_raw + (smem_base - smem_u32(smem_raw)) + R::kStages * R::kStageBytes);
    const int      tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[R::kStages]);
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < R::kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, kWarps);
        }
        fence_mbar_init();
    }
    __syncthreads();
    // The decode kernel behind this one relies on this order: its CTAs start once every CTA here has passed the wait.
    pdl_wait();
    pdl_launch_dependents();
    const int n_items = p.plan[0] * p.n_kv_heads * p.max_chunks;

    if (warp == kWarps) {
        // ------------------------------------------------------------------ producer: one lane
        if (lane != 0) return;
        int  it = 0;
        bool good = true;
        for (int i = blockIdx.x; i < n_items && good; i += gridDim.x) {
            Item w;
            if (!load_item(p, i, w)) continue;
            for (int key = w.key0; key < w.key1 && good; key += kKeys, ++it) {
                const int s = it % R::kStages;
                if (it >= R::kStages && !mbar_wait_bounded(empty0 + 8 * s, ((it / R::kStages) - 1) & 1)) {
                    atomicOr(p.status, kStatusTimeout);
                    atomicExch(&abort_flag, 1);
                    good = false;
                }
                if (good && *reinterpret_cast<volatile int *>(&abort_flag)) good = false;
                if (!good) break;
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
        }
        if (*reinterpret_cast<volatile int *>(&abort_flag))  // copies already issued land before the CTA retires
            for (int i = max(0, it - R::kStages); i < it; ++i) mbar_wait_bounded(full0 + 8 * (i % R::kStages), (i / R::kStages) & 1);
        return;
    }

    // ---------------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    int       it = 0;
    for (int i = blockIdx.x; i < n_items; i += gridDim.x) {
        Item w;
        if (!load_item(p, i, w)) continue;
        // Warps are arranged as row groups of 16 x key groups: a tile of few rows has its keys spread over the warps.
        const int groups = (w.rows + 15) >> 4;
        const int rg     = groups <= 1 ? 1 : groups <= 2 ? 2 : groups <= 4 ? 4 : 8;
        const int kg = kWarps / rg, wr = warp % rg, wk = warp / rg, span = kKeys / kg;
        const bool busy = wr < groups;

        // Q: rows g and g + 8 of this warp's 16, as hi + lo (the order of the head dimensions as in the decode kernel)
        uint32_t qh[4][4], ql[4][4];
        float    q_bias[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int  row  = 16 * wr + g + 8 * h;
            const bool live = row < w.rows;
            const int  at   = live ? row : 0;
            const int  stream = p.order[w.first + at / p.gqa], head = w.kvh * p.gqa + at % p.gqa;
            const float * qrow = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) head * p.q_nb_head);
            float xs[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int d0 = Q8 ? 32 * (c >> 1) + 8 * t + 4 * (c & 1) : 16 * c + 2 * t;
                const int d1 = Q8 ? d0 + 2 : d0 + 8;
                const float2 x = *reinterpret_cast<const float2 *>(qrow + d0);
                const float2 y = *reinterpret_cast<const float2 *>(qrow + d1);
                xs[c][0] = x.x; xs[c][1] = x.y; xs[c][2] = y.x; xs[c][3] = y.y;
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
                qh[c][h]     = pack_half2(hi[0], hi[1]);
                qh[c][h + 2] = pack_half2(hi[2], hi[3]);
                ql[c][h]     = pack_half2(lo[0], lo[1]);
                ql[c][h + 2] = pack_half2(lo[2], lo[3]);
                if constexpr (Q8) q_bias[h][c >> 1] += ((hi[0] + lo[0]) + (hi[1] + lo[1])) + ((hi[2] + lo[2]) + (hi[3] + lo[3]));
            }
            if constexpr (Q8) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    q_bias[h][b] += __shfl_xor_sync(0xffffffffu, q_bias[h][b], 1);
                    q_bias[h][b] += __shfl_xor_sync(0xffffffffu, q_bias[h][b], 2);
                    q_bias[h][b] *= 128.0f * kTwoM24;
                }
            }
        }

        float o[8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float v_bias[2][2] = {{0.f, 0.f}, {0.f, 0.f}}, v_unit = 1.0f, v_limit = -1.0f;
#pragma unroll
        for (int n = 0; n < 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        bool ok = true;
        for (int key = w.key0; key < w.key1; key += kKeys, ++it) {
            const int s = it % R::kStages;
            if (!mbar_wait_bounded(full0 + 8 * s, (it / R::kStages) & 1)) {
                *reinterpret_cast<volatile int *>(&abort_flag) = 1;
                ok = false;
                break;
            }
            if (busy) {
                for (int k0 = wk * span; k0 < (wk + 1) * span && key + k0 < w.key1; k0 += 16) {
                    const uint32_t box = smem_base + s * R::kStageBytes + (k0 >> 6) * R::kBoxBytes;
                    const int      r0  = k0 & 63, pos0 = key + k0;
                    const bool     edge = pos0 + 16 > w.key1;
                    float          sc[2][4];
                    if constexpr (!Q8) {
                        const int k_row = r0 + ((lane >> 4) << 3) + (lane & 7), k_chk = (lane >> 3) & 1;
#pragma unroll
                        for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4(box + k_row * 128 + (((2 * c + k_chk) ^ (k_row & 7)) << 4), b0, b1, b2, b3);
                            mma_16816(sc[0], qh[c], b0, b1);
                            mma_16816(sc[1], qh[c], b2, b3);
                            mma_16816(sc[0], ql[c], b0, b1);
                            mma_16816(sc[1], ql[c], b2, b3);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float part[2][4];
                            const int row = r0 + 8 * j + g;
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                part[b][0] = part[b][1] = -q_bias[0][b];
                                part[b][2] = part[b][3] = -q_bias[1][b];
                                const uint2 raw = lds64(box + row * 64 + (((2 * b + (t >> 1)) ^ ((row >> 1) & 3)) << 4) + ((t & 1) << 3));
                                const uint32_t x0 = u8_pair_to_half2(raw.x, 0x4140), x1 = u8_pair_to_half2(raw.x, 0x4342);
                                const uint32_t y0 = u8_pair_to_half2(raw.y, 0x4140), y1 = u8_pair_to_half2(raw.y, 0x4342);
                                mma_16816(part[b], qh[2 * b], x0, x1);
                                mma_16816(part[b], qh[2 * b + 1], y0, y1);
                                mma_16816(part[b], ql[2 * b], x0, x1);
                                mma_16816(part[b], ql[2 * b + 1], y0, y1);
                            }
                            const uint2 ds = lds64(box + kQ8KScaleOff + (r0 + 8 * j + 2 * t) * 4);
                            sc[j][0] = (part[0][0] * half_lo(ds.x) + part[1][0] * half_hi(ds.x)) * kTwo24;
                            sc[j][1] = (part[0][1] * half_lo(ds.y) + part[1][1] * half_hi(ds.y)) * kTwo24;
                            sc[j][2] = (part[0][2] * half_lo(ds.x) + part[1][2] * half_hi(ds.x)) * kTwo24;
                            sc[j][3] = (part[0][3] * half_lo(ds.y) + part[1][3] * half_hi(ds.y)) * kTwo24;
                        }
                    }
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (pos0 + 8 * j + 2 * t + (e & 1) >= w.key1) sc[j][e] = -INFINITY;
                    }
                    float alpha[2], m_exp[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float top = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const float m_new = fmaxf(m[h], top);
                        alpha[h] = m_new == -INFINITY ? 1.0f : ex2_approx(m[h] - m_new);
                        m_exp[h] = (m_new == -INFINITY ? 0.0f : m_new) - (Q8 ? 0.0f : 10.0f);
                        m[h]     = m_new;
                    }
                    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1];
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            l[h] *= alpha[h];
                            v_bias[h][0] *= alpha[h]; v_bias[h][1] *= alpha[h];
                        }
                    }
                    float pr[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) pr[j][e] = ex2_approx(sc[j][e] - m_exp[e >> 1]);
                    const int v_row = r0 + (((lane >> 3) & 1) << 3) + (lane & 7), v_chk = lane >> 4;
                    const uint32_t vb = box + R::kVOff;
                    if constexpr (!Q8) {
                        uint32_t ph[4], pl[4];
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float h0, l0, h1, l1;
                                split_hi_lo(pr[j][2 * h], h0, l0);
                                split_hi_lo(pr[j][2 * h + 1], h1, l1);
                                ph[2 * j + h] = pack_half2(h0, h1);
                                pl[2 * j + h] = pack_half2(l0, l1);
                                l[h] += (h0 + l0) + (h1 + l1);
                            }
#pragma unroll
                        for (int n2 = 0; n2 < 4; ++n2) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4_trans(vb + v_row * 128 + (((2 * n2 + v_chk) ^ (v_row & 7)) << 4), b0, b1, b2, b3);
                            if (edge) {  // rows past the length may hold anything: zero times a NaN is none
                                const uint32_t keep0 = keep_rows(pos0 + 2 * t, w.key1), keep1 = keep_rows(pos0 + 8 + 2 * t, w.key1);
                                b0 &= keep0; b1 &= keep1; b2 &= keep0; b3 &= keep1;
                            }
                            mma_16816(o[2 * n2], ph, b0, b1);
                            mma_16816(o[2 * n2 + 1], ph, b2, b3);
                            mma_16816(o[2 * n2], pl, b0, b1);
                            mma_16816(o[2 * n2 + 1], pl, b2, b3);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            l[h] += (pr[0][2 * h] + pr[0][2 * h + 1]) + (pr[1][2 * h] + pr[1][2 * h + 1]);
                        uint2 ds[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            ds[j] = lds64(box + kQ8VScaleOff + (r0 + 8 * j + 2 * t) * 4);
                            if (pos0 + 8 * j + 2 * t >= w.key1) ds[j].x = 0u;
                            if (pos0 + 8 * j + 2 * t + 1 >= w.key1) ds[j].y = 0u;
                        }
                        // products in units of v_unit, as in the decode kernel
                        const __half2 big = __hmax2(__hmax2(__habs2(as_half2(ds[0].x)), __habs2(as_half2(ds[0].y))),
                                                    __hmax2(__habs2(as_half2(ds[1].x)), __habs2(as_half2(ds[1].y))));
                        float dm = fmaxf(__low2float(big), __high2float(big));
                        if (__any_sync(0xffffffffu, dm > v_limit)) {
                            dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, 1));
                            dm = fmaxf(dm, __shfl_xor_sync(0xffffffffu, dm, 2));
                            const float unit = dm > 0.0f ? __uint_as_float(__float_as_uint(dm) & 0x7f800000u) : kTwoM24;
                            const float f    = v_unit / unit;
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                o[n][0] *= f; o[n][1] *= f; o[n][2] *= f; o[n][3] *= f;
                            }
#pragma unroll
                            for (int h = 0; h < 2; ++h) { v_bias[h][0] *= f; v_bias[h][1] *= f; }
                            v_unit  = unit;
                            v_limit = dm > 0.0f ? unit * 256.0f : 0.0f;
                        }
                        const float to_units = 32.0f / v_unit;
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            uint32_t ph[4], pl[4];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float s0 = to_units * (b ? half_hi(ds[j].x) : half_lo(ds[j].x)), s1 = to_units * (b ? half_hi(ds[j].y) : half_lo(ds[j].y));
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    float h0, l0, h1, l1;
                                    split_hi_lo(pr[j][2 * h] * s0, h0, l0);
                                    split_hi_lo(pr[j][2 * h + 1] * s1, h1, l1);
                                    ph[2 * j + h] = pack_half2(h0, h1);
                                    pl[2 * j + h] = pack_half2(l0, l1);
                                }
                            }
                            float sums[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_16816(sums, ph, 0x3c003c00u, 0x3c003c00u);
                            mma_16816(sums, pl, 0x3c003c00u, 0x3c003c00u);
                            v_bias[0][b] += sums[0];
                            v_bias[1][b] += sums[2];
                            uint32_t r[4];
                            ldmatrix_x4_trans(vb + v_row * 64 + (((v_chk + 2 * b) ^ ((v_row >> 1) & 3)) << 4), r[0], r[1], r[2], r[3]);
#pragma unroll
                            for (int n = 0; n < 4; ++n) {  // chunk n / 2 of 16 columns, even or odd ones
                                const uint32_t sel = n & 1 ? 0x4341 : 0x4240;
                                const uint32_t b0 = u8_pair_to_half2(r[2 * (n >> 1)], sel), b1 = u8_pair_to_half2(r[2 * (n >> 1) + 1], sel);
                                mma_16816(o[4 * b + n], ph, b0, b1);
                                mma_16816(o[4 * b + n], pl, b0, b1);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * s);
        }
        if (*reinterpret_cast<volatile int *>(&abort_flag)) ok = false;
        if (!named_bar_all(1, kWarps * 32, ok)) {
            if (tid == 0) {
                *reinterpret_cast<volatile int *>(&abort_flag) = 1;
                atomicOr(p.status, kStatusTimeout);
            }
            return;
        }

        // ---- the item's result: warps of one row group and several key groups are merged, half of them at a time
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (!Q8) m[h] -= 10.0f;
        }
        if constexpr (Q8) {
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][e] = fmaf(o[n][e], kTwo24, -128.0f * v_bias[e >> 1][n >> 2]) * (v_unit / 32.0f);
        }
        for (int half = kg >> 1; half >= 1; half >>= 1) {
            float * mine = merge + ((size_t) ((wk - half) * rg + wr) * 16) * kMergeStride;
            if (wk >= half && wk < 2 * half) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float * row = mine + (g + 8 * h) * kMergeStride;
                    if (t == 0) *reinterpret_cast<float2 *>(row) = make_float2(m[h], l[h]);
#pragma unroll
                    for (int n = 0; n < 8; ++n) *reinterpret_cast<float2 *>(row + 2 + 8 * n + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                }
            }
            named_bar_sync(1, kWarps * 32);
            if (wk < half) {
                const float * theirs = merge + ((size_t) (wk * rg + wr) * 16) * kMergeStride;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float * row = theirs + (g + 8 * h) * kMergeStride;
                    const float2  ml  = *reinterpret_cast<const float2 *>(row);
                    const float   mn  = fmaxf(m[h], ml.x);
                    const float   fa = m[h] == -INFINITY ? 0.0f : exp2f(m[h] - mn), fb = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - mn);
                    m[h] = mn;
                    l[h] = l[h] * fa + ml.y * fb;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const float2 x = *reinterpret_cast<const float2 *>(row + 2 + 8 * n + 2 * t);
                        o[n][2 * h]     = o[n][2 * h] * fa + x.x * fb;
                        o[n][2 * h + 1] = o[n][2 * h + 1] * fa + x.y * fb;
                    }
                }
            }
            named_bar_sync(1, kWarps * 32);
        }
        if (wk == 0 && busy) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = 16 * wr + g + 8 * h;
                if (row >= w.rows) continue;
                const size_t at = (size_t) w.slot * kPrefixRows + row;
                if (t == 0) p.ml[at] = make_float2(m[h], l[h]);
                float * out = reinterpret_cast<float *>(p.acc + (size_t) w.slot * 16 * kPrefixRows + row);
                auto    col = [](int d) { return (size_t) (d >> 2) * kPrefixRows * 4 + (d & 3); };  // place of output column d
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    if constexpr (Q8) {  // tile n: chunk n / 2, this lane 16 (n / 2) + 4t + (n % 2) and two further
                        const int d = 16 * (n >> 1) + 4 * t + (n & 1);
                        out[col(d)]     = o[n][2 * h];
                        out[col(d + 2)] = o[n][2 * h + 1];
                    } else {
                        *reinterpret_cast<float2 *>(out + col(8 * n + 2 * t)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Full row tiles on the 5th-generation tensor cores (f16 caches).
//
// One CTA takes one (row tile, kv head, chunk of keys).  Q (scaled by scale * log2 e) lies in shared memory as two f16 tiles,
// value and remainder; scores S = Q_lo.K + Q_hi.K (the small part first: the accumulator truncates) come 64 keys at a time
// into one of six score buffers in TMEM.  Two groups of four softmax warps take them in turn, a thread per row: 64 scores
// out of TMEM, weights 2^(S - ref) back over them as two packed f16 tiles (value and remainder, 22 bits), from where the
// tensor core takes them as the A operand of P.V.  Every group has an output accumulator and a reference maximum of its
// own, so the groups never wait for one another; they are joined once, at the end.  The reference of a row is raised only
// when a maximum exceeds it by 2^8 (its accumulator is then rescaled in TMEM).
//   warps 0-3, 4-7  softmax groups    warp 8  K/V copies    warp 9  issues S = Q.K    warp 10  issues O += P.V
constexpr int kTcThreads = 11 * 32;
constexpr int kTcStages  = 4;
constexpr int kSub       = 64;                    // keys of a score tile
constexpr int kSBufs     = 6;
constexpr int kTcOCol    = kSBufs * kSub;         // two accumulators of 64 columns behind the score buffers
constexpr int kQTile     = kPrefixRows * 128;
constexpr int kTcStage   = 2 * kKeys * 128;       // 128 rows of K, 128 rows of V
constexpr int kTcSmem    = 2 * kQTile + kTcStages * kTcStage + 1024;
constexpr float kTcShift = 6.0f;                  // weights up to 2^(8 + 6): their remainders stay normal f16 numbers

// multiply this thread's accumulator row by f; rare, kept out of line so that its registers do not weigh on the loop
__device__ __noinline__ void rescale_row(uint32_t t_o, float f) {
    tc_fence_after();
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        float o[32];
        tmem_ld32(t_o + 32 * h, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= f;
        tmem_st32(t_o + 32 * h, o);
    }
    tc_fence_before();
}

__global__ void __launch_bounds__(kTcThreads, 1)
shared_rows_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * kTcStages + 3 * kSBufs + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int      abort_flag;
    __shared__ float2   other_ml[kPrefixRows];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *      smem_gen  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t sQ = smem_base, sKV = sQ + 2 * kQTile;
    const int      tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = full0 + 8 * kTcStages, bS0 = empty0 + 8 * kTcStages, bP0 = bS0 + 8 * kSBufs,
                   bF0 = bP0 + 8 * kSBufs, bO = bF0 + 8 * kSBufs;
    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < kTcStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < kSBufs; ++s) {
            mbar_init(bS0 + 8 * s, 1);
            mbar_init(bP0 + 8 * s, 4);  // one arrival per warp of the group that took the tile
            mbar_init(bF0 + 8 * s, 1);
        }
        mbar_init(bO, 1);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc(smem_u32(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // The decode kernel behind this one relies on this order: its CTAs start once every CTA here has passed the wait.
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&tmem_slot);
    Item           w;
    const bool     work = (int) blockIdx.x < p.plan[0] * p.n_kv_heads * p.max_chunks && load_item(p, blockIdx.x, w);
    if (!work) w.key0 = w.key1 = 0;
    const int n_keys = w.key1 - w.key0, n_tiles = (n_keys + kKeys - 1) / kKeys, n_sub = (n_keys + kSub - 1) / kSub;

    auto give_up = [&]() {
        atomicOr(p.status, kStatusTimeout);
        atomicExch(&abort_flag, 1);
    };
    auto aborted   = [&]() { return *reinterpret_cast<volatile int *>(&abort_flag) != 0; };
    auto warp_wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity)) != 0; };
    auto load_tile = [&](int T) {  // one lane
        const int      st = T % kTcStages, boxes = n_keys - T * kKeys > kSub ? 2 : 1;
        const uint32_t bar = full0 + 8 * st, dst = sKV + st * kTcStage;
        mbar_expect_tx(bar, boxes * 2 * kSub * 128);
        for (int b = 0; b < boxes; ++b) {
            tma_load_5d(dst + b * kSub * 128, &map_k, bar, 0, w.key0 + T * kKeys + b * kSub, w.kvh, w.prefix, p.layer);
            tma_load_5d(dst + kKeys * 128 + b * kSub * 128, &map_v, bar, 0, w.key0 + T * kKeys + b * kSub, w.kvh, w.prefix, p.layer);
        }
    };
    if (warp == 8) {
        if (lane == 0)
            for (int T = 0; T < min(n_tiles, kTcStages); ++T) load_tile(T);
    } else if (warp < 8 && work) {
        // Q: two threads per row, 32 head dimensions each
        const int  row = tid >> 1, half = tid & 1;
        const bool live = row < w.rows;
        const int  at = live ? row : 0, stream = p.order[w.first + at / p.gqa], head = w.kvh * p.gqa + at % p.gqa;
        const float * src = reinterpret_cast<const float *>(p.q + (size_t) stream * p.q_nb_stream + (size_t) head * p.q_nb_head);
        float x[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 v = *reinterpret_cast<const float2 *>(src + 32 * half + 2 * i);
            x[2 * i] = v.x; x[2 * i + 1] = v.y;
        }
        if (p.rope != nullptr) {  // the other half of the row is the neighbouring thread's
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 r = p.rope[(size_t) stream * (kHeadDim / 2) + i];
                const float  y = __shfl_xor_sync(0xffffffffu, x[i], 1);
                x[i] = half ? __fadd_rn(__fmul_rn(y, r.y), __fmul_rn(x[i], r.x)) : __fsub_rn(__fmul_rn(x[i], r.x), __fmul_rn(y, r.y));
            }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float h0, l0, h1, l1;
                split_hi_lo(live ? x[8 * c + 2 * i] * p.scale_log2 : 0.0f, h0, l0);
                split_hi_lo(live ? x[8 * c + 2 * i + 1] * p.scale_log2 : 0.0f, h1, l1);
                hi[i] = pack_half2(h0, h1);
                lo[i] = pack_half2(l0, l1);
            }
            uint8_t * dst = smem_gen + row * 128 + (((4 * half + c) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4 *>(dst)          = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4 *>(dst + kQTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async_smem();
    }
    __syncthreads();

    if (warp == 8) {
        // ------------------------------------------------------------------ copies
        if (lane == 0) {
            bool ok = true;
            int  T  = min(n_tiles, kTcStages);
            for (; T < n_tiles && ok; ++T) {
                if (!mbar_wait_bounded(empty0 + 8 * (T % kTcStages), ((T / kTcStages) - 1) & 1) || aborted()) { ok = false; break; }
                load_tile(T);
            }
            if (!ok) {
                give_up();
                for (int i = max(0, T - kTcStages); i < T; ++i) mbar_wait_bounded(full0 + 8 * (i % kTcStages), (i / kTcStages) & 1);
            }
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ scores (all lanes in the loop, one issues)
        constexpr uint32_t idesc = idesc_f16(kSub, false);
        const uint64_t     dQ = smem_desc_sw128(sQ), dQlo = smem_desc_sw128(sQ + kQTile), dK = smem_desc_sw128(sKV);
        const bool         leader = elect_one();
        bool               ok = true;
        for (int U = 0; U < n_sub && ok; ++U) {
            const int T = U >> 1, st = T % kTcStages, sb = U % kSBufs;
            if (!warp_wait(full0 + 8 * st, (T / kTcStages) & 1) || (U >= kSBufs && !warp_wait(bF0 + 8 * sb, ((U / kSBufs) - 1) & 1))) { ok = false; break; }
            tc_fence_after();
            if (leader) {
                const uint32_t dS = tmem + kSub * sb;
                const uint64_t k0 = dK + (uint64_t) (st * (kTcStage >> 4) + (U & 1) * ((kSub * 128) >> 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16(dS, dQlo + k * 2, k0 + k * 2, idesc, k > 0);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16(dS, dQ + k * 2, k0 + k * 2, idesc, 1);
                tc_commit(bS0 + 8 * sb);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) give_up();
    } else if (warp == 10) {
        // ------------------------------------------------------------------ output
        constexpr uint32_t idesc = idesc_f16(kHeadDim, true);
        const uint64_t     dV = smem_desc_sw128_mn(sKV + kKeys * 128, 16);
        const bool         leader = elect_one();
        bool               ok = true;
        for (int U = 0; U < n_sub && ok; ++U) {
            const int T = U >> 1, st = T % kTcStages, sb = U % kSBufs;
            if (!warp_wait(full0 + 8 * st, (T / kTcStages) & 1) || !warp_wait(bP0 + 8 * sb, (U / kSBufs) & 1)) { ok = false; break; }
            tc_fence_after();
            if (leader) {
                const uint32_t tP = tmem + kSub * sb, tO = tmem + kTcOCol + kHeadDim * (U & 1);
                const uint64_t v0 = dV + (uint64_t) (st * (kTcStage >> 4) + (U & 1) * ((kSub * 128) >> 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16_ts(tO, tP + 8 * k, v0 + k * (2048 >> 4), idesc, U > 1 || k > 0);
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16_ts(tO, tP + kSub / 2 + 8 * k, v0 + k * (2048 >> 4), idesc, 1);
                tc_commit(bF0 + 8 * sb);
                if ((U & 1) || U == n_sub - 1) tc_commit(empty0 + 8 * st);
                if (U == n_sub - 1) tc_commit(bO);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) give_up();
    } else {
        // ------------------------------------------------------------------ softmax: a thread per row
        const int      group = warp >> 2, row = tid & 127;
        const uint32_t t_row = tmem + ((uint32_t) (32 * (warp & 3)) << 16), t_o = t_row + kTcOCol + kHeadDim * group;
        float          m = -INFINITY, l = 0.0f;
        bool           ok = true;
        for (int U = group; U < n_sub; U += 2) {
            const int sb = U % kSBufs, left = n_keys - U * kSub;  // keys of this tile and after
            if (!mbar_wait_bounded(bS0 + 8 * sb, (U / kSBufs) & 1)) { ok = false; break; }
            tc_fence_after();
            const uint32_t t_s = t_row + kSub * sb;
            uint32_t       r[kSub];
            tmem_ld64_sync(t_s, r);
            if (left < kSub) {
#pragma unroll
                for (int i = 0; i < kSub; ++i)
                    if (i >= left) r[i] = 0xff800000u;
                // rows past the prefix may hold anything, and zero times a NaN is none: V's are cleared
                const int T = U >> 1, st = T % kTcStages;
                if (!mbar_wait_bounded(full0 + 8 * st, (T / kTcStages) & 1)) { ok = false; break; }
                if (row >= left && row < kSub) {
                    uint4 * v = reinterpret_cast<uint4 *>(smem_gen + (sKV - smem_base) + st * kTcStage + kKeys * 128 + ((U & 1) * kSub + row) * 128);
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
            if (U < 2) {
                m = top;
            } else {
                const bool raise = top > m + 8.0f;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2_approx(m - top) : 1.0f;
                    if (raise) m = top;
                    l *= f;
                    // the accumulator is at rest once P.V of the group's last tile has retired
                    if (!mbar_wait_bounded(bF0 + 8 * ((U - 2) % kSBufs), ((U - 2) / kSBufs) & 1)) { ok = false; break; }
                    rescale_row(t_o, f);
                }
            }
            const float ref = m - kTcShift;
#pragma unroll
            for (int g = 0; g < kSub / 16; ++g) {
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
            __syncwarp();
            if (lane == 0) mbar_arrive(bP0 + 8 * sb);
        }
        if (ok && n_sub > 0 && !mbar_wait_bounded(bO, 0)) ok = false;
        if (!ok) give_up();
        ok = named_bar_all(1, 256, ok && !aborted());
        if (ok && work) {
            tc_fence_after();
            // the second group's part goes through the ring's memory (every copy has been consumed)
            float4 * const other = reinterpret_cast<float4 *>(smem_gen + (sKV - smem_base));
            const bool     both  = n_sub > 1;
            uint32_t       r[64];
            if (group == 0 || both) tmem_ld64_sync(t_o, r);
            if (group == 1 && both) {
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    other[c * kPrefixRows + row] = make_float4(__uint_as_float(r[4 * c]), __uint_as_float(r[4 * c + 1]), __uint_as_float(r[4 * c + 2]), __uint_as_float(r[4 * c + 3]));
                other_ml[row] = make_float2(m, l);
            }
            named_bar_sync(1, 256);
            if (group == 0 && row < w.rows) {
                float fa = 1.0f, fb = 0.0f;
                if (both) {
                    const float2 b  = other_ml[row];
                    const float  mn = fmaxf(m, b.x);
                    fa = m == -INFINITY ? 0.0f : exp2f(m - mn);
                    fb = b.x == -INFINITY ? 0.0f : exp2f(b.x - mn);
                    l  = l * fa + b.y * fb;
                    m  = mn;
                }
                p.ml[(size_t) w.slot * kPrefixRows + row] = make_float2(m - kTcShift, l);
                float4 * out = p.acc + (size_t) w.slot * 16 * kPrefixRows + row;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    float4 x = make_float4(__uint_as_float(r[4 * c]) * fa, __uint_as_float(r[4 * c + 1]) * fa, __uint_as_float(r[4 * c + 2]) * fa, __uint_as_float(r[4 * c + 3]) * fa);
                    if (both) {
                        const float4 y = other[c * kPrefixRows + row];
                        x = make_float4(fmaf(y.x, fb, x.x), fmaf(y.y, fb, x.y), fmaf(y.z, fb, x.z), fmaf(y.w, fb, x.w));
                    }
                    out[c * kPrefixRows] = x;
                }
            }
        }
    }
    // common exit: every role has left its loop; release TMEM
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Keys per chunk and chunks per prefix.  Enough items for every SM where the prefixes are long enough (a chunk holds at
// least one stage), and no more than kPrefixMaxChunks partials per row.
struct Chunks { int chunk, max_chunks; };
Chunks plan_chunks(int sms, int max_tiles, int n_kv_heads, int prefix_bound) {
    const int pairs  = std::max(1, max_tiles * n_kv_heads);
    const int wanted = std::min(kPrefixMaxChunks, std::max(1, (sms + pairs - 1) / pairs));
    const int bound  = std::max(1, prefix_bound);
    Chunks    c;
    c.chunk      = std::max(kKeys, ((bound + wanted - 1) / wanted + kKeys - 1) / kKeys * kKeys);
    c.max_chunks = (bound + c.chunk - 1) / c.chunk;
    return c;
}

size_t aligned(size_t n) { return (n + 255) & ~(size_t) 255; }

size_t shared_rows_bytes(const vox_prefix_plan * pl, int n_kv_heads, int prefix_bound) {
    const Chunks c     = plan_chunks(kDecodeMaxSms, pl->max_tiles, n_kv_heads, prefix_bound);
    const size_t slots = (size_t) pl->max_tiles * n_kv_heads * c.max_chunks;
    return aligned(slots * kPrefixRows * sizeof(float2)) + aligned(slots * kPrefixRows * kHeadDim * sizeof(float));
}

// Arranges the streams by prefix: a counting sort, then row tiles of one prefix each.  An entry out of range is refused
// before anything of the plan changes.
int arrange(vox_prefix_plan * pl, const int32_t * prefix_of) {
    for (int s = 0; s < pl->n_streams; ++s)
        VOX_REQUIRE(prefix_of[s] >= -1 && prefix_of[s] < pl->n_prefixes, VOX_ATTN_INVALID_ARGUMENT,
                    "prefix_of[%d] = %d: not a prefix in [0, %d), nor -1", s, prefix_of[s], pl->n_prefixes);
    std::vector<int32_t> start;
    try {
        start.assign((size_t) pl->n_prefixes + 1, 0);
        pl->host.assign(pl->words(), 0);
    } catch (const std::exception &) {
        set_error("out of host memory");
        return VOX_ATTN_OUT_OF_MEMORY;
    }
    int32_t * h = pl->host.data(), * order = h + pl->order_at(), * place = h + pl->place_at(), * of = h + pl->of_at();
    for (int s = 0; s < pl->n_streams; ++s)
        if (prefix_of[s] >= 0) start[prefix_of[s] + 1] += 1;
    for (int g = 0; g < pl->n_prefixes; ++g) start[g + 1] += start[g];
    // start[g] moves to the end of prefix g's streams while they are placed: afterwards it is the first of prefix g + 1
    for (int s = 0; s < pl->n_streams; ++s) {
        place[s] = -1;
        if (prefix_of[s] >= 0) order[start[prefix_of[s]]++] = s;
    }
    const int per_tile = kPrefixRows / pl->gqa;
    int       n_tiles  = 0;
    for (int g = 0, first = 0; g < pl->n_prefixes; first = start[g++])
        for (int m0 = first; m0 < start[g]; m0 += per_tile, ++n_tiles) {
            const int n = std::min(per_tile, start[g] - m0);
            int32_t * t = h + pl->tiles_at() + 4 * (size_t) n_tiles;
            t[0] = g; t[1] = m0; t[2] = n;
            for (int j = 0; j < n; ++j) {
                place[order[m0 + j]] = n_tiles * kPrefixRows + j;
                of[order[m0 + j]]    = g;
            }
        }
    h[0] = n_tiles;
    pl->full = 2 * start[pl->n_prefixes - 1] > n_tiles * per_tile;
    return VOX_ATTN_OK;
}

int check_shared(const vox_engine * e, const vox_decode_shared_args * a) {
    VOX_REQUIRE(e && a, VOX_ATTN_INVALID_ARGUMENT, "vox_attn_decode_shared: null argument");
    const int rc = check_decode(e, &a->own, "vox_attn_decode_shared");
    if (rc != VOX_ATTN_OK) return rc;
    const vox_kv_cache * c = a->own.cache;
    VOX_REQUIRE(a->own.stream_order == nullptr, VOX_ATTN_UNSUPPORTED, "vox_attn_decode_shared takes no stream_order");
    VOX_REQUIRE((reinterpret_cast<uintptr_t>(a->lse) & 3) == 0, VOX_ATTN_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    if (a->prefix == nullptr && a->plan == nullptr) return VOX_ATTN_OK;  // own rows only
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
    pl->max_tiles = n_streams / (kPrefixRows / pl->gqa) + std::min(n_streams, n_prefixes);
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
    if (a == nullptr || a->own.cache == nullptr) return 0;
    const int    HK  = a->own.cache->cfg.n_kv_heads;
    const size_t own = decode_workspace_bytes(a->own.n_streams, a->own.n_heads, HK, a->own.kv_bound);
    return aligned(own) + (a->plan != nullptr ? shared_rows_bytes(a->plan, HK, a->prefix_bound) : 0);
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
    cudaStream_t         st  = static_cast<cudaStream_t>(stream);
    const vox_kv_cache * c   = a->own.cache;
    const int            HK  = c->cfg.n_kv_heads;
    const size_t         own = aligned(decode_workspace_bytes(a->own.n_streams, a->own.n_heads, HK, a->own.kv_bound));
    SharedRows           rows{};
    rows.lse = a->lse;
    if (a->plan != nullptr && a->prefix_bound > 0) {
        const vox_prefix_plan * pl = a->plan;
        const vox_kv_cache *    pc = a->prefix;
        const bool              q8 = pc->cfg.type == VOX_TYPE_Q8_0;
        const Chunks            ch = plan_chunks(kDecodeMaxSms, pl->max_tiles, HK, a->prefix_bound);
        const size_t            slots = (size_t) pl->max_tiles * HK * ch.max_chunks;
        VOX_REQUIRE(slots < (1u << 30), VOX_ATTN_UNSUPPORTED, "vox_attn_decode_shared: more than 2^30 partial results");
        uint8_t * ws = static_cast<uint8_t *>(workspace) + own;
        rows.fold.ml  = reinterpret_cast<float2 *>(ws);
        rows.fold.acc = reinterpret_cast<float4 *>(ws + aligned(slots * kPrefixRows * sizeof(float2)));
        rows.fold.place = pl->dev + pl->place_at();
        rows.fold.of    = pl->dev + pl->of_at();
        rows.fold.len   = a->prefix_len;
        rows.fold.max_len = pc->cfg.max_len;
        rows.fold.chunk = ch.chunk; rows.fold.max_chunks = ch.max_chunks;
        SharedParams p;
        p.q = reinterpret_cast<const uint8_t *>(a->own.q);
        p.q_nb_head = a->own.q_nb_head; p.q_nb_stream = a->own.q_nb_stream;
        p.rope  = reinterpret_cast<const float2 *>(a->own.rope_table);
        p.plan  = pl->dev; p.tiles = pl->dev + pl->tiles_at(); p.order = pl->dev + pl->order_at();
        p.len   = a->prefix_len;
        p.ml = const_cast<float2 *>(rows.fold.ml); p.acc = const_cast<float4 *>(rows.fold.acc);
        p.n_prefixes = pl->n_prefixes; p.n_kv_heads = HK; p.gqa = pl->gqa; p.layer = a->own.layer; p.max_len = pc->cfg.max_len;
        p.chunk = ch.chunk; p.max_chunks = ch.max_chunks;
        p.scale_log2 = a->own.scale * 1.4426950408889634f;
        p.q8_tiles = pc->k_data + (size_t) a->own.layer * pc->nb_layer;
        p.q8_nb_head = pc->nb_head; p.q8_nb_stream = pc->nb_stream;
        p.status = e->status_dev;
        const bool     tc     = !q8 && pl->full;
        const auto     kernel = tc ? shared_rows_tc_kernel : q8 ? shared_rows_kernel<true> : shared_rows_kernel<false>;
        const int      smem   = tc ? kTcSmem : q8 ? Ring<true>::kSmemBytes : Ring<false>::kSmemBytes;
        const uint32_t bit    = 1u << (tc ? 21 : q8 ? 19 : 18);
        if (!(e->attr_mask & bit)) {
            VOX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            e->attr_mask |= bit;
        }
        const unsigned grid = (unsigned) (tc ? slots : std::min<size_t>(slots, (size_t) e->sm_count));
        launch_pdl(kernel, dim3(grid), dim3(tc ? kTcThreads : kThreads), (size_t) smem, st, pc->map_k, pc->map_v, p);
        rc = check_launch(e, tc ? "shared_rows_tc_kernel" : q8 ? "shared_rows_kernel<q8_0>" : "shared_rows_kernel<f16>");
        if (rc != VOX_ATTN_OK) return rc;
    }
    return launch_decode_shared(e, &a->own, rows, workspace, own, st);
}

}  // extern "C"
