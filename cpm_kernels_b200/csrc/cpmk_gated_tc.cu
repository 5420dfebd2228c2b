// Tensor-core products of the gated feed-forward block: persistent CTA pairs on 256 x 256 tiles (tcgen05.mma.cta_group::2.kind::f16,
// fp16 or bf16 operands, fp32 accumulators in tensor memory), with the block's element-wise work in the epilogue:
//
//   kEpiGated   h = act(x Wg^T) * (x Wu^T).  CTA 0 of the pair stages 128 rows of Wg, CTA 1 the same 128 rows of Wu: the pair's
//               256-column accumulator holds the gate sums in columns 0-127 and the up sums in columns 128-255 of the same outputs, so
//               x is staged once for both and the activation and the product need no exchange.  256 x 128 outputs per tile.
//   kEpiDact    dh = dy Wd stays in tensor memory; the epilogue reads g and u and stores dg = dh u act'(g) and du = dh act(g).
//   kEpiStore   plain products: h Wd^T; dg Wg + du Wu (one accumulator, k runs through the first pair of operands, then the second);
//               dg^T x and du^T x (two products of the same sizes in one launch), dy^T h.
//
// Bound by the tensor cores from a few hundred tokens on.  Roles per CTA as in the int8 GEMM: warp 0 issues TMA loads, warp 1 owns the
// tensor memory and (in the leading CTA) issues the MMAs, warps 2-9 drain accumulators; two accumulators, so the epilogue of one tile
// runs beside the next tile's products.  Every wait is bounded.
#include <string.h>

#include "cpmk_gated.cuh"
#include "cpmk_tc.cuh"

namespace cpmk {
namespace {

constexpr int kTileR = 256, kTileC = 256;              // outputs (accumulator rows and columns) of a CTA pair's tile
constexpr int kStageK = 64;                            // k per stage: one 128-byte swizzle row of 16-bit elements
constexpr int kStages = 5;
constexpr int kPBytes = 128 * 128;                     // 128 rows of P per CTA and stage
constexpr int kBlockBytes = 64 * 128;                  // 64 rows by 64 k
constexpr int kStageBytes = kPBytes + 2 * kBlockBytes; // and 128 rows of Q
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = (2 + kEpilogueWarps) * 32;
constexpr int kPieceBytes = 32 * 128;                  // a warp's staging tile: 32 rows by 64 columns
constexpr int kPieces = 2;                             // staging tiles per warp
constexpr int kSmemBytes = kStages * kStageBytes + kEpilogueWarps * kPieces * kPieceBytes + 1024 + 256;
constexpr int kTmemColumns = 512;
constexpr int kBandRows = 16;                          // row tiles walked together (below)

constexpr uint32_t kErrLoad = 0x201, kErrFull = 0x202, kErrAccumulator = 0x203, kErrEpilogue = 0x204;

// p, q: boxes of 128 rows by 64 k where one load can have them; q64: boxes of 64 rows (half tiles).  One load per operand and stage: with
// two of 64 rows each the gated product took 489 us instead of 459 (4096 x 4096 x 20480).
struct TcMaps {
    CUtensorMap p[2], q[2], q64[2], out[3];
};

// Tiles are walked in bands of kBandRows row tiles, row by row within a column of the band: the band's rows of P stay in L2 while the
// columns pass by (4096 tokens, gated: bands of 4, 8, 16 rows took 476, 459, 447 us).  The tiles left over by whole waves of the pairs are
// split into halves of 128 accumulator columns when that makes the last wave shorter (2 x left-over <= pairs).
struct TcParams {
    int32_t C;                         // row pitch of g and u (kEpiDact)
    int32_t R;
    int32_t blocks0, blocks;           // k blocks of the first pair of operands, of all
    int32_t tiles_r, tiles_c, per_product;
    int32_t whole, items;              // whole tiles, work items: items - whole halves follow
    int32_t p_boxes, q_boxes;          // loads per 128 rows of P and Q: 1, or 2 for a transposed operand whose rows are no multiple of 64
    const void *g, *u;
    uint32_t *status;
};

struct Item {
    int32_t product, row, col;         // first row; first column of the outputs
    bool half;
};

template <int EPI>
__device__ __forceinline__ Item item_of(const TcParams &prm, int i) {
    Item it;
    it.half = i >= prm.whole;
    int tile = it.half ? prm.whole + ((i - prm.whole) >> 1) : i;
    it.product = tile / prm.per_product;
    tile -= it.product * prm.per_product;
    const int band = tile / (kBandRows * prm.tiles_c), in_band = tile - band * kBandRows * prm.tiles_c;
    const int rows = min(kBandRows, prm.tiles_r - band * kBandRows);
    const int c = in_band / rows;
    it.row = (band * kBandRows + in_band - c * rows) * kTileR;
    constexpr int kWidth = EPI == kEpiGated ? kTileC / 2 : kTileC;
    it.col = c * kWidth + (it.half && ((i - prm.whole) & 1) ? kWidth / 2 : 0);
    return it;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&v);
    }
    return pack_half2(a, b);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (BF16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v));
    return __half22float2(*reinterpret_cast<__half2 *>(&v));
}

// One warp's staging tiles: 32 rows by 64 columns each, 16-byte chunk j of row r at chunk j ^ (r & 7) (no bank conflicts, and what the
// store's 128-byte swizzle expects).  Stores of out-of-range rows and columns are clipped by the hardware.
struct Staging {
    uint32_t base, lane;
    __device__ __forceinline__ void put(int piece, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
        st_shared_v4(base + (uint32_t)piece * kPieceBytes + lane * 128u + (((uint32_t)chunk ^ (lane & 7u)) << 4), a, b, c, d);
    }
    // both tiles are free: the stores out of them have read them
    __device__ __forceinline__ void acquire() const {
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
    }
    __device__ __forceinline__ void ready() const {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    }
    __device__ __forceinline__ void store(int piece, const CUtensorMap *map, int32_t col, int32_t row) const {
        tma_store_3d(map, base + (uint32_t)piece * kPieceBytes, col, row, 0);
    }
};

// 64 columns of plain sums, from tensor memory column `taddr`
template <bool BF16>
__device__ __forceinline__ void stage_sums(const Staging &st, int piece, uint32_t taddr) {
    uint32_t v[2][32];
    tmem_ld_32x32b_x32(taddr, v[0]);
    tmem_ld_32x32b_x32(taddr + 32, v[1]);
    tmem_ld_wait();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack2<BF16>(__uint_as_float(v[s][8 * g + 2 * e]), __uint_as_float(v[s][8 * g + 2 * e + 1]));
            st.put(piece, 4 * s + g, o[0], o[1], o[2], o[3]);
        }
}

// A warp's share of a finished accumulator: 32 rows from `row`, and the columns of its half.
template <bool BF16, int EPI, int ACT>
__device__ __forceinline__ void epilogue(const TcParams &prm, const TcMaps &maps, const Staging &st, uint32_t tmem, const Item &it, int row, int half) {
    const int lane = (int)st.lane;
    if (EPI == kEpiStore) {
        // 128 columns per warp, 64 in a half tile
        const int columns = it.half ? 64 : 128;
        const int col = it.col + half * columns;
        if (col >= prm.C) return;
        st.acquire();
        stage_sums<BF16>(st, 0, tmem + half * columns);
        const bool second = !it.half && col + 64 < prm.C;
        if (second) stage_sums<BF16>(st, 1, tmem + half * columns + 64);
        st.ready();
        if (lane == 0) {
            st.store(0, &maps.out[it.product], col, row);
            if (second) st.store(1, &maps.out[it.product], col + 64, row);
            bulk_commit();
        }
    } else if (EPI == kEpiGated) {
        // whole tile: 64 output columns per warp; half tile: 64 in all, for the first half's warps
        const int up = it.half ? 64 : 128;
        const int col = it.col + half * 64;
        if (col >= prm.C || (it.half && half)) return;
        const uint32_t gate_at = tmem + half * 64;
        st.acquire();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint32_t g[32], u[32];
            tmem_ld_32x32b_x32(gate_at + s * 32, g);
            tmem_ld_32x32b_x32(gate_at + up + s * 32, u);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * k + 2 * e;
                    o[e] = pack2<BF16>(act_value<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]),
                                       act_value<ACT>(__uint_as_float(g[i + 1])) * __uint_as_float(u[i + 1]));
                }
                st.put(0, 4 * s + k, o[0], o[1], o[2], o[3]);
            }
        }
        st.ready();
        if (lane == 0) {
            st.store(0, &maps.out[0], col, row);
            bulk_commit();
        }
        if (prm.g) {                                     // differentiated: the two projections as well
            st.acquire();
            stage_sums<BF16>(st, 0, gate_at);
            stage_sums<BF16>(st, 1, gate_at + up);
            st.ready();
            if (lane == 0) {
                st.store(0, &maps.out[1], col, row);
                st.store(1, &maps.out[2], col, row);
                bulk_commit();
            }
        }
    } else {
        const int pieces = it.half ? 1 : 2;
        for (int p = 0; p < pieces; ++p) {
            const int offset = half * 64 * pieces + p * 64;
            const int col = it.col + offset;
            if (col >= prm.C) return;
            const int64_t at = (int64_t)(row + lane) * prm.C + col;
            const bool in_row = row + lane < prm.R;
            const uint16_t *g_at = static_cast<const uint16_t *>(prm.g) + at, *u_at = static_cast<const uint16_t *>(prm.u) + at;
            st.acquire();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t v[32];
                uint4 g4[4], u4[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {            // C is a multiple of 8: the eight columns are in or out together
                    g4[k] = u4[k] = make_uint4(0u, 0u, 0u, 0u);
                    if (in_row && col + s * 32 + k * 8 < prm.C) {
                        g4[k] = __ldg(reinterpret_cast<const uint4 *>(g_at + s * 32 + k * 8));
                        u4[k] = __ldg(reinterpret_cast<const uint4 *>(u_at + s * 32 + k * 8));
                    }
                }
                tmem_ld_32x32b_x32(tmem + offset + s * 32, v);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t gw[4] = {g4[k].x, g4[k].y, g4[k].z, g4[k].w}, uw[4] = {u4[k].x, u4[k].y, u4[k].z, u4[k].w};
                    uint32_t dg[4], du[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 g2 = unpack2<BF16>(gw[e]), u2 = unpack2<BF16>(uw[e]);
                        const float d0 = __uint_as_float(v[8 * k + 2 * e]), d1 = __uint_as_float(v[8 * k + 2 * e + 1]);
                        float a0, s0, a1, s1;
                        act_value_slope<ACT>(g2.x, a0, s0);
                        act_value_slope<ACT>(g2.y, a1, s1);
                        dg[e] = pack2<BF16>(d0 * u2.x * s0, d1 * u2.y * s1);
                        du[e] = pack2<BF16>(d0 * a0, d1 * a1);
                    }
                    st.put(0, 4 * s + k, dg[0], dg[1], dg[2], dg[3]);
                    st.put(1, 4 * s + k, du[0], du[1], du[2], du[3]);
                }
            }
            st.ready();
            if (lane == 0) {
                st.store(0, &maps.out[0], col, row);
                st.store(1, &maps.out[1], col, row);
                bulk_commit();
            }
        }
    }
}

// Loads the rows of one operand from `row`, k from `k`.  A transposed operand whose rows are a multiple of 64 is mapped as
// (64 rows, k, blocks of 64 rows), so that a box holds several blocks; others as (rows, k), one block per box (`two`: two boxes).
template <bool MN>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap *map, int row, int k, bool two, bool plain, uint32_t bar) {
    if (!MN) tma_load_3d_pair(dst, map, k, row, 0, bar);
    else if (!two && !plain) tma_load_3d_pair(dst, map, 0, k, row / 64, bar);
    else {
        tma_load_3d_pair(dst, map, row, k, 0, bar);
        if (two) tma_load_3d_pair(dst + kBlockBytes, map, row + 64, k, 0, bar);
    }
}

// P_MN / Q_MN: the operand is stored (k, rows) instead of (rows, k).
template <bool BF16, bool P_MN, bool Q_MN, int EPI, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gated_tc_kernel(const __grid_constant__ TcMaps maps, const TcParams prm) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t tiles_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t staging_base = tiles_base + kStages * kStageBytes;
    const uint32_t full_bar = staging_base + kEpilogueWarps * kPieces * kPieceBytes;     // used in the leader only
    const uint32_t empty_bar = full_bar + 8 * kStages;
    const uint32_t acc_full_bar = empty_bar + 8 * kStages;
    const uint32_t acc_empty_bar = acc_full_bar + 16;                                    // used in the leader only
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_raw + (acc_empty_bar + 16 - smem_u32(smem_raw)));
    volatile uint32_t *abort_flag = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full_bar + 8 * a, 1);
            mbar_init(acc_empty_bar + 8 * a, 2 * kEpilogueWarps);                        // the epilogue warps of both CTAs
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemColumns);
    tcgen05_fence_before();
    cluster_sync_all();                                // barriers of both CTAs are initialised before anyone signals them
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (int i = pair; alive && i < prm.items; i += pairs) {
                const Item it = item_of<EPI>(prm, i);
                const int p_row = it.row + (int)rank * 128, q_rows = it.half ? 64 : 128;
                // gated: the same rows of the rank's weight; otherwise the rank's half of the tile's columns
                const int q_row = EPI == kEpiGated ? it.col : it.col + (int)rank * q_rows;
                for (int kb = 0; kb < prm.blocks; ++kb) {
                    if (!mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag, prm.status, kErrLoad)) { alive = false; break; }
                    const bool second = kb >= prm.blocks0;
                    const int k = (second ? kb - prm.blocks0 : kb) * kStageK;
                    const CUtensorMap *pm = &maps.p[second ? 1 : it.product];
                    const int which = EPI == kEpiGated ? (int)rank : second ? 1 : it.product;
                    const CUtensorMap *qm = it.half || (Q_MN && prm.q_boxes == 2) ? &maps.q64[which] : &maps.q[which];
                    const uint32_t dst = tiles_base + stage * kStageBytes, q_dst = dst + kPBytes;
                    if (leader) mbar_expect_tx(full_bar + 8 * stage, 2 * (kPBytes + (uint32_t)(q_rows / 64) * kBlockBytes));
                    const uint32_t bar = map_to_cta(full_bar + 8 * stage, 0);
                    load_rows<P_MN>(dst, pm, p_row, k, P_MN && prm.p_boxes == 2, false, bar);
                    load_rows<Q_MN>(q_dst, qm, q_row, k, Q_MN && prm.q_boxes == 2 && !it.half, Q_MN && prm.q_boxes == 2, bar);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leading CTA only) ----------------
        if (leader && lane == 0) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool alive = true;
            // fp32 accumulator (bits 4-5 = 1), A and B fp16 or bf16 (bits 7-9, 10-12 = 0 or 1), MN-major operands (bits 15, 16),
            // N / 8 at bits 17-22, M / 16 at bits 24-28
            constexpr uint32_t kType = BF16 ? 1u : 0u;
            constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | (P_MN ? (1u << 15) : 0u) | (Q_MN ? (1u << 16) : 0u) |
                                       ((uint32_t)(kTileR >> 4) << 24);
            for (int i = pair; alive && i < prm.items; i += pairs) {
                const uint32_t desc = kDesc | ((uint32_t)((i >= prm.whole ? 128 : 256) >> 3) << 17);
                if (!mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, prm.status, kErrAccumulator)) break;
                tcgen05_fence_after();
                const uint32_t d_tmem = tmem_base + acc * kTileC;
                for (int kb = 0; kb < prm.blocks; ++kb) {
                    if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag, prm.status, kErrFull)) { alive = false; break; }
                    tcgen05_fence_after();
                    const uint32_t src = tiles_base + stage * kStageBytes;
                    const uint64_t pd = P_MN ? make_mnmajor_sw128_desc(src, kBlockBytes) : make_kmajor_sw128_desc(src);
                    const uint64_t qd = Q_MN ? make_mnmajor_sw128_desc(src + kPBytes, kBlockBytes) : make_kmajor_sw128_desc(src + kPBytes);
#pragma unroll
                    for (int j = 0; j < kStageK / 16; ++j)                               // 16 of k: 32 bytes of a row, or 16 rows of 128 bytes
                        umma_f16_pair(d_tmem, pd + (uint64_t)((P_MN ? 128 : 2) * j), qd + (uint64_t)((Q_MN ? 128 : 2) * j), desc, (kb | j) != 0 ? 1u : 0u);
                    umma_commit_pair(empty_bar + 8 * stage, 3);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
                if (!alive) break;
                umma_commit_pair(acc_full_bar + 8 * acc, 3);
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
            }
        }
    } else {
        // ---------------- epilogue (both CTAs; each owns 128 of the tile's 256 rows) ----------------
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const Staging st = {staging_base + (uint32_t)(warp - 2) * kPieces * kPieceBytes, (uint32_t)lane};
        uint32_t acc = 0, acc_phase = 0;
        for (int i = pair; i < prm.items; i += pairs) {
            const Item it = item_of<EPI>(prm, i);
            if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, prm.status, kErrEpilogue)) break;
            tcgen05_fence_after();
            const int row = it.row + (int)rank * 128 + quarter * 32;
            if (row < prm.R)
                epilogue<BF16, EPI, ACT>(prm, maps, st, tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * kTileC, it, row, half);
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar + 8 * acc, 0));
            acc ^= 1u;
            if (acc == 0) acc_phase ^= 1u;
        }
        if (lane == 0) bulk_wait_all();                // this warp's stores have completed
    }

    // ---------------- teardown: neither CTA may leave while its partner can still touch its memory ----------------
    __syncwarp();
    tcgen05_fence_before();
    cluster_sync_all();
    if (*abort_flag) {
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);                                // copies in flight land first
    }
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemColumns);
    }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// An operand of 16-bit elements stored (rows, k), or (k, rows) when transposed: boxes of `box_rows` (64 or 128) rows by 64 k.  A transposed
// operand has 64 rows in a 128-byte swizzle row; as (64 rows, k, blocks of 64 rows) a box can hold two blocks, when there is no partial
// block (it would reach past the tensor's end); otherwise boxes are 64 rows.
bool encode_operand(CUtensorMap *map, const void *ptr, int64_t rows, int64_t k, bool transposed, uint32_t box_rows) {
    if (transposed && rows % 64 == 0) {
        const uint64_t dims[3] = {64, (uint64_t)k, (uint64_t)(rows / 64)}, strides[2] = {(uint64_t)rows * 2, 128};
        const uint32_t box[3] = {64, 64, box_rows / 64};
        return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
    }
    const uint64_t inner = (uint64_t)(transposed ? rows : k), outer = (uint64_t)(transposed ? k : rows);
    const uint64_t dims[3] = {inner, outer, 1}, strides[2] = {inner * 2, inner * outer * 2};
    const uint32_t box[3] = {64, transposed ? 64 : box_rows, 1};
    return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
}
int32_t boxes(int64_t rows, bool transposed) { return transposed && rows % 64 ? 2 : 1; }
bool encode_q(TcMaps *maps, int i, const void *ptr, int64_t rows, int64_t k, bool transposed) {
    return encode_operand(&maps->q[i], ptr, rows, k, transposed, 128) && encode_operand(&maps->q64[i], ptr, rows, k, transposed, 64);
}
// An output (R, C): boxes of 32 rows by 64 columns.
bool encode_output(CUtensorMap *map, void *ptr, int64_t R, int64_t C) {
    const uint64_t dims[3] = {(uint64_t)C, (uint64_t)R, 1}, strides[2] = {(uint64_t)C * 2, (uint64_t)R * (uint64_t)C * 2};
    const uint32_t box[3] = {64, 32, 1};
    return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
}

template <bool BF16, bool P_MN, bool Q_MN, int EPI, int ACT>
int32_t launch(const Call &call, const TcMaps &maps, TcParams prm, int64_t products) {
    auto kernel = gated_tc_kernel<BF16, P_MN, Q_MN, EPI, ACT>;
    CPMK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    const int64_t pairs = call.info.sm_count / 2;        // advisory: a pair that is not resident at launch starts when another retires
    const int64_t per_product = (int64_t)prm.tiles_r * prm.tiles_c, total = per_product * products;
    CPMK_REQUIRE(total < (int64_t(1) << 30), "too many output tiles");
    const int64_t left = total % pairs;
    const bool split = left > 0 && 2 * left <= pairs;
    prm.per_product = (int32_t)per_product;
    prm.whole = (int32_t)(split ? total - left : total);
    prm.items = (int32_t)(split ? total + left : total);
    const unsigned grid = (unsigned)(2 * (prm.items < pairs ? prm.items : pairs));
    kernel<<<grid, kThreads, kSmemBytes, call.stream>>>(maps, prm);
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

int32_t prepare(TcParams *prm, int64_t R, int64_t C, int64_t K0, int64_t K1, int64_t width) {
    uint32_t *status;
    const int32_t rc = get_device_status(&status);
    if (rc) return rc;
    memset(prm, 0, sizeof(*prm));
    prm->R = (int32_t)R;
    prm->C = (int32_t)C;
    prm->blocks0 = (int32_t)ceil_div64(K0, kStageK);
    prm->blocks = prm->blocks0 + (int32_t)ceil_div64(K1, kStageK);
    prm->tiles_r = (int32_t)ceil_div64(R, kTileR);
    prm->tiles_c = (int32_t)ceil_div64(C, width);
    prm->status = status;
    return CPMK_OK;
}

int32_t encode_failed() {
    set_error("cuTensorMapEncodeTiled failed");
    return CPMK_ECUDA;
}

}  // namespace

int32_t tc_product(const Call &call, int32_t R, int32_t C, int32_t K, bool p_t, bool q_t, const void *p0, const void *q0, const void *p1,
                   const void *q1, bool sum, void *out0, void *out1) {
    TcParams prm;
    const int32_t rc = prepare(&prm, R, C, K, sum ? K : 0, kTileC);
    if (rc) return rc;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    bool ok = encode_operand(&maps.p[0], p0, R, K, p_t, 128) && encode_q(&maps, 0, q0, C, K, q_t) && encode_output(&maps.out[0], out0, R, C);
    if (ok && p1) ok = encode_operand(&maps.p[1], p1, R, K, p_t, 128) && encode_q(&maps, 1, q1, C, K, q_t);
    prm.p_boxes = boxes(R, p_t);
    prm.q_boxes = boxes(C, q_t);
    if (ok && out1) ok = encode_output(&maps.out[1], out1, R, C);
    if (!ok) return encode_failed();
    const int64_t products = out1 ? 2 : 1;
    const bool bf16 = call.dtype == CPMK_BF16;
    if (!p_t && !q_t) return bf16 ? launch<true, false, false, kEpiStore, 0>(call, maps, prm, products) : launch<false, false, false, kEpiStore, 0>(call, maps, prm, products);
    if (!p_t) return bf16 ? launch<true, false, true, kEpiStore, 0>(call, maps, prm, products) : launch<false, false, true, kEpiStore, 0>(call, maps, prm, products);
    CPMK_REQUIRE(q_t, "operand order not built");
    return bf16 ? launch<true, true, true, kEpiStore, 0>(call, maps, prm, products) : launch<false, true, true, kEpiStore, 0>(call, maps, prm, products);
}

int32_t tc_gated(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u) {
    TcParams prm;
    const int32_t rc = prepare(&prm, tokens, n, k, 0, kTileC / 2);
    if (rc) return rc;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    bool ok = encode_operand(&maps.p[0], x, tokens, k, false, 128) && encode_q(&maps, 0, wg, n, k, false) && encode_q(&maps, 1, wu, n, k, false) && encode_output(&maps.out[0], h, tokens, n);
    if (ok && g) ok = encode_output(&maps.out[1], g, tokens, n) && encode_output(&maps.out[2], u, tokens, n);
    if (!ok) return encode_failed();
    prm.g = g;
    prm.u = u;
    const bool silu = call.act == CPMK_ACT_SILU;
    if (call.dtype == CPMK_BF16)
        return silu ? launch<true, false, false, kEpiGated, CPMK_ACT_SILU>(call, maps, prm, 1) : launch<true, false, false, kEpiGated, CPMK_ACT_GELU>(call, maps, prm, 1);
    return silu ? launch<false, false, false, kEpiGated, CPMK_ACT_SILU>(call, maps, prm, 1) : launch<false, false, false, kEpiGated, CPMK_ACT_GELU>(call, maps, prm, 1);
}

int32_t tc_dact(const Call &call, int32_t tokens, int32_t n, int32_t m, const void *dy, const void *wd, const void *g, const void *u, void *dg, void *du) {
    TcParams prm;
    const int32_t rc = prepare(&prm, tokens, n, m, 0, kTileC);
    if (rc) return rc;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    if (!(encode_operand(&maps.p[0], dy, tokens, m, false, 128) && encode_q(&maps, 0, wd, n, m, true) && encode_output(&maps.out[0], dg, tokens, n) &&
          encode_output(&maps.out[1], du, tokens, n)))
        return encode_failed();
    prm.q_boxes = boxes(n, true);
    prm.g = g;
    prm.u = u;
    const bool silu = call.act == CPMK_ACT_SILU;
    if (call.dtype == CPMK_BF16)
        return silu ? launch<true, false, true, kEpiDact, CPMK_ACT_SILU>(call, maps, prm, 1) : launch<true, false, true, kEpiDact, CPMK_ACT_GELU>(call, maps, prm, 1);
    return silu ? launch<false, false, true, kEpiDact, CPMK_ACT_SILU>(call, maps, prm, 1) : launch<false, false, true, kEpiDact, CPMK_ACT_GELU>(call, maps, prm, 1);
}

}  // namespace cpmk
