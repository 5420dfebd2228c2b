// Tensor-core products of the gated feed-forward block: persistent CTA pairs on 256 x 256 tiles (tcgen05.mma.cta_group::2.kind::f16,
// fp16 or bf16 operands, fp32 accumulators in tensor memory), with the block's element-wise work in the epilogue:
//
//   kEpiGated   h = act(x Wg^T) * (x Wu^T).  CTA 0 of the pair stages 128 rows of Wg, CTA 1 the same 128 rows of Wu: the pair's
//               256-column accumulator holds the gate sums in columns 0-127 and the up sums in columns 128-255 of the same outputs, so
//               x is staged once for both and the activation and the product need no exchange.  256 x 128 outputs per tile.
//   kEpiDact    dh = dy Wd stays in tensor memory; the epilogue reads g and u and stores dg = dh u act'(g) and du = dh act(g).
//   kEpiStore   plain products: h Wd^T; dg Wg + du Wu (one accumulator, k runs through the first pair of operands, then the second);
//               dg^T x, du^T x and dy^T h (three products in one launch).
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

constexpr uint32_t kErrLoad = 0x201, kErrFull = 0x202, kErrAccumulator = 0x203, kErrEpilogue = 0x204, kErrInputs = 0x205;

// Boxes of 128 rows by 64 k where one load can have them: with two boxes of 64 rows each the gated product took 489 us instead of 459
// (4096 x 4096 x 20480).
struct TcMaps {
    CUtensorMap p[3], q[3], out[3], in[2];               // in: g and u (kEpiDact)
};

// Whole waves of tiles are walked in bands of kBandRows row tiles, row by row within a column of the band: the band's rows of P stay in
// L2 while the columns pass by (4096 tokens, gated: bands of 4, 8, 16 rows took 476, 459, 447 us).  The tiles that are left over (all
// of them, when there are fewer tiles than pairs) would occupy a part of the SMs for the time of a whole tile.  Where that costs more
// than it takes to join sums (plan_of), their k blocks form one list that is cut into equal pieces, one per pair; a piece leaves
// fp32 partial sums in scratch, tc_join_kernel adds a tile's pieces in order of k and finishes its outputs.
struct TcParams {
    // up to three products of the same k in one launch (kEpiStore): the weights' gradients
    int32_t R[3], C[3], tiles_r[3], tiles_c[3], first_tile[3];
    int32_t p_boxes[3], q_boxes[3];    // loads per 128 rows of P and Q: 1, or 2 for a transposed operand whose rows are no multiple of 64
    int32_t products;
    int32_t blocks0, blocks;           // k blocks of the first pair of operands, of all (two pairs: one product)
    int32_t whole;                     // tiles done whole; the others are split
    int32_t split_tiles, split_pairs;  // how many are split, over how many pairs
    const void *g, *u;                 // kEpiDact: read;  kEpiGated: not null when they are wanted
    float *partial;                    // [split tile + pair][accumulator column][row of the tile]
    uint32_t *status;
};

struct Item {
    int32_t product, row, col;         // first row; first column of the outputs
    int32_t block, count;              // k blocks
    int32_t slot;                      // where the partial sums go, -1 for a whole tile
    int32_t R, C, p_boxes, q_boxes;    // the product's
};

template <int EPI>
__device__ __forceinline__ void place(const TcParams &prm, int tile, Item &it) {
    // selected by comparisons, not by index, so that the parameters stay in the constant bank (indexed, dy^T h took 267 us, not 218)
    const bool b = EPI == kEpiStore && prm.products > 1 && tile >= prm.first_tile[1], c = EPI == kEpiStore && prm.products > 2 && tile >= prm.first_tile[2];
    auto of = [&](const int32_t (&v)[3]) { return c ? v[2] : b ? v[1] : v[0]; };
    it.product = c ? 2 : b ? 1 : 0;
    it.R = of(prm.R);
    it.C = of(prm.C);
    it.p_boxes = of(prm.p_boxes);
    it.q_boxes = of(prm.q_boxes);
    const int tiles_r = of(prm.tiles_r), tiles_c = of(prm.tiles_c);
    tile -= of(prm.first_tile);
    const int band = tile / (kBandRows * tiles_c), in_band = tile - band * kBandRows * tiles_c;
    const int rows = min(kBandRows, tiles_r - band * kBandRows);
    const int col = in_band / rows;
    it.row = (band * kBandRows + in_band - col * rows) * kTileR;
    it.col = col * (EPI == kEpiGated ? kTileC / 2 : kTileC);
}

// Pair p of P owns the units [p units / P, (p + 1) units / P) of the split tiles' k blocks.
__device__ __forceinline__ int first_unit(const TcParams &prm, int pair) {
    return (int)((int64_t)pair * prm.split_tiles * prm.blocks / prm.split_pairs);
}
__device__ __forceinline__ int owner_of(const TcParams &prm, int unit) {
    return (int)((((int64_t)unit + 1) * prm.split_pairs - 1) / ((int64_t)prm.split_tiles * prm.blocks));
}

// A pair's work, in the order in which all its roles go through it.
template <int EPI>
struct Walk {
    const TcParams &prm;
    int tile, pairs, unit, end, slot;
    __device__ __forceinline__ Walk(const TcParams &p, int pair, int n) : prm(p), tile(pair), pairs(n) {
        unit = end = slot = 0;
        if (pair < prm.split_pairs) {
            unit = first_unit(prm, pair);
            end = first_unit(prm, pair + 1);
            slot = pair + unit / prm.blocks;
        }
    }
    __device__ __forceinline__ bool next(Item &it) {
        if (tile < prm.whole) {
            place<EPI>(prm, tile, it);
            tile += pairs;
            it.block = 0;
            it.count = prm.blocks;
            it.slot = -1;
            return true;
        }
        if (unit >= end) return false;
        const int t = unit / prm.blocks;
        place<EPI>(prm, prm.whole + t, it);
        it.block = unit - t * prm.blocks;
        it.count = min(end - unit, prm.blocks - it.block);
        it.slot = slot++;
        unit += it.count;
        return true;
    }
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&v);
    }
    return pack_half2(a, b);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(F2 v) {
    const float2 x = both(v);
    return pack2<BF16>(x.x, x.y);
}
template <bool BF16>
__device__ __forceinline__ F2 unpack2(uint32_t v) {
    const float2 x = BF16 ? __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v)) : __half22float2(*reinterpret_cast<__half2 *>(&v));
    return f2(x.x, x.y);
}

// dg = dh u act'(g), du = dh act(g) for two neighbouring outputs
template <bool BF16, int ACT>
__device__ __forceinline__ void dact_pair(float d0, float d1, uint32_t g, uint32_t u, uint32_t &dg, uint32_t &du) {
    const F2 d = f2(d0, d1);
    F2 value, slope;
    act2<ACT, true>(unpack2<BF16>(g), value, slope);
    dg = pack2<BF16>(d * unpack2<BF16>(u) * slope);
    du = pack2<BF16>(d * value);
}

// One warp's staging tiles: 32 rows by 64 columns each, 16-byte chunk j of row r at chunk j ^ (r & 7) (no bank conflicts, and what the
// store's 128-byte swizzle expects).  Stores of out-of-range rows and columns are clipped by the hardware.
struct Staging {
    uint32_t base, lane;
    __device__ __forceinline__ void put(int piece, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
        st_shared_v4(base + (uint32_t)piece * kPieceBytes + lane * 128u + (((uint32_t)chunk ^ (lane & 7u)) << 4), a, b, c, d);
    }
    __device__ __forceinline__ uint4 get(int piece, int chunk) const {
        return ld_shared_v4(base + (uint32_t)piece * kPieceBytes + lane * 128u + (((uint32_t)chunk ^ (lane & 7u)) << 4));
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

// The epilogues run in rolled loops of 16 columns: unrolled over a tile they were 60 KB of instructions, which a kernel of one tile per
// SM fetches as it goes (dy Wd at 201 tokens, k = 512: 19 us, 12 of them the epilogue of its only tile).

// 64 columns of plain sums, from tensor memory column `taddr`
template <bool BF16>
__device__ __forceinline__ void stage_sums(const Staging &st, int piece, uint32_t taddr) {
#pragma unroll 1
    for (int s = 0; s < 4; ++s) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(taddr + s * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack2<BF16>(__uint_as_float(v[8 * k + 2 * e]), __uint_as_float(v[8 * k + 2 * e + 1]));
            st.put(piece, 2 * s + k, o[0], o[1], o[2], o[3]);
        }
    }
}

// g and u of a warp's 32 rows by 64 columns, loaded into its two staging tiles, where dg and du replace them.  (Read by each lane from its
// row in memory, 16 bytes of 32 lines at a time, they kept the SM's load unit busy for 8 thousand cycles a tile.)
struct DactInputs {
    uint32_t bar, phase;
    __device__ __forceinline__ void request(const Staging &st, const TcMaps &maps, int col, int row) const {
        st.acquire();
        if (st.lane == 0) {
            // the tiles were last touched through the generic proxy: order that before the loads that overwrite them
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_expect_tx(bar, 2 * kPieceBytes);
            tma_load_3d(st.base, &maps.in[0], col, row, 0, bar);
            tma_load_3d(st.base + kPieceBytes, &maps.in[1], col, row, 0, bar);
        }
    }
    __device__ __forceinline__ bool arrived(const Staging &st, volatile uint32_t *abort_flag, uint32_t *status) {
        int ok = 1;
        if (st.lane == 0) ok = mbar_wait(bar, phase, abort_flag, status, kErrInputs) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        (void)mbar_try_wait(bar, phase);                 // every lane observes the completed phase before it reads the tiles
        phase ^= 1u;
        return ok != 0;
    }
};

// A warp's share of a finished accumulator: 32 rows from `row`, and the columns of its half.  False: a wait ran out.
template <bool BF16, int EPI, int ACT>
__device__ __forceinline__ bool epilogue(const TcParams &prm, const TcMaps &maps, const Staging &st, uint32_t tmem, const Item &it, int row, int half,
                                         DactInputs &in, volatile uint32_t *abort_flag) {
    const int lane = (int)st.lane, C = it.C;
    if (EPI == kEpiStore) {                              // 128 columns per warp
        const int col = it.col + half * 128;
        if (col >= C) return true;
        st.acquire();
        stage_sums<BF16>(st, 0, tmem + half * 128);
        const bool second = col + 64 < C;
        if (second) stage_sums<BF16>(st, 1, tmem + half * 128 + 64);
        st.ready();
        if (lane == 0) {
            st.store(0, &maps.out[it.product], col, row);
            if (second) st.store(1, &maps.out[it.product], col + 64, row);
            bulk_commit();
        }
    } else if (EPI == kEpiGated) {                       // 64 output columns per warp: gate sums, and 128 columns on the up sums
        constexpr int up = 128;
        const int col = it.col + half * 64;
        if (col >= C) return true;
        const uint32_t gate_at = tmem + half * 64;
        st.acquire();
#pragma unroll 1
        for (int s = 0; s < 4; ++s) {
            uint32_t g[16], u[16];
            tmem_ld_32x32b_x16(gate_at + s * 16, g);
            tmem_ld_32x32b_x16(gate_at + up + s * 16, u);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 8 * k + 2 * e;
                    o[e] = pack2<BF16>(act_value2<ACT>(f2(__uint_as_float(g[i]), __uint_as_float(g[i + 1]))) *
                                       f2(__uint_as_float(u[i]), __uint_as_float(u[i + 1])));
                }
                st.put(0, 2 * s + k, o[0], o[1], o[2], o[3]);
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
    } else {                                             // 128 columns per warp, 64 at a time
        const int col0 = it.col + half * 128;
#pragma unroll 1
        for (int p = 0; p < 2; ++p) {
            const int col = col0 + p * 64;
            if (col >= C) break;
            if (p) in.request(st, maps, col, row);       // the first were requested before the sums were there
            if (!in.arrived(st, abort_flag, prm.status)) return false;
#pragma unroll 1
            for (int s = 0; s < 4; ++s) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(tmem + half * 128 + p * 64 + s * 16, v);
                const uint4 g4[2] = {st.get(0, 2 * s), st.get(0, 2 * s + 1)}, u4[2] = {st.get(1, 2 * s), st.get(1, 2 * s + 1)};
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t gw[4] = {g4[k].x, g4[k].y, g4[k].z, g4[k].w}, uw[4] = {u4[k].x, u4[k].y, u4[k].z, u4[k].w};
                    uint32_t dg[4], du[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        dact_pair<BF16, ACT>(__uint_as_float(v[8 * k + 2 * e]), __uint_as_float(v[8 * k + 2 * e + 1]), gw[e], uw[e], dg[e], du[e]);
                    st.put(0, 2 * s + k, dg[0], dg[1], dg[2], dg[3]);
                    st.put(1, 2 * s + k, du[0], du[1], du[2], du[3]);
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
    return true;
}

// A warp's share of a piece's partial sums: its 32 rows, its 128 accumulator columns; a column's 32 rows are 128 bytes.
__device__ __forceinline__ void store_partial(const TcParams &prm, uint32_t tmem, const Item &it, int tile_row, int half, int lane) {
    float *to = prm.partial + ((int64_t)it.slot * kTileC + half * 128) * kTileR + tile_row + lane;
#pragma unroll 1
    for (int s = 0; s < 8; ++s, to += 16 * kTileR) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + half * 128 + s * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 16; ++c) __stcg(to + c * kTileR, __uint_as_float(v[c]));
    }
}

// Where one operand's 128 rows of a stage come from.  A transposed operand whose rows are a multiple of 64 is mapped as (64 rows, k,
// blocks of 64 rows), so that a box holds two blocks; others as (rows, k), one block per box.  Everything but k is worked out once per
// tile: the loads are issued by one thread, which has 512 cycles for a stage.
template <bool MN>
struct Source {
    const CUtensorMap *map;
    int32_t row, block;
    bool two;
    __device__ __forceinline__ Source(const CUtensorMap *m, int first_row, int boxes)
        : map(m), row(MN && boxes == 1 ? 0 : first_row), block(MN && boxes == 1 ? first_row / 64 : 0), two(MN && boxes == 2) {}
    __device__ __forceinline__ void load(uint32_t dst, int k, uint32_t bar) const {
        tma_load_3d_pair(dst, map, MN ? row : k, MN ? k : row, block, bar);
        if (MN && two) tma_load_3d_pair(dst + kBlockBytes, map, row + 64, k, 0, bar);
    }
};

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
    const uint32_t in_bar = acc_empty_bar + 16;                                          // one per epilogue warp
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_raw + (in_bar + 8 * kEpilogueWarps - smem_u32(smem_raw)));
    volatile uint32_t *abort_flag = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_cta_rank();
    const bool leader = rank == 0;
    launch_dependents();                               // the join, or the call's next product
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
        for (int w = 0; w < kEpilogueWarps; ++w) mbar_init(in_bar + 8 * w, 1);
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(const_cast<uint32_t *>(tmem_slot)), kTmemColumns);
    tcgen05_fence_before();
    cluster_sync_all();                                // barriers of both CTAs are initialised before anyone signals them
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    wait_for_prior_grid();                             // of the same call: this CTA started when one of its CTAs left the SM

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            const uint32_t leader_bar = map_to_cta(full_bar, 0);
            // k blocks [begin, end) of one pair of operands
            auto stream = [&](const Source<P_MN> &p, const Source<Q_MN> &q, int begin, int end) {
                for (int kb = begin; kb < end; ++kb) {
                    if (!mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag, prm.status, kErrLoad)) return false;
                    const uint32_t dst = tiles_base + stage * kStageBytes;
                    if (leader) mbar_expect_tx(full_bar + 8 * stage, 2 * kStageBytes);
                    p.load(dst, kb * kStageK, leader_bar + 8 * stage);
                    q.load(dst + kPBytes, kb * kStageK, leader_bar + 8 * stage);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
                return true;
            };
            Walk<EPI> walk(prm, pair, pairs);
            Item it;
            while (alive && walk.next(it)) {
                const int p_row = it.row + (int)rank * 128;
                // gated: the same rows of the rank's weight; otherwise the rank's half of the tile's columns
                const int q_row = EPI == kEpiGated ? it.col : it.col + (int)rank * 128;
                const int end = it.block + it.count;
                alive = stream(Source<P_MN>(&maps.p[it.product], p_row, it.p_boxes),
                               Source<Q_MN>(&maps.q[EPI == kEpiGated ? (int)rank : it.product], q_row, it.q_boxes), it.block, min(end, prm.blocks0));
                if (EPI == kEpiStore && alive && end > prm.blocks0)
                    alive = stream(Source<P_MN>(&maps.p[1], p_row, it.p_boxes), Source<Q_MN>(&maps.q[1], q_row, it.q_boxes),
                                   max(it.block - prm.blocks0, 0), end - prm.blocks0);
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
                                       ((uint32_t)(kTileC >> 3) << 17) | ((uint32_t)(kTileR >> 4) << 24);
            Walk<EPI> walk(prm, pair, pairs);
            Item it;
            while (alive && walk.next(it)) {
                if (!mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, prm.status, kErrAccumulator)) break;
                tcgen05_fence_after();
                const uint32_t d_tmem = tmem_base + acc * kTileC;
                for (int kb = 0; kb < it.count; ++kb) {
                    if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag, prm.status, kErrFull)) { alive = false; break; }
                    tcgen05_fence_after();
                    const uint32_t src = tiles_base + stage * kStageBytes;
                    const uint64_t pd = P_MN ? make_mnmajor_sw128_desc(src, kBlockBytes) : make_kmajor_sw128_desc(src);
                    const uint64_t qd = Q_MN ? make_mnmajor_sw128_desc(src + kPBytes, kBlockBytes) : make_kmajor_sw128_desc(src + kPBytes);
#pragma unroll
                    for (int j = 0; j < kStageK / 16; ++j)                               // 16 of k: 32 bytes of a row, or 16 rows of 128 bytes
                        umma_f16_pair(d_tmem, pd + (uint64_t)((P_MN ? 128 : 2) * j), qd + (uint64_t)((Q_MN ? 128 : 2) * j), kDesc, (kb | j) != 0 ? 1u : 0u);
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
        DactInputs in = {in_bar + 8 * (uint32_t)(warp - 2), 0u};
        Walk<EPI> walk(prm, pair, pairs);
        Item it;
        while (walk.next(it)) {
            const int tile_row = (int)rank * 128 + quarter * 32, row = it.row + tile_row;
            if (EPI == kEpiDact && it.slot < 0 && row < it.R && it.col + half * 128 < it.C) in.request(st, maps, it.col + half * 128, row);
            if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, prm.status, kErrEpilogue)) break;
            tcgen05_fence_after();
            const uint32_t tmem = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * kTileC;
            if (row < it.R) {
                if (it.slot >= 0) store_partial(prm, tmem, it, tile_row, half, lane);
                else if (!epilogue<BF16, EPI, ACT>(prm, maps, st, tmem, it, row, half, in, abort_flag)) break;
            }
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

// Finishes the split tiles.  A block has 32 rows by 64 outputs of a tile: a warp 32 rows of 8 neighbouring outputs, so that it reads 128
// bytes per column and piece, and a thread writes 16 bytes.
constexpr int kJoinColumns = 8, kJoinBlockColumns = 64;

template <bool BF16, int EPI, int ACT>
__global__ void __launch_bounds__(256) tc_join_kernel(const TcParams prm, void *out0, void *out1, void *out2) {
    constexpr int kWidth = EPI == kEpiGated ? kTileC / 2 : kTileC, kAcross = kWidth / kJoinBlockColumns, kPerTile = kAcross * (kTileR / 32);
    const int t = blockIdx.x / kPerTile, part = blockIdx.x - t * kPerTile;
    Item it;
    place<EPI>(prm, prm.whole + t, it);
    const int tile_row = part / kAcross * 32 + (threadIdx.x & 31), tile_col = part % kAcross * kJoinBlockColumns + (threadIdx.x >> 5) * kJoinColumns;
    const int row = it.row + tile_row, col = it.col + tile_col;
    const int first = owner_of(prm, t * prm.blocks), last = owner_of(prm, (t + 1) * prm.blocks - 1);
    launch_dependents();
    wait_for_prior_grid();
    const int C = it.C;
    if (row >= it.R || col >= C) return;
    float a[kJoinColumns], b[EPI == kEpiGated ? kJoinColumns : 1];
#pragma unroll
    for (int c = 0; c < kJoinColumns; ++c) a[c] = b[EPI == kEpiGated ? c : 0] = 0.f;
    const float *at = prm.partial + ((int64_t)(first + t) * kTileC + tile_col) * kTileR + tile_row;
    // 32 values in flight per thread: one after the other, a tile of seven pieces took 18 us
    constexpr int kAhead = EPI == kEpiGated ? 2 : 4;
    for (int p = first; p <= last; p += kAhead, at += (int64_t)kAhead * kTileC * kTileR) {
        float v[kAhead][kJoinColumns], w[EPI == kEpiGated ? kAhead : 1][kJoinColumns];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int c = 0; c < kJoinColumns; ++c) {
                v[i][c] = p + i <= last ? __ldcg(at + (int64_t)i * kTileC * kTileR + c * kTileR) : 0.f;
                if (EPI == kEpiGated) w[EPI == kEpiGated ? i : 0][c] = p + i <= last ? __ldcg(at + (int64_t)i * kTileC * kTileR + (128 + c) * kTileR) : 0.f;
            }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int c = 0; c < kJoinColumns; ++c) {
                a[c] += v[i][c];
                if (EPI == kEpiGated) b[EPI == kEpiGated ? c : 0] += w[EPI == kEpiGated ? i : 0][c];
            }
    }
    const int64_t to = (int64_t)row * C + col;
    uint32_t o[3][kJoinColumns / 2];
    if (EPI == kEpiDact) {
#pragma unroll
        for (int k = 0; k < kJoinColumns / 8; ++k) {
            if (col + 8 * k >= C) break;
            const uint4 g4 = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(prm.g) + to + 8 * k));
            const uint4 u4 = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(prm.u) + to + 8 * k));
            const uint32_t gw[4] = {g4.x, g4.y, g4.z, g4.w}, uw[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) dact_pair<BF16, ACT>(a[8 * k + 2 * e], a[8 * k + 2 * e + 1], gw[e], uw[e], o[0][4 * k + e], o[1][4 * k + e]);
        }
    } else {
#pragma unroll
        for (int c = 0; c < kJoinColumns; c += 2) {
            if (EPI == kEpiGated) {
                constexpr int kOne = EPI == kEpiGated ? 1 : 0;
                o[0][c / 2] = pack2<BF16>(act_value2<ACT>(f2(a[c], a[c + 1])) * f2(b[c * kOne], b[(c + 1) * kOne]));
                o[1][c / 2] = pack2<BF16>(a[c], a[c + 1]);
                o[2][c / 2] = pack2<BF16>(b[c * kOne], b[(c + 1) * kOne]);
            } else {
                o[0][c / 2] = pack2<BF16>(a[c], a[c + 1]);
            }
        }
    }
    void *out[3] = {EPI != kEpiStore || it.product == 0 ? out0 : it.product == 1 ? out1 : out2, EPI == kEpiStore ? nullptr : out1, out2};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if ((EPI == kEpiStore && k) || (EPI == kEpiDact && k == 2) || !out[k]) break;
        uint4 *p = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out[k]) + to);
#pragma unroll
        for (int c = 0; c < kJoinColumns / 8; ++c)
            if (col + 8 * c < C) p[c] = make_uint4(o[k][4 * c], o[k][4 * c + 1], o[k][4 * c + 2], o[k][4 * c + 3]);
    }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// An operand of 16-bit elements stored (rows, k), or (k, rows) when transposed: boxes of 128 rows by 64 k.  A transposed operand has 64
// rows in a 128-byte swizzle row; as (64 rows, k, blocks of 64 rows) a box can hold two blocks, when there is no partial block (it
// would reach past the tensor's end); otherwise boxes are 64 rows.
bool encode_operand(CUtensorMap *map, const void *ptr, int64_t rows, int64_t k, bool transposed) {
    if (transposed && rows % 64 == 0) {
        const uint64_t dims[3] = {64, (uint64_t)k, (uint64_t)(rows / 64)}, strides[2] = {(uint64_t)rows * 2, 128};
        const uint32_t box[3] = {64, 64, 2};
        return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
    }
    const uint64_t inner = (uint64_t)(transposed ? rows : k), outer = (uint64_t)(transposed ? k : rows);
    const uint64_t dims[3] = {inner, outer, 1}, strides[2] = {inner * 2, inner * outer * 2};
    const uint32_t box[3] = {64, transposed ? 64u : 128u, 1};
    return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
}
int32_t boxes(int64_t rows, bool transposed) { return transposed && rows % 64 ? 2 : 1; }
// An output (or g, u), (R, C): boxes of 32 rows by 64 columns.
bool encode_output(CUtensorMap *map, const void *ptr, int64_t R, int64_t C) {
    const uint64_t dims[3] = {(uint64_t)C, (uint64_t)R, 1}, strides[2] = {(uint64_t)C * 2, (uint64_t)R * (uint64_t)C * 2};
    const uint32_t box[3] = {64, 32, 1};
    return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
}

struct Plan {
    int64_t blocks0, blocks, whole, split_tiles, split_pairs, bytes;
};
// `total` tiles; K1: the second pair's k when its product is added (0: none).
Plan plan_of(const DeviceInfo &info, int64_t total, int64_t K0, int64_t K1) {
    Plan p;
    p.blocks0 = ceil_div64(K0, kStageK);
    p.blocks = p.blocks0 + ceil_div64(K1, kStageK);
    const int64_t pairs = info.sm_count / 2, left = total % pairs;
    // at least eight k blocks per piece; a k block takes a pair 0.3 us, a piece's sums 1/12 us to write and read back, a join 3 us
    const int64_t most = left * p.blocks / 8, split = most < pairs ? most : pairs;
    const bool pays = left > 0 && split > left && 0.3 * p.blocks > 0.3 * left * p.blocks / split + (left + split) / 12.0 + 3.0;
    p.whole = pays ? total - left : total;
    p.split_tiles = pays ? left : 0;
    p.split_pairs = pays ? split : 0;
    p.bytes = pays ? (left + split) * kTileR * kTileC * (int64_t)sizeof(float) : 0;
    return p;
}
// Tiles of an (R, C) result; width: outputs per tile along C.
int64_t tiles_of(int64_t R, int64_t C, int64_t width) { return ceil_div64(R, kTileR) * ceil_div64(C, width); }

template <bool BF16, bool P_MN, bool Q_MN, int EPI, int ACT>
int32_t launch(const Call &call, const TcMaps &maps, TcParams prm, const Plan &plan, void *out0, void *out1, void *out2) {
    auto kernel = gated_tc_kernel<BF16, P_MN, Q_MN, EPI, ACT>;
    CPMK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    CPMK_REQUIRE(plan.whole + plan.split_tiles < (int64_t(1) << 30) && plan.split_tiles * plan.blocks < (int64_t(1) << 30), "too many output tiles");
    const int64_t pairs = call.info.sm_count / 2;        // advisory: a pair that is not resident at launch starts when another retires
    const int64_t used = plan.whole < pairs ? (plan.whole > plan.split_pairs ? plan.whole : plan.split_pairs) : pairs;
    if (call.launched) CPMK_CUDA_TRY(launch_after_prior(kernel, dim3((unsigned)(2 * used)), dim3(kThreads), kSmemBytes, call.stream, maps, prm));
    else kernel<<<(unsigned)(2 * used), kThreads, kSmemBytes, call.stream>>>(maps, prm);
    CPMK_LAUNCH_CHECK();
    call.launched = true;
    if (!plan.split_tiles) return CPMK_OK;
    const int64_t parts = (EPI == kEpiGated ? kTileC / 2 : kTileC) / kJoinBlockColumns * (kTileR / 32);
    CPMK_CUDA_TRY(launch_after_prior(tc_join_kernel<BF16, EPI, ACT>, dim3((unsigned)(plan.split_tiles * parts)), dim3(256), 0, call.stream, prm, out0, out1,
                                     out2));
    return CPMK_OK;
}

int32_t prepare(const Call &call, TcParams *prm, const Plan &plan, void *scratch) {
    uint32_t *status;
    const int32_t rc = status_of(call, &status);
    if (rc) return rc;
    CPMK_REQUIRE(scratch || !plan.bytes, "scratch is needed");
    memset(prm, 0, sizeof(*prm));
    prm->blocks0 = (int32_t)plan.blocks0;
    prm->blocks = (int32_t)plan.blocks;
    prm->whole = (int32_t)plan.whole;
    prm->split_tiles = (int32_t)plan.split_tiles;
    prm->split_pairs = (int32_t)plan.split_pairs;
    prm->partial = static_cast<float *>(scratch);
    prm->status = status;
    return CPMK_OK;
}
void add_product(TcParams *prm, int64_t R, int64_t C, int64_t width, bool p_t, bool q_t) {
    const int i = prm->products++;
    prm->R[i] = (int32_t)R;
    prm->C[i] = (int32_t)C;
    prm->tiles_r[i] = (int32_t)ceil_div64(R, kTileR);
    prm->tiles_c[i] = (int32_t)ceil_div64(C, width);
    prm->first_tile[i] = i ? prm->first_tile[i - 1] + prm->tiles_r[i - 1] * prm->tiles_c[i - 1] : 0;
    prm->p_boxes[i] = boxes(R, p_t);
    prm->q_boxes[i] = boxes(C, q_t);
}

int32_t encode_failed() {
    set_error("cuTensorMapEncodeTiled failed");
    return CPMK_ECUDA;
}

}  // namespace

int64_t tc_products_scratch(const DeviceInfo &info, int32_t K, const Product *products, int count) {
    int64_t total = 0;
    for (int i = 0; i < count; ++i) total += tiles_of(products[i].R, products[i].C, kTileC);
    return plan_of(info, total, K, 0).bytes;
}
int64_t tc_sum_scratch(const DeviceInfo &info, int32_t R, int32_t C, int32_t K) { return plan_of(info, tiles_of(R, C, kTileC), K, K).bytes; }
int64_t tc_gated_scratch(const DeviceInfo &info, int32_t tokens, int32_t k, int32_t n) {
    return plan_of(info, tiles_of(tokens, n, kTileC / 2), k, 0).bytes;
}
int64_t tc_dact_scratch(const DeviceInfo &info, int32_t tokens, int32_t n, int32_t m) { return plan_of(info, tiles_of(tokens, n, kTileC), m, 0).bytes; }

int32_t tc_products(const Call &call, int32_t K, bool transposed, const Product *products, int count, void *scratch) {
    int64_t total = 0;
    for (int i = 0; i < count; ++i) total += tiles_of(products[i].R, products[i].C, kTileC);
    const Plan plan = plan_of(call.info, total, K, 0);
    TcParams prm;
    const int32_t rc = prepare(call, &prm, plan, scratch);
    if (rc) return rc;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    void *out[3] = {nullptr, nullptr, nullptr};
    for (int i = 0; i < count; ++i) {
        const Product &p = products[i];
        add_product(&prm, p.R, p.C, kTileC, transposed, transposed);
        if (!(encode_operand(&maps.p[i], p.p, p.R, K, transposed) && encode_operand(&maps.q[i], p.q, p.C, K, transposed) &&
              encode_output(&maps.out[i], p.out, p.R, p.C)))
            return encode_failed();
        out[i] = p.out;
    }
#define CPMK_TC_STORE(BF16, MN) return launch<BF16, MN, MN, kEpiStore, 0>(call, maps, prm, plan, out[0], out[1], out[2])
    if (call.dtype == CPMK_BF16 && transposed) CPMK_TC_STORE(true, true);
    if (call.dtype == CPMK_BF16) CPMK_TC_STORE(true, false);
    if (transposed) CPMK_TC_STORE(false, true);
    CPMK_TC_STORE(false, false);
#undef CPMK_TC_STORE
}

int32_t tc_sum(const Call &call, int32_t R, int32_t C, int32_t K, const void *p0, const void *q0, const void *p1, const void *q1, void *out, void *scratch) {
    const Plan plan = plan_of(call.info, tiles_of(R, C, kTileC), K, K);
    TcParams prm;
    const int32_t rc = prepare(call, &prm, plan, scratch);
    if (rc) return rc;
    add_product(&prm, R, C, kTileC, false, true);
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    if (!(encode_operand(&maps.p[0], p0, R, K, false) && encode_operand(&maps.q[0], q0, C, K, true) && encode_operand(&maps.p[1], p1, R, K, false) &&
          encode_operand(&maps.q[1], q1, C, K, true) && encode_output(&maps.out[0], out, R, C)))
        return encode_failed();
    return call.dtype == CPMK_BF16 ? launch<true, false, true, kEpiStore, 0>(call, maps, prm, plan, out, nullptr, nullptr)
                                   : launch<false, false, true, kEpiStore, 0>(call, maps, prm, plan, out, nullptr, nullptr);
}

int32_t tc_gated(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u,
                 void *scratch) {
    const Plan plan = plan_of(call.info, tiles_of(tokens, n, kTileC / 2), k, 0);
    TcParams prm;
    const int32_t rc = prepare(call, &prm, plan, scratch);
    if (rc) return rc;
    add_product(&prm, tokens, n, kTileC / 2, false, false);
    prm.g = g;
    prm.u = u;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    bool ok = encode_operand(&maps.p[0], x, tokens, k, false) && encode_operand(&maps.q[0], wg, n, k, false) &&
              encode_operand(&maps.q[1], wu, n, k, false) && encode_output(&maps.out[0], h, tokens, n);
    if (ok && g) ok = encode_output(&maps.out[1], g, tokens, n) && encode_output(&maps.out[2], u, tokens, n);
    if (!ok) return encode_failed();
#define CPMK_TC_GATED(BF16, ACT) return launch<BF16, false, false, kEpiGated, ACT>(call, maps, prm, plan, h, g, u)
    if (call.dtype == CPMK_BF16 && call.act == CPMK_ACT_SILU) CPMK_TC_GATED(true, CPMK_ACT_SILU);
    if (call.dtype == CPMK_BF16) CPMK_TC_GATED(true, CPMK_ACT_GELU);
    if (call.act == CPMK_ACT_SILU) CPMK_TC_GATED(false, CPMK_ACT_SILU);
    CPMK_TC_GATED(false, CPMK_ACT_GELU);
#undef CPMK_TC_GATED
}

int32_t tc_dact(const Call &call, int32_t tokens, int32_t n, int32_t m, const void *dy, const void *wd, const void *g, const void *u, void *dg, void *du,
                void *scratch) {
    const Plan plan = plan_of(call.info, tiles_of(tokens, n, kTileC), m, 0);
    TcParams prm;
    const int32_t rc = prepare(call, &prm, plan, scratch);
    if (rc) return rc;
    add_product(&prm, tokens, n, kTileC, false, true);
    prm.g = g;
    prm.u = u;
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    if (!(encode_operand(&maps.p[0], dy, tokens, m, false) && encode_operand(&maps.q[0], wd, n, m, true) && encode_output(&maps.out[0], dg, tokens, n) &&
          encode_output(&maps.out[1], du, tokens, n) && encode_output(&maps.in[0], g, tokens, n) && encode_output(&maps.in[1], u, tokens, n)))
        return encode_failed();
#define CPMK_TC_DACT(BF16, ACT) return launch<BF16, false, true, kEpiDact, ACT>(call, maps, prm, plan, dg, du, nullptr)
    if (call.dtype == CPMK_BF16 && call.act == CPMK_ACT_SILU) CPMK_TC_DACT(true, CPMK_ACT_SILU);
    if (call.dtype == CPMK_BF16) CPMK_TC_DACT(true, CPMK_ACT_GELU);
    if (call.act == CPMK_ACT_SILU) CPMK_TC_DACT(false, CPMK_ACT_SILU);
    CPMK_TC_DACT(false, CPMK_ACT_GELU);
#undef CPMK_TC_DACT
}

}  // namespace cpmk
