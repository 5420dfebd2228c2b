// The gated feed-forward block's forward products for few tokens (decoding), where the time is that of reading the weights once.
//
// The roles of the operands are swapped: D[weight row, token] = W x^T, so that 128 weight rows fill the tensor core's M and the tokens,
// padded to a multiple of 16, its N (tcgen05.mma.cta_group::1.kind::f16).  A tile is 128 rows of Wd, or 64 rows of Wg above the same 64
// rows of Wu.  All tiles' k blocks form one list that is cut into equal pieces, one per SM: every SM streams the same number of bytes
// through a ring that fills its shared memory, whatever the number of tiles.  A piece that ends inside a tile leaves fp32 partial sums
// in scratch; few_join_kernel adds a tile's pieces in order and applies the activation (or only rounds).  The four kernels of a block
// are launched so that each starts while the one in front drains: the second product's weights are on their way before h is known.
//
// 4096 / 10240, one token: 252 MB of weights, 38 us at the measured copy rate.
#include <string.h>

#include <type_traits>

#include "cpmk_gated.cuh"
#include "cpmk_tc.cuh"

namespace cpmk {
namespace {

constexpr int kRows = 128;                             // weight rows per tile (UMMA M, tensor-memory lanes)
constexpr int kStageK = 64;
constexpr int kWeightBytes = kRows * 128;              // per stage
constexpr int kThreads = 192;                          // warp 0: TMA, warp 1: MMA and tensor memory, warps 2-5: partial sums
constexpr int kRingBytes = 208 * 1024;
constexpr int kMaxStages = 12;
constexpr int kSmemBytes = kRingBytes + 1024 + 512;
constexpr uint32_t kErrLoad = 0x301, kErrFull = 0x302, kErrAccumulator = 0x303, kErrPartial = 0x304;

struct FewMaps {
    CUtensorMap w[2], x;
};
struct FewParams {
    int64_t units;                     // tiles x k blocks
    int32_t blocks;                    // k blocks of a tile
    int32_t tokens, padded;            // padded: to a multiple of 16
    int32_t stages, stage_bytes, tmem_columns;
    int32_t after_prior;               // x is written by the kernel in front of this one
    float *partial;                    // [tile + CTA][token][weight row of the tile]
    uint32_t *status;
};

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// CTA c of G owns the units [c units / G, (c + 1) units / G).
__host__ __device__ __forceinline__ int64_t first_unit(int64_t c, int64_t ctas, int64_t units) { return c * units / ctas; }
__host__ __device__ __forceinline__ int64_t owner_of(int64_t unit, int64_t ctas, int64_t units) { return ((unit + 1) * ctas - 1) / units; }

template <bool BF16, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ FewMaps maps, const FewParams prm) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t full_bar = ring + kRingBytes, empty_bar = full_bar + 8 * kMaxStages, acc_full_bar = empty_bar + 8 * kMaxStages;
    const uint32_t acc_empty_bar = acc_full_bar + 16;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem_raw + (acc_empty_bar + 16 - smem_u32(smem_raw)));
    volatile uint32_t *abort_flag = tmem_slot + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    launch_dependents();
    const int64_t u0 = first_unit(blockIdx.x, gridDim.x, prm.units), u1 = first_unit((int64_t)blockIdx.x + 1, gridDim.x, prm.units);
    const int32_t count = (int32_t)(u1 - u0);
    const int32_t tile0 = (int32_t)(u0 / prm.blocks), block0 = (int32_t)(u0 - (int64_t)tile0 * prm.blocks);
    const int32_t ahead = min(prm.stages, count);
    int tile = tile0, block = block0;                    // the producer's next
    auto load_weights = [&](uint32_t stage) {
        const uint32_t dst = ring + stage * (uint32_t)prm.stage_bytes, bar = full_bar + 8 * stage;
        mbar_expect_tx(bar, (uint32_t)prm.stage_bytes);
        if (GATED) {
            tma_load_3d(dst, &maps.w[0], block * kStageK, tile * 64, 0, bar);
            tma_load_3d(dst + kWeightBytes / 2, &maps.w[1], block * kStageK, tile * 64, 0, bar);
        } else {
            tma_load_3d(dst, &maps.w[0], block * kStageK, tile * kRows, 0, bar);
        }
    };
    auto load_x = [&](uint32_t stage, int x_block) {
        tma_load_3d(ring + stage * (uint32_t)prm.stage_bytes + kWeightBytes, &maps.x, x_block * kStageK, 0, 0, full_bar + 8 * stage);
    };
    auto advance = [&]() {
        if (++block == prm.blocks) { block = 0; ++tile; }
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < prm.stages; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full_bar + 8 * a, 1);
            mbar_init(acc_empty_bar + 8 * a, 4);
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // the first ring's worth of weights is requested before anything else is set up, and before x is there
        for (int i = 0; i < ahead; ++i) {
            load_weights((uint32_t)i);
            advance();
        }
    }
    if (warp == 1) tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), (uint32_t)prm.tmem_columns);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            if (prm.after_prior) wait_for_prior_grid();
            int x_block = block0;
            for (int i = 0; i < ahead; ++i) {
                load_x((uint32_t)i, x_block);
                if (++x_block == prm.blocks) x_block = 0;
            }
            uint32_t stage = 0, phase = 0;               // of the next wait for an empty stage
            for (int i = ahead; i < count; ++i) {
                if (!mbar_wait(empty_bar + 8 * stage, phase, abort_flag, prm.status, kErrLoad)) break;
                load_weights(stage);
                load_x(stage, block);
                advance();
                if (++stage == (uint32_t)prm.stages) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            constexpr uint32_t kType = BF16 ? 1u : 0u;
            const uint32_t desc = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(prm.padded >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
            bool alive = true;
            int block = block0;
            for (int left = count; alive && left > 0;) {
                const int length = min(left, prm.blocks - block);
                if (!mbar_wait(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag, prm.status, kErrAccumulator)) break;
                tcgen05_fence_after();
                const uint32_t d_tmem = tmem_base + acc * (uint32_t)(prm.tmem_columns / 2);
                for (int b = 0; b < length; ++b) {
                    if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag, prm.status, kErrFull)) { alive = false; break; }
                    tcgen05_fence_after();
                    const uint32_t src = ring + stage * (uint32_t)prm.stage_bytes;
                    const uint64_t wd = make_kmajor_sw128_desc(src), xd = make_kmajor_sw128_desc(src + kWeightBytes);
#pragma unroll
                    for (int j = 0; j < kStageK / 16; ++j)
                        umma_f16(d_tmem, wd + (uint64_t)(2 * j), xd + (uint64_t)(2 * j), desc, (b | j) != 0 ? 1u : 0u);
                    umma_commit(empty_bar + 8 * stage);
                    if (++stage == (uint32_t)prm.stages) { stage = 0; phase ^= 1u; }
                }
                if (!alive) break;
                umma_commit(acc_full_bar + 8 * acc);
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
                left -= length;
                block = 0;
            }
        }
    } else {
        const int quarter = warp & 3;
        uint32_t acc = 0, acc_phase = 0;
        int block = block0;
        int64_t slot = (int64_t)tile0 + blockIdx.x;
        for (int left = count; left > 0; ++slot) {
            const int length = min(left, prm.blocks - block);
            if (!mbar_wait(acc_full_bar + 8 * acc, acc_phase, abort_flag, prm.status, kErrPartial)) break;
            tcgen05_fence_after();
            float *to = prm.partial + slot * prm.tokens * kRows + quarter * 32 + lane;
            for (int t0 = 0; t0 < prm.tokens; t0 += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (uint32_t)(prm.tmem_columns / 2) + (uint32_t)t0, v);
                tmem_ld_wait();
#pragma unroll
                for (int t = 0; t < 16; ++t)             // a warp's 32 rows of one token: 128 bytes
                    if (t0 + t < prm.tokens) to[(int64_t)(t0 + t) * kRows] = __uint_as_float(v[t]);
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty_bar + 8 * acc);
            acc ^= 1u;
            if (acc == 0) acc_phase ^= 1u;
            left -= length;
            block = 0;
        }
    }

    __syncwarp();
    tcgen05_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);                                // copies in flight land first
    }
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, (uint32_t)prm.tmem_columns);
    }
}

__device__ __forceinline__ void add4(float4 &a, const float4 &b) {
    a.x += b.x;
    a.y += b.y;
    a.z += b.z;
    a.w += b.w;
}
template <typename T>
__device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
    T v[4] = {from_f32<T>(a), from_f32<T>(b), from_f32<T>(c), from_f32<T>(d)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(v);
}

// Four neighbouring outputs of one token per thread: the sums of their tile's pieces, in order of k.
template <typename T, bool GATED, int ACT>
__global__ void __launch_bounds__(256) few_join_kernel(int32_t tokens, int32_t n, int64_t units, int32_t blocks, int32_t ctas,
                                                       const float *__restrict__ partial, T *__restrict__ out, T *__restrict__ g_out,
                                                       T *__restrict__ u_out) {
    launch_dependents();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int32_t groups = n / 4, token = (int32_t)(i / groups), f = (int32_t)(i - (int64_t)token * groups) * 4;
    constexpr int kWidth = GATED ? 64 : kRows;
    const int32_t tile = f / kWidth;
    const int64_t c0 = owner_of((int64_t)tile * blocks, ctas, units), c1 = owner_of((int64_t)(tile + 1) * blocks - 1, ctas, units);
    wait_for_prior_grid();
    if (token >= tokens) return;
    const float *at = partial + ((c0 + tile) * tokens + token) * kRows + (f - tile * kWidth);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int64_t c = c0; c <= c1; ++c, at += (int64_t)tokens * kRows) {
        add4(a, __ldcg(reinterpret_cast<const float4 *>(at)));
        if (GATED) add4(b, __ldcg(reinterpret_cast<const float4 *>(at + 64)));
    }
    const int64_t to = (int64_t)token * n + f;
    if (!GATED) {
        store4(out + to, a.x, a.y, a.z, a.w);
        return;
    }
    const float2 h0 = both(act_value2<ACT>(f2(a.x, a.y)) * f2(b.x, b.y)), h1 = both(act_value2<ACT>(f2(a.z, a.w)) * f2(b.z, b.w));
    store4(out + to, h0.x, h0.y, h1.x, h1.y);
    if (g_out) {
        store4(g_out + to, a.x, a.y, a.z, a.w);
        store4(u_out + to, b.x, b.y, b.z, b.w);
    }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
struct Plan {
    int64_t tiles, units, bytes;
    int32_t blocks, ctas;
};
// At least four k blocks per CTA: below that the partial sums weigh more than the weights.
Plan plan_of(const DeviceInfo &info, int64_t tokens, int64_t rows, int64_t k, bool gated) {
    Plan p;
    p.tiles = ceil_div64(rows, gated ? 64 : kRows);
    p.blocks = (int32_t)ceil_div64(k, kStageK);
    p.units = p.tiles * p.blocks;
    const int64_t most = ceil_div64(p.units, 4);
    p.ctas = (int32_t)(most < info.sm_count ? most : info.sm_count);
    p.bytes = (p.tiles + p.ctas) * tokens * kRows * (int64_t)sizeof(float);
    return p;
}

// Rows of a (rows, k) matrix of 16-bit elements, `box` of them by 64 k.
bool encode_rows(CUtensorMap *map, const void *ptr, int64_t rows, int64_t k, uint32_t box_rows) {
    const uint64_t dims[3] = {(uint64_t)k, (uint64_t)rows, 1}, strides[2] = {(uint64_t)k * 2, (uint64_t)(rows * k) * 2};
    const uint32_t box[3] = {64, box_rows, 1};
    return encode_tiled_3d(map, 2, ptr, dims, strides, box, true);
}

template <bool BF16, bool GATED>
int32_t run(const Call &call, int32_t tokens, int32_t rows, int32_t k, const void *w0, const void *w1, const void *x, bool after_prior, float *partial,
            void *out, void *g, void *u) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    const Plan plan = plan_of(call.info, tokens, rows, k, GATED);
    FewMaps maps;
    memset(&maps, 0, sizeof(maps));
    FewParams prm;
    memset(&prm, 0, sizeof(prm));
    prm.units = plan.units;
    prm.blocks = plan.blocks;
    prm.tokens = tokens;
    prm.padded = (tokens + 15) / 16 * 16;
    prm.stage_bytes = kWeightBytes + prm.padded * 128;
    prm.stages = kRingBytes / prm.stage_bytes < kMaxStages ? kRingBytes / prm.stage_bytes : kMaxStages;
    prm.tmem_columns = 32;
    while (prm.tmem_columns < 2 * prm.padded) prm.tmem_columns *= 2;
    prm.after_prior = after_prior;
    prm.partial = partial;
    const int32_t rc = status_of(call, &prm.status);
    if (rc) return rc;
    if (!(encode_rows(&maps.w[0], w0, rows, k, GATED ? 64 : kRows) && (!GATED || encode_rows(&maps.w[1], w1, rows, k, 64)) &&
          encode_rows(&maps.x, x, tokens, k, (uint32_t)prm.padded))) {
        set_error("cuTensorMapEncodeTiled failed");
        return CPMK_ECUDA;
    }
    auto kernel = few_kernel<BF16, GATED>;
    CPMK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    if (after_prior) {
        CPMK_CUDA_TRY(launch_after_prior(kernel, dim3(plan.ctas), dim3(kThreads), kSmemBytes, call.stream, maps, prm));
    } else {
        kernel<<<plan.ctas, kThreads, kSmemBytes, call.stream>>>(maps, prm);
        CPMK_LAUNCH_CHECK();
    }
    constexpr int kSilu = GATED ? CPMK_ACT_SILU : CPMK_ACT_GELU;                         // a plain product has no activation
    auto join = call.act == kSilu ? few_join_kernel<T, GATED, kSilu> : few_join_kernel<T, GATED, CPMK_ACT_GELU>;
    CPMK_CUDA_TRY(launch_after_prior(join, dim3((unsigned)ceil_div64((int64_t)tokens * (rows / 4), 256)), dim3(256), 0, call.stream, tokens, rows, plan.units,
                                     plan.blocks, plan.ctas, static_cast<const float *>(partial), static_cast<T *>(out), static_cast<T *>(g),
                                     static_cast<T *>(u)));
    return CPMK_OK;
}

}  // namespace

int64_t few_scratch(const DeviceInfo &info, int32_t tokens, int32_t k, int32_t n, int32_t m) {
    return plan_of(info, tokens, n, k, true).bytes + (m ? plan_of(info, tokens, m, n, false).bytes : 0);
}

int32_t few_gated(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u,
                  void *scratch) {
    float *partial = static_cast<float *>(scratch);
    return call.dtype == CPMK_BF16 ? run<true, true>(call, tokens, n, k, wg, wu, x, false, partial, h, g, u)
                                   : run<false, true>(call, tokens, n, k, wg, wu, x, false, partial, h, g, u);
}

int32_t few_down(const Call &call, int32_t tokens, int32_t k, int32_t n, int32_t m, const void *h, const void *wd, void *y, void *scratch) {
    // scratch of its own: the join of the first product may still read its partial sums
    float *partial = reinterpret_cast<float *>(static_cast<char *>(scratch) + plan_of(call.info, tokens, n, k, true).bytes);
    return call.dtype == CPMK_BF16 ? run<true, false>(call, tokens, m, n, wd, nullptr, h, true, partial, y, nullptr, nullptr)
                                   : run<false, false>(call, tokens, m, n, wd, nullptr, h, true, partial, y, nullptr, nullptr);
}

}  // namespace cpmk
