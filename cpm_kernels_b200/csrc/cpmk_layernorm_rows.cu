// Layer norm of the rows of a (rows, n) matrix, forward and backward, in fp16, bf16 and fp32.
//
//   forward   m = 1/n sum x (0 when rd_mean = 0), r = (1/n sum (x - m)^2 + eps)^-1/2, y = (x - m) r w + b
//   backward  xh = (x - m) r, g = dy w:  dx = r (g - mean(g) [rd_mean] - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// All sums and statistics are fp32; the deviations are taken from the mean before they are squared (no cancellation between
// sum x^2 and n m^2), and every output is rounded once.
#include "cpmk_common.cuh"
#include "cpmk_ptx.cuh"
#include "cpmk_types.cuh"
#include <algorithm>

namespace cpmk {
namespace {

// Bound by memory: forward 2, backward 3 tensors of traffic.  A fixed number of blocks walks the rows, the row held in registers, the
// next row requested before the current one's sums are known.  Forms of each pass, chosen by the row's length and alignment (layout_of):
//   * G threads share a row, NV 16-byte vectors each (VEC = 16 / element size).  Short rows take one warp (no block-wide step), longer
//     ones a block.
//   * the same with single elements (VEC = 1), for rows whose length or address is no multiple of 16 bytes.
//   * forward, 16-bit rows of 1025 to about 16,000 elements (SHIFT): a row whose length is no multiple of 16 bytes starts anywhere in a
//     16-byte vector, but rows 8 apart start at the same place of one.  A block takes every 8th (16th, ...) row, so that the shift and the
//     weights behind a thread's elements stay the same, and reads whole vectors.  Single elements -> shifted vectors, both without the
//     correction of the mean (spread_of; with it 8192 x 2047 takes 28.3 us, 4096 x 4095 24.6, 1027 x 5001 10.8, 2048 x 12289 40.7): 8192 x 2047
//     34.2 -> 25.8 us, 4096 x 4095 34.1 -> 23.7, 1027 x 5001 12.8 -> 10.2, 2048 x 12289 61.4 -> 39.8, one row of 5001 5.5 -> 3.5;
//     but 8192 x 511 12.1 -> 13.2 (in a warp, by single elements: 9.0), 2048 x 20001 65 -> 100 (weights gathered per row), fp32
//     8192 x 1023 18.3 -> 18.1, and the backward pass, which holds two rows, 4096 x 4095 36.6 -> 40.5.
//   * rows too long for that: a block walks the row several times (it is in L1 and L2 after the first), by vectors where it can (1000 x
//     60000 fp16 62 us, by single elements 110).
// load_once, store_once: data that passes through once leaves L2 first, so that the partial sums stay there (16384 x 4096: 79 -> 77 us).
template <typename T, int VEC> struct Pack;
template <typename T> struct Pack<T, 1> {
    T v[1];
    __device__ __forceinline__ void load(const T *p) { v[0] = *p; }
    __device__ __forceinline__ void load_once(const T *p) { v[0] = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = v[0]; }
    __device__ __forceinline__ void store_once(T *p) const { *p = v[0]; }
    __device__ __forceinline__ void clear() { v[0] = from_f32<T>(0.f); }
};
template <typename T, int VEC> struct alignas(16) Pack {
    T v[VEC];
    __device__ __forceinline__ void load(const T *p) { *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void load_once(const T *p) { *reinterpret_cast<uint4 *>(v) = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v); }
    __device__ __forceinline__ void store_once(T *p) const { __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(v)); }
    __device__ __forceinline__ void clear() { *reinterpret_cast<uint4 *>(v) = make_uint4(0u, 0u, 0u, 0u); }
};

// Elements [i, i + VEC) of a row of n.  SHIFT: i may be negative; the vector is read whole, with the neighbouring rows' elements in it,
// unless it reaches over the end of the tensor (`left` elements behind the row's start), and clean() zeroes what is not the row's before
// use.  Both handle whole 32-bit words: single 16-bit elements would be taken apart, and so waited for, where they are read.
template <typename T>
__device__ __forceinline__ uint32_t word_of(const T *row, int i, int64_t left) {
    const uint16_t *bits = reinterpret_cast<const uint16_t *>(row);
    return (i < left ? (uint32_t)bits[i] : 0u) | (i + 1 < left ? (uint32_t)bits[i + 1] << 16 : 0u);
}
template <bool SHIFT, typename T, int VEC>
__device__ __forceinline__ void load_part(Pack<T, VEC> &p, const T *row, int i, int n, int64_t left) {
    if (i >= n) return;
    if (!SHIFT || i + VEC <= left) {
        p.load(row + i);
    } else if constexpr (SHIFT) {
        *reinterpret_cast<uint4 *>(p.v) = make_uint4(word_of(row, i, left), word_of(row, i + 2, left), word_of(row, i + 4, left), word_of(row, i + 6, left));
    }
}
__device__ __forceinline__ uint32_t mask_of(int i, int n) {
    return (i >= 0 && i < n ? 0xffffu : 0u) | (i + 1 >= 0 && i + 1 < n ? 0xffff0000u : 0u);
}
template <bool SHIFT, typename T, int VEC>
__device__ __forceinline__ void clean(Pack<T, VEC> &p, int i, int n) {
    if constexpr (SHIFT) {
        if (i >= 0 && i + VEC <= n) return;
        uint4 *words = reinterpret_cast<uint4 *>(p.v);
        *words = make_uint4(words->x & mask_of(i, n), words->y & mask_of(i + 2, n), words->z & mask_of(i + 4, n), words->w & mask_of(i + 6, n));
    }
}
template <bool SHIFT, typename T, int VEC>
__device__ __forceinline__ void store_part(const Pack<T, VEC> &p, T *row, int i, int n) {
    if (SHIFT ? i >= 0 && i + VEC <= n : i < n) {
        p.store(row + i);
    } else if (SHIFT) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (i + e >= 0 && i + e < n) row[i + e] = p.v[e];
    }
}
// the same elements of a vector that every row shares (weight, bias), whatever its alignment
template <typename T, int VEC>
__device__ __forceinline__ void gather(Pack<T, VEC> &p, const T *v, int i, int n) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.v[e] = i + e >= 0 && i + e < n ? v[i + e] : from_f32<T>(0.f);
}
// VEC floats between registers and shared memory (16-byte aligned when VEC > 1)
template <int VEC>
__device__ __forceinline__ void load_floats(float (&v)[VEC], const float *p) {
    if constexpr (VEC == 1) v[0] = *p;
    else
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4 *>(v + e) = *reinterpret_cast<const float4 *>(p + e);
}
template <int VEC>
__device__ __forceinline__ void store_floats(float *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = v[0];
    else
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4 *>(p + e) = *reinterpret_cast<const float4 *>(v + e);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sums of up to four warps of a block, read by everyone.
__device__ __forceinline__ float four_warps(const float *red) {
    const float4 v = *reinterpret_cast<const float4 *>(red);
    return (v.x + v.y) + (v.z + v.w);
}

// Sum over the threads that share a row (a warp, or the block, of MOST threads at most); every thread gets it.  `red`: one float per warp,
// not written again before the block's next barrier but one (callers alternate between two arrays), so one barrier per sum is enough.
// MOST = 128: `red` is 16-byte aligned, and zero behind the block's last warp.
template <bool BLOCK, int MOST>
__device__ __forceinline__ float row_sum(float v, float *red) {
    v = warp_sum(v);
    if (!BLOCK) return v;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    if (MOST == 128) return four_warps(red);
    return warp_sum(lane < warps ? red[lane] : 0.f);
}
// The sum over a block and what its rounding left out, where the warps' sums are exact: their upper 12 bits and the rest are added up apart,
// each without rounding.  Of up to 16 warps, the lower lanes add up the one and the upper lanes the other.
template <int MOST>
__device__ __forceinline__ float2 row_sum_and_rest(float v, float *red) {
    v = warp_sum(v);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, from = MOST > 512 ? lane : lane & 15;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = from < warps ? red[from] : 0.f;
    float high = __uint_as_float(__float_as_uint(v) & 0xfffff000u), low = v - high;
    if (MOST > 512) {
        high = warp_sum(high);
        low = warp_sum(low);
    } else {
        v = lane & 16 ? low : high;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        low = __shfl_xor_sync(0xffffffffu, v, 16);
        high = lane & 16 ? low : v;
        low = lane & 16 ? v : low;
    }
    const float sum = high + low;
    return make_float2(sum, (high - sum) + low);
}
// Two sums at a time.  Of up to 16 warps, the lower lanes add up one and the upper ones the other.
template <bool BLOCK, int MOST>
__device__ __forceinline__ float2 row_sums(float a, float b, float (*red)[32]) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (!BLOCK) return make_float2(a, b);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) {
        red[0][threadIdx.x >> 5] = a;
        red[1][threadIdx.x >> 5] = b;
    }
    __syncthreads();
    if (MOST == 128) return make_float2(four_warps(red[0]), four_warps(red[1]));
    if (MOST > 512) return make_float2(warp_sum(lane < warps ? red[0][lane] : 0.f), warp_sum(lane < warps ? red[1][lane] : 0.f));
    float v = (lane & 15) < warps ? red[lane >> 4][lane & 15] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const float w = __shfl_xor_sync(0xffffffffu, v, 16);
    return lane & 16 ? make_float2(w, v) : make_float2(v, w);
}

// A row's mean is rounded, and the deviations d from it are off by what it is off by, `off`: some 2^-24 of the values, far more than the
// spread of a row whose values are alike (1000 times 1000.0, mean by a reciprocal: 6e-5, and y 0.02 for 0).  So the variance is
// mean(d^2) - off^2 and y = (d - off) r w + b.  Where off comes from:
//   * 16-bit values that are alike are 12 bits in one unit.  A warp's 1024 of them at most have a sum that is exact, a block's 4096 too, and of
//     more row_sum_and_rest has what the rounding leaves out: off is what is left of the division, (sum + rest - n mean) / n.
//     16384 x 4096 bf16 50.0 us with and without it, 30000 x 256 8.6 -> 9.0, 4096 x 8192 28.7 -> 30.5, 4096 x 4095 23.6 -> 24.6.
//   * fp32 values, and the longest rows: off is the mean of the deviations, a sum of small numbers beside that of the squares.  8192 x 1024
//     fp32 13.3 -> 13.4 us, 8192 x 1023 18.5 -> 21.0; as the only way it took 16384 x 4096 bf16 from 50 to 55, and so did a branch for
//     the rows that need it.
struct Spread {
    float off, rstd;
};
template <bool BLOCK, int MOST, bool EXACT_SUM>
__device__ __forceinline__ Spread spread_of(float left, float sum_d, float sum_d2, int rd_mean, float inv_n, float eps, float (*red)[32]) {
    float off = 0.f, squares;
    if (EXACT_SUM || !rd_mean) {
        off = left * inv_n;                              // 0 without a mean
        squares = row_sum<BLOCK, MOST>(sum_d2, red[0]);
    } else {
        const float2 s = row_sums<BLOCK, MOST>(sum_d, sum_d2, red);
        off = s.x * inv_n;
        squares = s.y;
    }
    // (a NaN stays in `off`; the squares of a row without a mean may be one)
    const float variance = squares * inv_n, reduced = fmaf(-off, off, variance);
    return {off, 1.f / sqrtf((off == 0.f ? variance : fmaxf(reduced, 0.f)) + eps)};
}

// Asks L2 for a row that the block reads next: one request per 128-byte line, no registers.
template <typename T>
__device__ __forceinline__ void prefetch_row(const T *row, int32_t n) {
    const int64_t bytes = (int64_t)n * (int64_t)sizeof(T);
    for (int64_t at = (int64_t)threadIdx.x * 128; at < bytes; at += (int64_t)blockDim.x * 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char *>(row) + at));
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// BLOCK: the whole block shares one row; otherwise each warp has its own.  MOST: threads of a block at most.  With more than 512 that share
// a row (64 registers each) the next row is asked for in L2 instead of in registers.
template <typename T, int VEC, int NV, bool BLOCK, int MOST, bool SHIFT>
__global__ void __launch_bounds__(MOST, MOST == 1024 ? 1 : MOST == 512 ? (VEC * NV > 16 ? 1 : 2) : VEC * NV > 16 ? 5 : 8)
ln_rows_forward_kernel(int32_t rows, int32_t n, float inv_n, float eps, int rd_mean, const T *__restrict__ x, const T *__restrict__ w,
                       const T *__restrict__ b, T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ __align__(16) float red[2][3][32];
    if (BLOCK && MOST == 128) {
        for (int i = threadIdx.x; i < 2 * 3 * 32; i += blockDim.x) red[0][0][i] = 0.f;
        __syncthreads();
    }
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, stride = (BLOCK ? blockDim.x : 32) * VEC;
    const int64_t first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t step = BLOCK ? gridDim.x : (int64_t)gridDim.x * 4;
    const int shift = SHIFT ? (int)((first * n) % VEC) : 0;         // where the walker's rows start in a vector
    // SHIFT: weight and bias are gathered by element, once, and kept in the thread's own slots of shared memory (64 registers hold no more),
    // with four vectors a thread in registers (of which there are 128 then)
    constexpr bool kMany = MOST == 1024;
    constexpr bool kExactSum = sizeof(T) == 2, kRest = kExactSum && BLOCK && MOST > 128;
    static_assert(!SHIFT || (BLOCK && MOST == 512), "shifted rows are a block's of 512 threads at most");
    constexpr bool kKeep = SHIFT && NV <= 2, kHold = SHIFT && NV > 2;
    __shared__ uint4 kept[kKeep ? 2 * NV : 1][kKeep ? 512 : 1];
    Pack<T, VEC> held[kHold ? 2 * NV : 1];
    Pack<T, VEC> in[NV];
    auto request = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) load_part<SHIFT>(in[j], x + row * n, t * VEC + j * stride - shift, n, (rows - row) * n);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        in[j].clear();
        if constexpr (kKeep) {
            Pack<T, VEC> pw, pb;
            gather(pw, w, t * VEC + j * stride - shift, n);
            if (b) gather(pb, b, t * VEC + j * stride - shift, n);
            else pb.clear();
            kept[kKeep ? 2 * j : 0][kKeep ? threadIdx.x : 0] = *reinterpret_cast<const uint4 *>(pw.v);
            kept[kKeep ? 2 * j + 1 : 0][kKeep ? threadIdx.x : 0] = *reinterpret_cast<const uint4 *>(pb.v);
        }
        if constexpr (kHold) {
            gather(held[2 * j], w, t * VEC + j * stride - shift, n);
            if (b) gather(held[2 * j + 1], b, t * VEC + j * stride - shift, n);
            else held[2 * j + 1].clear();
        }
    }
    if (first < rows) request(first);
    int parity = 0;
    for (int64_t row = first; row < rows; row += step, parity ^= 1) {
        float v[NV][VEC], mean = 0.f, left = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            clean<SHIFT>(in[j], t * VEC + j * stride - shift, n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = to_f32(in[j].v[e]);
        }
        if (row + step < rows) {
            if (kMany) prefetch_row(x + (row + step) * n, n);
            else request(row + step);
        }
        if (rd_mean) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += v[j][e];
            float rest = 0.f;
            if constexpr (kRest) {
                const float2 both = row_sum_and_rest<MOST>(s, red[parity][0]);
                s = both.x;
                rest = both.y;
            } else {
                s = row_sum<BLOCK, MOST>(s, red[parity][0]);
            }
            mean = s / (float)n;
            left = fmaf(-mean, (float)n, s) + rest;
        }
        float d = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = t * VEC + j * stride - shift;
                v[j][e] -= mean;
                if (SHIFT ? i + e >= 0 && i + e < n : i < n) {
                    d += v[j][e];
                    q = fmaf(v[j][e], v[j][e], q);
                }
            }
        const Spread spread = spread_of<BLOCK, MOST, kExactSum>(left, d, q, rd_mean, inv_n, eps, red[parity] + 1);
        const float rstd = spread.rstd, back = rd_mean ? -spread.off * rstd : 0.f;
        if (t == 0 && rstd_out) {
            mean_out[row] = mean + spread.off;
            rstd_out[row] = rstd;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride - shift;
            if (i >= n) break;
            Pack<T, VEC> pw, pb, out;
            if constexpr (kKeep) {
                *reinterpret_cast<uint4 *>(pw.v) = kept[kKeep ? 2 * j : 0][kKeep ? threadIdx.x : 0];
                *reinterpret_cast<uint4 *>(pb.v) = kept[kKeep ? 2 * j + 1 : 0][kKeep ? threadIdx.x : 0];
            } else if constexpr (kHold) {
                pw = held[2 * j];
                pb = held[2 * j + 1];
            } else {
                pw.load(w + i);                          // out of L1 after the first row
                if (b) pb.load(b + i);
                else pb.clear();
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) out.v[e] = from_f32<T>(fmaf(fmaf(v[j][e], rstd, back), to_f32(pw.v[e]), to_f32(pb.v[e])));
            store_part<SHIFT>(out, y + row * n, i, n);
        }
        if (kMany && row + step < rows) request(row + step);
    }
}

constexpr int kWideThreads = 512;

template <typename T, int VEC>
__global__ void __launch_bounds__(kWideThreads) ln_rows_forward_wide_kernel(int32_t n, float inv_n, float eps, int rd_mean, const T *__restrict__ x,
                                                                            const T *__restrict__ w, const T *__restrict__ b, T *__restrict__ y,
                                                                            float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[3][32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * n;
    const int32_t first = threadIdx.x * VEC, step = kWideThreads * VEC;
    float mean = 0.f;
    if (rd_mean) {
        float s = 0.f;
        for (int32_t i = first; i < n; i += step) {
            Pack<T, VEC> px;
            px.load(xr + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += to_f32(px.v[e]);
        }
        mean = row_sum<true, kWideThreads>(s, red[0]) / (float)n;
    }
    float sum_d = 0.f, q = 0.f;
    for (int32_t i = first; i < n; i += step) {
        Pack<T, VEC> px;
        px.load(xr + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = to_f32(px.v[e]) - mean;
            sum_d += d;
            q = fmaf(d, d, q);
        }
    }
    const Spread spread = spread_of<true, kWideThreads, false>(0.f, sum_d, q, rd_mean, inv_n, eps, red + 1);
    const float rstd = spread.rstd, back = rd_mean ? -spread.off * rstd : 0.f;
    if (threadIdx.x == 0 && rstd_out) {
        mean_out[row] = mean + spread.off;
        rstd_out[row] = rstd;
    }
    for (int32_t i = first; i < n; i += step) {
        Pack<T, VEC> px, pw, pb, out;
        px.load(xr + i);
        pw.load(w + i);
        if (b) pb.load(b + i);
        else pb.clear();
#pragma unroll
        for (int e = 0; e < VEC; ++e) out.v[e] = from_f32<T>(fmaf(fmaf(to_f32(px.v[e]) - mean, rstd, back), to_f32(pw.v[e]), to_f32(pb.v[e])));
        out.store(y + row * n + i);
    }
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// A fixed number of blocks walks the rows (block p takes rows p, p + blocks, ...); each thread keeps the sums dy xh and dy of its
// columns in registers, and the block leaves one fp32 row of partial sums for dw and one for db: x and dy are read once.
// ln_rows_columns_kernel adds the blocks' rows.
template <typename T, int VEC, int NV, bool BLOCK, bool COLUMNS>
__global__ void __launch_bounds__(BLOCK ? 512 : 256, BLOCK || VEC * NV > 16 ? 1 : 2)
ln_rows_backward_kernel(int32_t rows, int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy, const T *__restrict__ x,
                        const float *__restrict__ mean_in, const float *__restrict__ rstd_in, const T *__restrict__ w, T *__restrict__ dx,
                        float *__restrict__ partial, int32_t pitch) {
    __shared__ float red[2][2][32];
    extern __shared__ __align__(16) float columns[];     // warps with rows of their own: their sums, 2 n each
    if (COLUMNS) launch_dependents();
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, stride = (BLOCK ? blockDim.x : 32) * VEC;
    const int64_t first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t step = BLOCK ? gridDim.x : (int64_t)gridDim.x * (blockDim.x >> 5);
    Pack<T, VEC> pw[NV], px[NV], pd[NV];
    float sw[NV][VEC], sb[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = t * VEC + j * stride;
        if (i < n) pw[j].load(w + i);
        else pw[j].clear();
        px[j].clear();
        pd[j].clear();
#pragma unroll
        for (int e = 0; e < VEC; ++e) sw[j][e] = sb[j][e] = 0.f;
    }
    float mean = 0.f, rstd = 0.f;
    auto request = [&](int64_t row) {
        mean = mean_in[row];
        rstd = rstd_in[row];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride;
            if (i < n) {
                px[j].load_once(x + row * n + i);
                pd[j].load_once(dy + row * n + i);
            }
        }
    };
    if (first < rows) request(first);
    int parity = 0;
    for (int64_t row = first; row < rows; row += step, parity ^= 1) {
        Pack<T, VEC> cx[NV], cd[NV];
        const float r = rstd, m = mean;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            cx[j] = px[j];
            cd[j] = pd[j];
        }
        if (row + step < rows) request(row + step);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = to_f32(cd[j].v[e]);      // zero beyond the row's end
                const float xh = (to_f32(cx[j].v[e]) - m) * r, g = d * to_f32(pw[j].v[e]);
                s1 += g;
                s2 = fmaf(g, xh, s2);
                if (COLUMNS) {
                    sw[j][e] = fmaf(d, xh, sw[j][e]);
                    sb[j][e] += d;
                }
            }
        }
        if (!dx) continue;
        float c1 = warp_sum(s1), c2 = warp_sum(s2);
        if (BLOCK) {
            const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
            if (lane == 0) {
                red[parity][0][threadIdx.x >> 5] = c1;
                red[parity][1][threadIdx.x >> 5] = c2;
            }
            __syncthreads();
            c1 = warp_sum(lane < warps ? red[parity][0][lane] : 0.f);
            c2 = warp_sum(lane < warps ? red[parity][1][lane] : 0.f);
        }
        c1 = rd_mean ? c1 * inv_n : 0.f;
        c2 *= inv_n;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride;
            if (i >= n) break;
            Pack<T, VEC> out;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = (to_f32(cx[j].v[e]) - m) * r, g = to_f32(cd[j].v[e]) * to_f32(pw[j].v[e]);
                out.v[e] = from_f32<T>(r * (g - c1 - xh * c2));
            }
            out.store_once(dx + row * n + i);
        }
    }
    if (!COLUMNS) return;
    float *mine = partial + (int64_t)blockIdx.x * 2 * pitch;
    const int warps = blockDim.x >> 5;
    float *to = BLOCK ? mine : columns + (threadIdx.x >> 5) * 2 * n;
    const int second = BLOCK ? pitch : n;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = t * VEC + j * stride;
        if (i < n) {                                     // 16 bytes at a time: single floats, 32 bytes apart across a warp, took 5 us
            store_floats<VEC>(to + i, sw[j]);
            store_floats<VEC>(to + second + i, sb[j]);
        }
    }
    if (BLOCK) return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) {
        float s = 0.f;
        for (int v = 0; v < warps; ++v) s += columns[v * 2 * n + i];
        mine[i < n ? i : pitch + i - n] = s;
    }
}

// The same for rows of up to 16384 elements or 4096 vectors that do not fit the registers beside their column sums: 1024 threads, the
// block's sums in shared memory (each thread adds to its own columns), the next row asked for in L2.  Per row 16 bytes of shared-memory
// traffic a column, half of what the SM moves while the 12 bytes a column of an fp32 row arrive.
template <typename T, int VEC, int NV, bool COLUMNS>
__global__ void __launch_bounds__(1024, 1) ln_rows_backward_long_kernel(int32_t rows, int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy,
                                                                        const T *__restrict__ x, const float *__restrict__ mean_in,
                                                                        const float *__restrict__ rstd_in, const T *__restrict__ w, T *__restrict__ dx,
                                                                        float *__restrict__ partial, int32_t pitch) {
    __shared__ float red[2][2][32];
    extern __shared__ __align__(16) float columns[];     // 2 n
    if (COLUMNS) launch_dependents();
    const int t = threadIdx.x, stride = 1024 * VEC, lane = t & 31;
    if (COLUMNS)
        for (int i = t; i < 2 * n; i += 1024) columns[i] = 0.f;
    __syncthreads();
    int parity = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, parity ^= 1) {
        const float m = mean_in[row], r = rstd_in[row];
        Pack<T, VEC> px[NV], pd[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride;
            if (i < n) {
                px[j].load_once(x + row * n + i);
                pd[j].load_once(dy + row * n + i);
            }
        }
        if (row + gridDim.x < rows) {
            prefetch_row(x + (row + gridDim.x) * n, n);
            prefetch_row(dy + (row + gridDim.x) * n, n);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride;
            if (i >= n) break;
            Pack<T, VEC> pw;
            pw.load(w + i);
            float aw[VEC], ab[VEC];
            if (COLUMNS) {
                load_floats<VEC>(aw, columns + i);
                load_floats<VEC>(ab, columns + n + i);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = to_f32(pd[j].v[e]), xh = (to_f32(px[j].v[e]) - m) * r, g = d * to_f32(pw.v[e]);
                s1 += g;
                s2 = fmaf(g, xh, s2);
                if (COLUMNS) {
                    aw[e] = fmaf(d, xh, aw[e]);
                    ab[e] += d;
                }
            }
            if (COLUMNS) {
                store_floats<VEC>(columns + i, aw);
                store_floats<VEC>(columns + n + i, ab);
            }
        }
        if (!dx) continue;
        float c1 = warp_sum(s1), c2 = warp_sum(s2);
        if (lane == 0) {
            red[parity][0][t >> 5] = c1;
            red[parity][1][t >> 5] = c2;
        }
        __syncthreads();
        c1 = rd_mean ? warp_sum(red[parity][0][lane]) * inv_n : 0.f;
        c2 = warp_sum(red[parity][1][lane]) * inv_n;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = t * VEC + j * stride;
            if (i >= n) break;
            Pack<T, VEC> pw, out;
            pw.load(w + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = (to_f32(px[j].v[e]) - m) * r, g = to_f32(pd[j].v[e]) * to_f32(pw.v[e]);
                out.v[e] = from_f32<T>(r * (g - c1 - xh * c2));
            }
            out.store_once(dx + row * n + i);
        }
    }
    if (!COLUMNS) return;
    __syncthreads();
    float *mine = partial + (int64_t)blockIdx.x * 2 * pitch;
    for (int i = t; i < n; i += 1024) {
        mine[i] = columns[i];
        mine[pitch + i] = columns[n + i];
    }
}

// Rows too long for registers, dx only: the row is read twice (1000 x 60000 fp16 95 us, by single elements 195).
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) ln_rows_backward_wide_kernel(int32_t rows, int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy,
                                                                     const T *__restrict__ x, const float *__restrict__ mean_in,
                                                                     const float *__restrict__ rstd_in, const T *__restrict__ w, T *__restrict__ dx) {
    __shared__ float red[2][32];
    const int32_t begin = threadIdx.x * VEC, step = 1024 * VEC;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * n, *dyr = dy + row * n;
        const float mean = mean_in[row], rstd = rstd_in[row];
        float s1 = 0.f, s2 = 0.f;
        auto walk = [&](auto use) {
#pragma unroll VEC == 1 ? 4 : 2
            for (int32_t i = begin; i < n; i += step) {
                Pack<T, VEC> px, pd, pw;
                px.load(xr + i);
                pd.load(dyr + i);
                pw.load(w + i);
                use(px, pd, pw, i);
            }
        };
        walk([&](const Pack<T, VEC> &px, const Pack<T, VEC> &pd, const Pack<T, VEC> &pw, int32_t) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = to_f32(pd.v[e]) * to_f32(pw.v[e]);
                s1 += g;
                s2 = fmaf(g, (to_f32(px.v[e]) - mean) * rstd, s2);
            }
        });
        const float c1 = row_sum<true, 1024>(s1, red[0]) * (rd_mean ? inv_n : 0.f);
        const float c2 = row_sum<true, 1024>(s2, red[1]) * inv_n;
        walk([&](const Pack<T, VEC> &px, const Pack<T, VEC> &pd, const Pack<T, VEC> &pw, int32_t i) {
            Pack<T, VEC> out;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = to_f32(pd.v[e]) * to_f32(pw.v[e]), xh = (to_f32(px.v[e]) - mean) * rstd;
                out.v[e] = from_f32<T>(rstd * (g - c1 - xh * c2));
            }
            out.store(dx + row * n + i);
        });
    }
}

// The sums of dw and db alone, where a row's sums find no room beside the row: x and dy are read once more, but without a step that waits
// for a whole row.  A thread has one vector's columns and adds every gridDim.y-th row to them; the block's sums go to row blockIdx.y of
// `partial`.  2048 x 16384 bf16 24.5 us with the kernel that joins them (84 % of the copy rate; 27.9 without load_once, 29.3 with two rows
// on their way).
constexpr int kStripThreads = 128;
template <typename T, int VEC>
__global__ void __launch_bounds__(kStripThreads, 8) ln_rows_strip_kernel(int32_t rows, int32_t n, const T *__restrict__ dy, const T *__restrict__ x,
                                                                         const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                                         float *__restrict__ partial, int32_t pitch) {
    constexpr int kAhead = VEC == 1 ? 8 : 4;             // rows on their way at a time
    launch_dependents();
    const int64_t i = ((int64_t)blockIdx.x * kStripThreads + threadIdx.x) * VEC;
    if (i >= n) return;
    float sw[VEC], sb[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sw[e] = sb[e] = 0.f;
    const int64_t step = (int64_t)gridDim.y;
    int64_t row = blockIdx.y;
    const T *xr = x + row * n + i, *dr = dy + row * n + i;
    auto take = [&](const Pack<T, VEC> &px, const Pack<T, VEC> &pd, float m, float r) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = to_f32(pd.v[e]);
            sw[e] = fmaf(d, (to_f32(px.v[e]) - m) * r, sw[e]);
            sb[e] += d;
        }
    };
    for (; row + (kAhead - 1) * step < rows; row += kAhead * step) {
        Pack<T, VEC> px[kAhead], pd[kAhead];
        float m[kAhead], r[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            px[a].load_once(xr + a * step * n);
            pd[a].load_once(dr + a * step * n);
            m[a] = mean_in[row + a * step];
            r[a] = rstd_in[row + a * step];
        }
        xr += kAhead * step * n;
        dr += kAhead * step * n;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) take(px[a], pd[a], m[a], r[a]);
    }
    for (; row < rows; row += step, xr += step * n, dr += step * n) {
        Pack<T, VEC> px, pd;
        px.load_once(xr);
        pd.load_once(dr);
        take(px, pd, mean_in[row], rstd_in[row]);
    }
    float *mine = partial + (int64_t)blockIdx.y * 2 * pitch + i;
    store_floats<VEC>(mine, sw);
    store_floats<VEC>(mine + pitch, sb);
}

// dw and db: the sums of the blocks' partial rows.  A block has 32 columns: 8 threads of four columns, 64 lanes of rows, the lanes
// added by a fixed tree.  Launched so that it starts while the rows are still walked, and waits for them.
constexpr int kColumnThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kColumnThreads) ln_rows_columns_kernel(int32_t parts, int32_t n, int32_t pitch, const float *__restrict__ partial,
                                                                         T *__restrict__ dw, T *__restrict__ db) {
    __shared__ float sums[64][33];
    T *out = blockIdx.y == 0 ? dw : db;
    wait_for_prior_grid();
    if (!out) return;
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const float *at = partial + (int64_t)blockIdx.y * pitch + blockIdx.x * 32 + tx * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = ty; p < parts; p += 64) {
        const float4 v = *reinterpret_cast<const float4 *>(at + (int64_t)p * 2 * pitch);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    sums[ty][tx * 4] = s.x;
    sums[ty][tx * 4 + 1] = s.y;
    sums[ty][tx * 4 + 2] = s.z;
    sums[ty][tx * 4 + 3] = s.w;
    __syncthreads();
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < 2; ++k) {                        // warp v adds columns v and v + 16
        const int c = (threadIdx.x >> 5) + 16 * k;
        const float v = warp_sum(sums[lane][c] + sums[lane + 32][c]);
        if (lane == 0 && (int)blockIdx.x * 32 + c < n) out[blockIdx.x * 32 + c] = from_f32<T>(v);
    }
}

// ------------------------------------------------------------------------------------------------
// which form
// ------------------------------------------------------------------------------------------------
struct Layout {
    int vec, nv, threads;                // threads: that share a row; 0: the kernel for long rows
};

// `per_warp`: vectors per lane (times four: single elements) up to which a warp takes a row; `most`: the same per thread of a block of
// 512.  Above a warp's reach as few per thread as 128, then 512 threads allow.
Layout layout_of(int32_t n, int per_vector, bool aligned, int per_warp, int most) {
    const bool v = aligned && n % per_vector == 0;
    const int vec = v ? per_vector : 1, units = n / vec, each = v ? 1 : 4;       // 1, 2, 4 vectors; 4, 8, 16 single elements
    auto threads = [&](int nv) { return (units + nv * 32 - 1) / (nv * 32) * 32; };
    for (int i = 1; i <= per_warp; i *= 2)
        if (units <= 32 * i * each) return {vec, i * each, 32};
    if (units <= 128 * each) return {vec, each, threads(each)};
    for (int i = 2; i <= most; i *= 2)
        if (units <= 512 * i * each) return {vec, i * each, threads(i * each)};
    if (units <= 1024 * 4 * each) return {vec, 4 * each, 1024};
    return {vec, 0, 0};
}
// Many rows: few threads with four vectors each, since a row's sums cost every warp that shares it the same (two vectors and twice the
// threads -> four: 30000 x 1024 fp16 31.7 -> 22.3 us, 30000 x 768 26.6 -> 18.5, 16384 x 4096 bf16 53.1 -> 49.2; 148 x 4096 2.8 -> 3.3), unless
// that leaves an eighth of the threads idle (4000 x 2560 10.5 -> 10.9).
Layout forward_layout(int32_t n, int per_vector, bool aligned, bool many_rows) {
    Layout l = layout_of(n, per_vector, aligned, many_rows ? 4 : 2, 4);
    const int units = n / l.vec, threads = (units + 127) / 128 * 32;
    if (many_rows && l.vec > 1 && l.threads > 32 && threads <= 128 && units * 8 >= threads * 4 * 7) l = {l.vec, 4, threads};
    return l;
}
// A column's two sums are registers too: two vectors a thread, or four in a warp (255 registers, 256 threads per SM) where there are rows for
// every warp, for the reason given above: 30000 x 1024 fp16 48.3 -> 39.4 us, 30000 x 768 39.5 -> 34.7, 8192 x 511 16.9 -> 13.0, fp32
// 30000 x 500 47.2 -> 36.7; 200 x 768 4.3 -> 7.4.  Four in a block were no faster (16384 x 4096 77.9 -> 80.9).
Layout backward_layout(const DeviceInfo &info, int32_t rows, int32_t n, int per_vector, bool aligned) {
    return layout_of(n, per_vector, aligned, rows >= 32 * info.sm_count ? 4 : 2, 2);
}

// Blocks of the backward pass: about 512 threads per SM, 256 with four vectors each (the register file holds no more), but at least four
// rows for each that walks rows, so that the partial rows stay small beside the input.
int backward_blocks(const DeviceInfo &info, int32_t rows, const Layout &l) {
    const bool warps = l.threads == 32;
    const int64_t threads = warps ? 256 : l.threads ? l.threads : kWideThreads, most = l.vec * l.nv > 16 ? 256 : 512;
    const int64_t blocks = ceil_div64(rows, warps ? 32 : 4), held = (int64_t)info.sm_count * (threads >= most ? 1 : most / threads);
    return (int)(blocks < held ? blocks : held);
}
int32_t column_pitch(int32_t n) { return (n + 31) / 32 * 32; }

// Whether dw and db take a pass of their own.  Beside a row in shared memory (one pass) -> pass of their own, bf16 or fp16: 2048 x 16384
// 73.7 -> 68.7 us, 2048 x 8200 47.9 -> 46.2, 20 x 16384 24.0 -> 15.9; the rows move half the bytes of their sums there.  fp32 rows and single
// elements keep to one pass (2048 x 8192 fp32 43.0 against 61, 2048 x 12289 bf16 63.5 against 88).
constexpr bool sums_beside_vectors(int element_size) { return element_size == 4; }
bool strips_for(const Layout &l, int element_size) { return l.threads == 0 || (l.threads == 1024 && l.vec > 1 && !sums_beside_vectors(element_size)); }
// Rows of partial sums: one per block, of that pass as many as fill the SMs with strips of `vec` columns a thread, no more than that.
int partial_rows(const DeviceInfo &info, int32_t rows, int32_t n, const Layout &l, int element_size, int vec) {
    const int blocks = backward_blocks(info, rows, l);
    if (!strips_for(l, element_size)) return blocks;
    return (int)std::min<int64_t>(blocks, std::max<int64_t>(1, 8 * info.sm_count / ceil_div64(n, kStripThreads * vec)));
}
// room for those of any type and alignment
int64_t most_partial_rows(const DeviceInfo &info, int32_t rows, int32_t n) {
    int most = 0;
    for (const int element_size : {2, 4})
        for (const bool aligned : {false, true})
            for (const bool strip_aligned : {false, true}) {
                const int per_vector = 16 / element_size, vec = strip_aligned && n % per_vector == 0 ? per_vector : 1;
                most = std::max(most, partial_rows(info, rows, n, backward_layout(info, rows, n, per_vector, aligned), element_size, vec));
            }
    return most;
}

int32_t check_common(DeviceInfo *info, int32_t rows, int32_t n, int32_t dtype) {
    const int32_t rc = current_device_info(info);
    if (rc) return rc;
    CPMK_REQUIRE(rows >= 0 && n >= 1 && n <= (1 << 30), "bad size: rows=%d n=%d (at most 2^30)", rows, n);
    CPMK_REQUIRE(dtype == CPMK_F16 || dtype == CPMK_BF16 || dtype == CPMK_F32, "unknown element type %d", dtype);
    return CPMK_OK;
}

bool aligned_to(const void *p, int64_t a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }

template <typename T>
int32_t forward(const DeviceInfo &info, int32_t rows, int32_t n, const void *xv, float eps, int rd_mean, const void *wv, const void *bv, void *yv,
                float *mean, float *rstd, cudaStream_t stream) {
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *b = static_cast<const T *>(bv);
    T *y = static_cast<T *>(yv);
    constexpr int kVec = 16 / (int)sizeof(T);
    const bool rows_aligned = aligned16(x) && aligned16(y), aligned = rows_aligned && aligned16(w) && aligned16(b);
    const bool many_rows = rows >= 8 * info.sm_count;
    Layout l = forward_layout(n, kVec, aligned, many_rows);
    // shifted rows touch up to a vector more at each end; the layout of the next longer row whose length is whole vectors
    const bool shift = sizeof(T) == 2 && rows_aligned && l.vec == 1 && n > 1024 && n <= 4 * 8 * 512 - 16;
    if (shift) l = forward_layout((n + 2 * (kVec - 1)) / kVec * kVec, kVec, true, false);
    const float inv_n = 1.f / (float)n;
    // as many blocks as the SMs hold (launch bounds: 1024 threads of 64 registers; with four vectors 640 of 102 or, in large blocks, 512 of 128)
    const int64_t threads = l.threads == 32 ? 128 : l.threads, lanes = l.threads == 32 ? 4 : 1;
    const bool narrow = l.vec > 1 && l.nv == 4 && l.threads <= 128 && !shift;
    const int64_t per_sm = l.threads == 0 ? 1 : (l.vec * l.nv <= 16 ? 1024 : narrow ? 640 : 512) / threads;
    const int64_t want = ceil_div64(rows, lanes), most = info.sm_count * (per_sm > 0 ? per_sm : 1);
    const unsigned grid = (unsigned)(want <= most ? want : shift ? most / 8 * 8 : most);         // shifted: one row each, or a multiple of 8 walkers
#define CPMK_LN_FORWARD(VEC, NV, BLOCK, MOST, SHIFT, THREADS) \
    ln_rows_forward_kernel<T, VEC, NV, BLOCK, MOST, SHIFT><<<grid, THREADS, 0, stream>>>(rows, n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd)
#define CPMK_LN_FORWARD_BLOCK(VEC, EACH) \
    if (l.nv == EACH) CPMK_LN_FORWARD(VEC, EACH, true, 512, false, l.threads); \
    else if (l.nv == 2 * EACH) CPMK_LN_FORWARD(VEC, 2 * EACH, true, 512, false, l.threads); \
    else CPMK_LN_FORWARD(VEC, 4 * EACH, true, 512, false, l.threads)
#define CPMK_LN_FORWARD_WARP(VEC, EACH) \
    if (l.nv == EACH) CPMK_LN_FORWARD(VEC, EACH, false, 128, false, 128); \
    else if (l.nv == 2 * EACH) CPMK_LN_FORWARD(VEC, 2 * EACH, false, 128, false, 128); \
    else CPMK_LN_FORWARD(VEC, 4 * EACH, false, 128, false, 128)
    if (l.threads == 0) {
        if (l.vec > 1) ln_rows_forward_wide_kernel<T, kVec><<<rows, kWideThreads, 0, stream>>>(n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd);
        else ln_rows_forward_wide_kernel<T, 1><<<rows, kWideThreads, 0, stream>>>(n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd);
    } else if (shift) {
        if constexpr (sizeof(T) == 2) {                  // (129 vectors and more: two or four a thread)
            if (l.nv == 2) CPMK_LN_FORWARD(kVec, 2, true, 512, true, l.threads);
            else CPMK_LN_FORWARD(kVec, 4, true, 512, true, l.threads);
        }
    } else if (l.vec == kVec) {
        if (l.threads == 32) { CPMK_LN_FORWARD_WARP(kVec, 1); }
        else if (l.threads == 1024) CPMK_LN_FORWARD(kVec, 4, true, 1024, false, 1024);
        else if (narrow) CPMK_LN_FORWARD(kVec, 4, true, 128, false, l.threads);
        else { CPMK_LN_FORWARD_BLOCK(kVec, 1); }
    } else {
        if (l.threads == 32) { CPMK_LN_FORWARD_WARP(1, 4); }
        else if (l.threads == 1024) CPMK_LN_FORWARD(1, 16, true, 1024, false, 1024);
        else { CPMK_LN_FORWARD_BLOCK(1, 4); }
    }
#undef CPMK_LN_FORWARD_BLOCK
#undef CPMK_LN_FORWARD_WARP
#undef CPMK_LN_FORWARD
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

// in shared memory: of a row that 1024 threads take, of eight that a warp takes each
constexpr int kMostSums = 2 * 16384 * (int)sizeof(float), kMostWarpSums = 8 * 2 * 1024 * (int)sizeof(float);

template <typename T, bool COLUMNS>
int32_t backward_rows(const Layout &l, int blocks, int32_t rows, int32_t n, const T *dy, const T *x, int rd_mean, const T *w, const float *mean, const float *rstd,
                      T *dx, float *partial, cudaStream_t stream) {
    constexpr int kVec = 16 / (int)sizeof(T);
    const float inv_n = 1.f / (float)n;
    const int32_t pitch = column_pitch(n);
    const size_t sums = COLUMNS ? 2 * (size_t)n * sizeof(float) : 0;
#define CPMK_LN_BACKWARD(VEC, NV, BLOCK, THREADS, SMEM) \
    ln_rows_backward_kernel<T, VEC, NV, BLOCK, COLUMNS><<<blocks, THREADS, SMEM, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx, partial, pitch)
// (the attribute is the same for every size, so that two threads' calls cannot undo each other's)
#define CPMK_LN_BACKWARD_LONG(VEC, NV) \
    { \
        if constexpr (!COLUMNS || VEC == 1 || sums_beside_vectors(sizeof(T))) { \
            if (COLUMNS) CPMK_CUDA_TRY(cudaFuncSetAttribute(ln_rows_backward_long_kernel<T, VEC, NV, COLUMNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSums)); \
            ln_rows_backward_long_kernel<T, VEC, NV, COLUMNS><<<blocks, 1024, sums, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx, partial, pitch); \
        } \
    }
#define CPMK_LN_BACKWARD_WARP4(VEC, NV) \
    { \
        if (COLUMNS) CPMK_CUDA_TRY(cudaFuncSetAttribute(ln_rows_backward_kernel<T, VEC, NV, false, COLUMNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostWarpSums)); \
        CPMK_LN_BACKWARD(VEC, NV, false, 256, 8 * sums); \
    }
#define CPMK_LN_BACKWARD_IF(VEC, EACH) \
    else if (l.vec == VEC && l.threads == 32 && l.nv == EACH) CPMK_LN_BACKWARD(VEC, EACH, false, 256, 8 * sums); \
    else if (l.vec == VEC && l.threads == 32 && l.nv == 2 * EACH) CPMK_LN_BACKWARD(VEC, 2 * EACH, false, 256, 8 * sums); \
    else if (l.vec == VEC && l.threads == 32) CPMK_LN_BACKWARD_WARP4(VEC, 4 * EACH) \
    else if (l.vec == VEC && l.threads == 1024) CPMK_LN_BACKWARD_LONG(VEC, 4 * EACH) \
    else if (l.vec == VEC && l.nv == EACH) CPMK_LN_BACKWARD(VEC, EACH, true, l.threads, 0); \
    else if (l.vec == VEC) CPMK_LN_BACKWARD(VEC, 2 * EACH, true, l.threads, 0);
    if (l.threads == 0 && l.vec > 1) ln_rows_backward_wide_kernel<T, kVec><<<blocks, 1024, 0, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx);
    else if (l.threads == 0) ln_rows_backward_wide_kernel<T, 1><<<blocks, 1024, 0, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx);
    CPMK_LN_BACKWARD_IF(kVec, 1)
    CPMK_LN_BACKWARD_IF(1, 4)
#undef CPMK_LN_BACKWARD_IF
#undef CPMK_LN_BACKWARD_LONG
#undef CPMK_LN_BACKWARD_WARP4
#undef CPMK_LN_BACKWARD
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

template <typename T>
int32_t backward(const DeviceInfo &info, int32_t rows, int32_t n, const void *dyv, const void *xv, int rd_mean, const void *wv, const float *mean,
                 const float *rstd, void *dxv, void *dw, void *db, float *partial, cudaStream_t stream) {
    const T *dy = static_cast<const T *>(dyv), *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    T *dx = static_cast<T *>(dxv);
    constexpr int kVec = 16 / (int)sizeof(T);
    const Layout l = backward_layout(info, rows, n, kVec, aligned16(x) && aligned16(dy) && aligned16(w) && aligned16(dx));
    const int blocks = backward_blocks(info, rows, l);
    const bool sums = dw || db, strips = sums && strips_for(l, sizeof(T));
    const int vec = n % kVec == 0 && aligned16(x) && aligned16(dy) ? kVec : 1, parts = partial_rows(info, rows, n, l, sizeof(T), vec);
    int32_t rc = CPMK_OK;
    if (strips) {
        const int64_t across = ceil_div64(n, kStripThreads * vec);
        if (vec > 1) ln_rows_strip_kernel<T, kVec><<<dim3((unsigned)across, (unsigned)parts), kStripThreads, 0, stream>>>(rows, n, dy, x, mean, rstd, partial, column_pitch(n));
        else ln_rows_strip_kernel<T, 1><<<dim3((unsigned)across, (unsigned)parts), kStripThreads, 0, stream>>>(rows, n, dy, x, mean, rstd, partial, column_pitch(n));
        CPMK_LAUNCH_CHECK();
    } else if (sums) {
        rc = backward_rows<T, true>(l, blocks, rows, n, dy, x, rd_mean, w, mean, rstd, dx, partial, stream);
        if (rc) return rc;
    }
    if (sums)
        CPMK_CUDA_TRY(launch_after_prior(ln_rows_columns_kernel<T>, dim3((n + 31) / 32, 2), dim3(kColumnThreads), 0, stream, parts, n, column_pitch(n),
                                         static_cast<const float *>(partial), static_cast<T *>(dw), static_cast<T *>(db)));
    if (dx && (strips || !sums)) rc = backward_rows<T, false>(l, blocks, rows, n, dy, x, rd_mean, w, mean, rstd, dx, nullptr, stream);
    return rc;
}

}  // namespace
}  // namespace cpmk

using namespace cpmk;

extern "C" {

int32_t cpmk_layernorm_rows_forward(int32_t rows, int32_t n, int32_t dtype, const void *x, float eps, int32_t rd_mean, const void *weight,
                                    const void *bias, void *y, void *mean, void *rstd, cpmk_stream_t stream) {
    DeviceInfo info;
    const int32_t rc = check_common(&info, rows, n, dtype);
    if (rc) return rc;
    CPMK_REQUIRE(eps >= 0.f, "eps must not be negative");
    if (rows == 0) return CPMK_OK;
    CPMK_REQUIRE(x && weight && y, "null pointer");
    CPMK_REQUIRE((mean == nullptr) == (rstd == nullptr), "mean and rstd are wanted together or not at all");
    const int64_t es = dtype_size(dtype);
    CPMK_REQUIRE(aligned_to(x, es) && aligned_to(weight, es) && aligned_to(y, es) && aligned_to(bias, es) && aligned_to(mean, 4) && aligned_to(rstd, 4),
                 "misaligned pointer");
    const cudaStream_t s = as_stream(stream);
    float *m = static_cast<float *>(mean), *r = static_cast<float *>(rstd);
    if (dtype == CPMK_F16) return forward<__half>(info, rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
    if (dtype == CPMK_BF16) return forward<__nv_bfloat16>(info, rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
    return forward<float>(info, rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
}

int32_t cpmk_layernorm_rows_backward_scratch(int32_t rows, int32_t n, int64_t *bytes) {
    DeviceInfo info;
    const int32_t rc = check_common(&info, rows, n, CPMK_F16);
    if (rc) return rc;
    CPMK_REQUIRE(bytes, "null pointer");
    *bytes = most_partial_rows(info, rows, n) * 2 * column_pitch(n) * (int64_t)sizeof(float);
    return CPMK_OK;
}

int32_t cpmk_layernorm_rows_backward(int32_t rows, int32_t n, int32_t dtype, const void *dy, const void *x, int32_t rd_mean, const void *weight,
                                     const void *mean, const void *rstd, void *dx, void *dweight, void *dbias, void *scratch, cpmk_stream_t stream) {
    DeviceInfo info;
    const int32_t rc = check_common(&info, rows, n, dtype);
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return CPMK_OK;
    const int64_t es = dtype_size(dtype);
    const cudaStream_t s = as_stream(stream);
    if (rows == 0) {                                   // no rows: the sums over them are zero
        if (dweight) CPMK_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)n * es, s));
        if (dbias) CPMK_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)n * es, s));
        return CPMK_OK;
    }
    CPMK_REQUIRE(dy && x && weight && mean && rstd, "null pointer");
    CPMK_REQUIRE(aligned_to(dy, es) && aligned_to(x, es) && aligned_to(weight, es) && aligned_to(dx, es) && aligned_to(dweight, es) &&
                     aligned_to(dbias, es) && aligned_to(mean, 4) && aligned_to(rstd, 4) && aligned_to(scratch, 16),
                 "misaligned pointer");
    CPMK_REQUIRE(scratch || (!dweight && !dbias), "the sums over the rows need scratch");
    const float *m = static_cast<const float *>(mean), *r = static_cast<const float *>(rstd);
    float *part = static_cast<float *>(scratch);
    if (dtype == CPMK_F16) return backward<__half>(info, rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, part, s);
    if (dtype == CPMK_BF16) return backward<__nv_bfloat16>(info, rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, part, s);
    return backward<float>(info, rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, part, s);
}

}  // extern "C"
