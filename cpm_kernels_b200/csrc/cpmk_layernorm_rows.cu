// Layer norm of the rows of a (rows, n) matrix, forward and backward, in fp16, bf16 and fp32.
//
//   forward   m = 1/n sum x (0 when rd_mean = 0), r = (1/n sum (x - m)^2 + eps)^-1/2, y = (x - m) r w + b
//   backward  xh = (x - m) r, g = dy w:  dx = r (g - mean(g) [rd_mean] - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// All sums and statistics are fp32; the deviations are taken from the mean before they are squared (no cancellation between
// sum x^2 and n m^2), and every output is rounded once.
#include "cpmk_common.cuh"
#include "cpmk_types.cuh"

namespace cpmk {
namespace {

// Three forms of each pass, chosen by the row's length and alignment (layout_of):
//   * 16-byte vectors, the row in registers: G threads share a row, NV vectors each.  Rows of up to 1024 16-bit elements take one
//     warp (no block-wide step), longer ones a block.
//   * the same with single elements (VEC = 1), for rows whose length or address is no multiple of 16 bytes.
//   * rows too long for that: a block walks the row several times (they are in L1 and L2 after the first).
template <typename T, int VEC> struct Pack;
template <typename T> struct Pack<T, 1> {
    T v[1];
    __device__ __forceinline__ void load(const T *p) { v[0] = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = v[0]; }
    __device__ __forceinline__ void clear() { v[0] = from_f32<T>(0.f); }
};
template <typename T, int VEC> struct alignas(16) Pack {
    T v[VEC];
    __device__ __forceinline__ void load(const T *p) { *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(v); }
    __device__ __forceinline__ void clear() { *reinterpret_cast<uint4 *>(v) = make_uint4(0u, 0u, 0u, 0u); }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the threads that share a row (a warp, or the block); every thread gets it.  `red`: one float per warp, not written again
// before the block's next barrier but one (callers alternate between two arrays), so one barrier per sum is enough.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float *red) {
    v = warp_sum(v);
    if (!BLOCK) return v;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < warps ? red[lane] : 0.f);
}

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// BLOCK: the whole block shares one row; otherwise each warp has its own.
template <typename T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 128) ln_rows_forward_kernel(int32_t rows, int32_t n, float inv_n, float eps, int rd_mean,
                                                                            const T *__restrict__ x, const T *__restrict__ w, const T *__restrict__ b,
                                                                            T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[2][32];
    const int64_t row = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;                            // whole warps only
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, stride = (BLOCK ? blockDim.x : 32) * VEC;
    const T *xr = x + row * n;
    Pack<T, VEC> in[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = t * VEC + j * stride;
        if (i < n) in[j].load(xr + i);
        else in[j].clear();
    }
    float v[NV][VEC], mean = 0.f;
    if (rd_mean) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += to_f32(in[j].v[e]);
        mean = row_sum<BLOCK>(s, red[0]) * inv_n;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[j][e] = to_f32(in[j].v[e]) - mean;
            if (t * VEC + j * stride < n) q = fmaf(v[j][e], v[j][e], q);
        }
    const float rstd = 1.f / sqrtf(row_sum<BLOCK>(q, red[1]) * inv_n + eps);
    if (t == 0 && rstd_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = t * VEC + j * stride;
        if (i >= n) break;
        Pack<T, VEC> pw, pb, out;
        pw.load(w + i);
        if (b) pb.load(b + i);
        else pb.clear();
#pragma unroll
        for (int e = 0; e < VEC; ++e) out.v[e] = from_f32<T>(fmaf(v[j][e] * rstd, to_f32(pw.v[e]), to_f32(pb.v[e])));
        out.store(y + row * n + i);
    }
}

constexpr int kWideThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kWideThreads) ln_rows_forward_wide_kernel(int32_t n, float inv_n, float eps, int rd_mean, const T *__restrict__ x,
                                                                            const T *__restrict__ w, const T *__restrict__ b, T *__restrict__ y,
                                                                            float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[2][32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * n;
    float mean = 0.f;
    if (rd_mean) {
        float s = 0.f;
        for (int i = threadIdx.x; i < n; i += kWideThreads) s += to_f32(xr[i]);
        mean = row_sum<true>(s, red[0]) * inv_n;
    }
    float q = 0.f;
    for (int i = threadIdx.x; i < n; i += kWideThreads) {
        const float d = to_f32(xr[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<true>(q, red[1]) * inv_n + eps);
    if (threadIdx.x == 0 && rstd_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int i = threadIdx.x; i < n; i += kWideThreads)
        y[row * n + i] = from_f32<T>(fmaf((to_f32(xr[i]) - mean) * rstd, to_f32(w[i]), b ? to_f32(b[i]) : 0.f));
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// A fixed number of blocks walks the rows (block p takes rows p, p + blocks, ...); each thread keeps the sums dy xh and dy of its
// columns in registers, and the block leaves one fp32 row of partial sums for dw and one for db: x and dy are read once.
// ln_rows_columns_kernel adds the blocks' rows.  Up to two vectors per thread the next row's x and dy are requested before the current
// row's sums are known; with four, those registers (and the weight's) are not there, and the block's other half hides the latency.
template <typename T, int VEC, int NV, bool BLOCK, bool COLUMNS>
__global__ void __launch_bounds__(BLOCK ? 512 : 256, BLOCK ? 1 : 2)
ln_rows_backward_kernel(int32_t rows, int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy, const T *__restrict__ x,
                        const float *__restrict__ mean_in, const float *__restrict__ rstd_in, const T *__restrict__ w, T *__restrict__ dx,
                        float *__restrict__ partial) {
    __shared__ float red[2][2][32];
    extern __shared__ float columns[];                   // warps with rows of their own: the block's sums, 2 n
    constexpr bool kAhead = VEC * NV <= 16;
    const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, stride = (BLOCK ? blockDim.x : 32) * VEC;
    const int64_t first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t step = BLOCK ? gridDim.x : (int64_t)gridDim.x * (blockDim.x >> 5);
    Pack<T, VEC> kept[kAhead ? NV : 1], px[NV], pd[NV];
    float sw[NV][VEC], sb[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = t * VEC + j * stride;
        if (kAhead) {
            if (i < n) kept[kAhead ? j : 0].load(w + i);
            else kept[kAhead ? j : 0].clear();
        }
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
                px[j].load(x + row * n + i);
                pd[j].load(dy + row * n + i);
            }
        }
    };
    if (kAhead && first < rows) request(first);
    int parity = 0;
    for (int64_t row = first; row < rows; row += step, parity ^= 1) {
        if (!kAhead) request(row);
        Pack<T, VEC> cx[NV], cd[NV];
        const float r = rstd, m = mean;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            cx[j] = px[j];
            cd[j] = pd[j];
        }
        if (kAhead && row + step < rows) request(row + step);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Pack<T, VEC> pw;
            const int i = t * VEC + j * stride;
            if (kAhead) pw = kept[kAhead ? j : 0];
            else if (i < n) pw.load(w + i);
            else pw.clear();
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = to_f32(cd[j].v[e]);      // zero beyond the row's end
                const float xh = (to_f32(cx[j].v[e]) - m) * r, g = d * to_f32(pw.v[e]);
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
            Pack<T, VEC> pw, out;
            if (kAhead) pw = kept[kAhead ? j : 0];
            else pw.load(w + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float xh = (to_f32(cx[j].v[e]) - m) * r, g = to_f32(cd[j].v[e]) * to_f32(pw.v[e]);
                out.v[e] = from_f32<T>(r * (g - c1 - xh * c2));
            }
            out.store(dx + row * n + i);
        }
    }
    if (!COLUMNS) return;
    float *mine = partial + (int64_t)blockIdx.x * 2 * n;
    if (BLOCK) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int i = t * VEC + j * stride + e;
                if (i < n) {
                    mine[i] = sw[j][e];
                    mine[n + i] = sb[j][e];
                }
            }
        return;
    }
    // one warp after the other adds its sums: the order does not depend on timing
    for (int turn = 0; turn < (int)(blockDim.x >> 5); ++turn) {
        if ((int)(threadIdx.x >> 5) == turn) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = t * VEC + j * stride + e;
                    if (i < n) {
                        columns[i] = turn ? columns[i] + sw[j][e] : sw[j][e];
                        columns[n + i] = turn ? columns[n + i] + sb[j][e] : sb[j][e];
                    }
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) mine[i] = columns[i];
}

// Long rows: the block's partial sums lie in its own rows of `partial`, where each thread adds to the columns it owns.
template <typename T, bool COLUMNS>
__global__ void __launch_bounds__(kWideThreads) ln_rows_backward_wide_kernel(int32_t rows, int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy,
                                                                             const T *__restrict__ x, const float *__restrict__ mean_in,
                                                                             const float *__restrict__ rstd_in, const T *__restrict__ w,
                                                                             T *__restrict__ dx, float *__restrict__ partial) {
    __shared__ float red[2][32];
    float *mine = COLUMNS ? partial + (int64_t)blockIdx.x * 2 * n : nullptr;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * n, *dyr = dy + row * n;
        const float mean = mean_in[row], rstd = rstd_in[row];
        float s1 = 0.f, s2 = 0.f;
        for (int i = threadIdx.x; i < n; i += kWideThreads) {
            const float d = to_f32(dyr[i]), g = d * to_f32(w[i]), xh = (to_f32(xr[i]) - mean) * rstd;
            s1 += g;
            s2 = fmaf(g, xh, s2);
            if (COLUMNS) {
                mine[i] = row == blockIdx.x ? d * xh : fmaf(d, xh, mine[i]);
                mine[n + i] = row == blockIdx.x ? d : mine[n + i] + d;
            }
        }
        if (!dx) continue;
        const float c1 = row_sum<true>(s1, red[0]) * (rd_mean ? inv_n : 0.f);
        const float c2 = row_sum<true>(s2, red[1]) * inv_n;
        for (int i = threadIdx.x; i < n; i += kWideThreads) {
            const float g = to_f32(dyr[i]) * to_f32(w[i]), xh = (to_f32(xr[i]) - mean) * rstd;
            dx[row * n + i] = from_f32<T>(rstd * (g - c1 - xh * c2));
        }
    }
}

// dw and db: the sums of the blocks' partial rows, 32 columns and 32 lanes of rows per block, lanes added by a fixed tree.
template <typename T>
__global__ void __launch_bounds__(1024) ln_rows_columns_kernel(int32_t parts, int32_t n, const float *__restrict__ partial, T *__restrict__ dw,
                                                               T *__restrict__ db) {
    __shared__ float sums[32][33];
    T *out = blockIdx.y == 0 ? dw : db;
    if (!out) return;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + tx;
    float s = 0.f;
    if (c < n)
        for (int p = ty; p < parts; p += 32) s += partial[((int64_t)p * 2 + blockIdx.y) * n + c];
    sums[ty][tx] = s;
    __syncthreads();
    s = warp_sum(sums[tx][ty]);                          // warp ty holds column ty of the block
    if (tx == 0 && (int)blockIdx.x * 32 + ty < n) out[blockIdx.x * 32 + ty] = from_f32<T>(s);
}

// ------------------------------------------------------------------------------------------------
// which form
// ------------------------------------------------------------------------------------------------
struct Layout {
    int vec, nv, threads;                // threads: that share a row; 0: the kernel for long rows
};

// `most`: threads per row at most; `per_warp`: elements (single ones) or vectors per lane up to which a warp takes a row.  Above that
// as few per thread as the threads allow.
Layout layout_of(int32_t n, int per_vector, bool aligned, int per_warp, int most) {
    const bool v = aligned && n % per_vector == 0;
    const int vec = v ? per_vector : 1, units = n / vec, each = v ? 1 : 4;       // 1, 2, 4 vectors; 4, 8, 16 single elements
    for (int i = 1; i <= per_warp; i *= 2)
        if (units <= 32 * i * each) return {vec, i * each, 32};
    if (units <= 128 * each) return {vec, each, (units + each * 32 - 1) / (each * 32) * 32};
    for (int i = 2; i <= 4; i *= 2)
        if (units <= most * i * each) return {vec, i * each, (units + i * each * 32 - 1) / (i * each * 32) * 32};
    return {1, 0, 0};
}
// backward: a warp takes up to two vectors per lane (a column's two sums are registers too), a block of 512 threads the rest
Layout backward_layout(int32_t n, int per_vector, bool aligned) { return layout_of(n, per_vector, aligned, 2, 512); }

// Blocks of the backward pass: about 512 threads per SM (the register file holds no more), but at least four rows for each that
// walks rows, so that the partial rows stay small beside the input.  Depends on the sizes and the device only: `threads` is taken for
// the layout of aligned 16-bit rows, whatever the tensors' type and address.
int backward_blocks(const DeviceInfo &info, int32_t rows, int32_t n) {
    const Layout l = backward_layout(n, 8, true);
    const bool warps = l.threads == 32;
    const int64_t threads = warps ? 256 : l.threads ? l.threads : kWideThreads;
    const int64_t blocks = ceil_div64(rows, warps ? 32 : 4), most = (int64_t)info.sm_count * (threads >= 512 ? 1 : 512 / threads);
    return (int)(blocks < most ? blocks : most);
}

int32_t check_common(int32_t rows, int32_t n, int32_t dtype) {
    DeviceInfo info;
    const int32_t rc = current_device_info(&info);
    if (rc) return rc;
    CPMK_REQUIRE(rows >= 0 && n >= 1, "bad size: rows=%d n=%d", rows, n);
    CPMK_REQUIRE(dtype == CPMK_F16 || dtype == CPMK_BF16 || dtype == CPMK_F32, "unknown element type %d", dtype);
    return CPMK_OK;
}

bool aligned_to(const void *p, int64_t a) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(a - 1)) == 0; }

template <typename T>
int32_t forward(int32_t rows, int32_t n, const void *xv, float eps, int rd_mean, const void *wv, const void *bv, void *yv, float *mean, float *rstd,
                cudaStream_t stream) {
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv), *b = static_cast<const T *>(bv);
    T *y = static_cast<T *>(yv);
    constexpr int kVec = 16 / (int)sizeof(T);
    const Layout l = layout_of(n, kVec, aligned16(x) && aligned16(w) && aligned16(b) && aligned16(y), 4, 1024);
    const float inv_n = 1.f / (float)n;
#define CPMK_LN_FORWARD(VEC, NV) \
    else if (l.vec == VEC && l.nv == NV && l.threads == 32) \
        ln_rows_forward_kernel<T, VEC, NV, false><<<(rows + 3) / 4, 128, 0, stream>>>(rows, n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd); \
    else if (l.vec == VEC && l.nv == NV) \
        ln_rows_forward_kernel<T, VEC, NV, true><<<rows, l.threads, 0, stream>>>(rows, n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd)
    if (l.threads == 0) ln_rows_forward_wide_kernel<T><<<rows, kWideThreads, 0, stream>>>(n, inv_n, eps, rd_mean, x, w, b, y, mean, rstd);
    CPMK_LN_FORWARD(kVec, 1);
    CPMK_LN_FORWARD(kVec, 2);
    CPMK_LN_FORWARD(kVec, 4);
    CPMK_LN_FORWARD(1, 4);
    CPMK_LN_FORWARD(1, 8);
    CPMK_LN_FORWARD(1, 16);
#undef CPMK_LN_FORWARD
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

template <typename T, bool COLUMNS>
int32_t backward_rows(int blocks, int32_t rows, int32_t n, const T *dy, const T *x, int rd_mean, const T *w, const float *mean, const float *rstd, T *dx,
                      float *partial, cudaStream_t stream) {
    constexpr int kVec = 16 / (int)sizeof(T);
    const Layout l = backward_layout(n, kVec, aligned16(x) && aligned16(dy) && aligned16(w) && aligned16(dx));
    const float inv_n = 1.f / (float)n;
#define CPMK_LN_BACKWARD_WARP(VEC, NV) \
    else if (l.vec == VEC && l.nv == NV && l.threads == 32) \
        ln_rows_backward_kernel<T, VEC, NV, false, COLUMNS><<<blocks, 256, COLUMNS ? 2 * n * sizeof(float) : 0, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, \
                                                                                                                       rstd, w, dx, partial)
#define CPMK_LN_BACKWARD_BLOCK(VEC, NV) \
    else if (l.vec == VEC && l.nv == NV) \
        ln_rows_backward_kernel<T, VEC, NV, true, COLUMNS><<<blocks, l.threads, 0, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx, partial)
    if (l.threads == 0) ln_rows_backward_wide_kernel<T, COLUMNS><<<blocks, kWideThreads, 0, stream>>>(rows, n, inv_n, rd_mean, dy, x, mean, rstd, w, dx, partial);
    CPMK_LN_BACKWARD_WARP(kVec, 1);
    CPMK_LN_BACKWARD_WARP(kVec, 2);
    CPMK_LN_BACKWARD_WARP(1, 4);
    CPMK_LN_BACKWARD_WARP(1, 8);
    CPMK_LN_BACKWARD_BLOCK(kVec, 1);
    CPMK_LN_BACKWARD_BLOCK(kVec, 2);
    CPMK_LN_BACKWARD_BLOCK(kVec, 4);
    CPMK_LN_BACKWARD_BLOCK(1, 4);
    CPMK_LN_BACKWARD_BLOCK(1, 8);
    CPMK_LN_BACKWARD_BLOCK(1, 16);
#undef CPMK_LN_BACKWARD_WARP
#undef CPMK_LN_BACKWARD_BLOCK
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

template <typename T>
int32_t backward(const DeviceInfo &info, int32_t rows, int32_t n, const void *dyv, const void *xv, int rd_mean, const void *wv, const float *mean,
                 const float *rstd, void *dxv, void *dw, void *db, float *partial, cudaStream_t stream) {
    const T *dy = static_cast<const T *>(dyv), *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    T *dx = static_cast<T *>(dxv);
    const int blocks = backward_blocks(info, rows, n);
    if (!dw && !db) return backward_rows<T, false>(blocks, rows, n, dy, x, rd_mean, w, mean, rstd, dx, nullptr, stream);
    const int32_t rc = backward_rows<T, true>(blocks, rows, n, dy, x, rd_mean, w, mean, rstd, dx, partial, stream);
    if (rc) return rc;
    ln_rows_columns_kernel<T><<<dim3((n + 31) / 32, 2), 1024, 0, stream>>>(blocks, n, partial, static_cast<T *>(dw), static_cast<T *>(db));
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

}  // namespace
}  // namespace cpmk

using namespace cpmk;

extern "C" {

int32_t cpmk_layernorm_rows_forward(int32_t rows, int32_t n, int32_t dtype, const void *x, float eps, int32_t rd_mean, const void *weight,
                                    const void *bias, void *y, void *mean, void *rstd, cpmk_stream_t stream) {
    const int32_t rc = check_common(rows, n, dtype);
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
    if (dtype == CPMK_F16) return forward<__half>(rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
    if (dtype == CPMK_BF16) return forward<__nv_bfloat16>(rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
    return forward<float>(rows, n, x, eps, rd_mean != 0, weight, bias, y, m, r, s);
}

int32_t cpmk_layernorm_rows_backward_scratch(int32_t rows, int32_t n, int64_t *bytes) {
    DeviceInfo info;
    const int32_t rc = current_device_info(&info);
    if (rc) return rc;
    CPMK_REQUIRE(rows >= 0 && n >= 1 && bytes, "bad size: rows=%d n=%d", rows, n);
    *bytes = (int64_t)backward_blocks(info, rows, n) * 2 * n * (int64_t)sizeof(float);
    return CPMK_OK;
}

int32_t cpmk_layernorm_rows_backward(int32_t rows, int32_t n, int32_t dtype, const void *dy, const void *x, int32_t rd_mean, const void *weight,
                                     const void *mean, const void *rstd, void *dx, void *dweight, void *dbias, void *scratch, cpmk_stream_t stream) {
    DeviceInfo info;
    int32_t rc = check_common(rows, n, dtype);
    if (rc) return rc;
    rc = current_device_info(&info);
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
