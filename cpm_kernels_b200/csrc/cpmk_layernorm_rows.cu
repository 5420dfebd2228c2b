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

constexpr int kLnThreads = 256;

// Sum over the block; every thread gets it.  `red` holds one float per warp.
__device__ __forceinline__ float block_sum(float v, float *red) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) return v;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();                                   // red may be written again
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kLnThreads) ln_rows_forward_kernel(int32_t n, float inv_n, float eps, int rd_mean, const T *__restrict__ x,
                                                                     const T *__restrict__ w, const T *__restrict__ b, T *__restrict__ y,
                                                                     float *__restrict__ mean_out, float *__restrict__ rstd_out) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * n;
    float mean = 0.f;
    if (rd_mean) {
        float s = 0.f;
        for (int i = threadIdx.x; i < n; i += kLnThreads) s += to_f32(xr[i]);
        mean = block_sum(s, red) * inv_n;
    }
    float q = 0.f;
    for (int i = threadIdx.x; i < n; i += kLnThreads) {
        const float d = to_f32(xr[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum(q, red) * inv_n + eps);
    if (threadIdx.x == 0 && rstd_out) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
    for (int i = threadIdx.x; i < n; i += kLnThreads) {
        const float v = (to_f32(xr[i]) - mean) * rstd;
        y[row * n + i] = from_f32<T>(b ? fmaf(v, to_f32(w[i]), to_f32(b[i])) : v * to_f32(w[i]));
    }
}

template <typename T>
__global__ void __launch_bounds__(kLnThreads) ln_rows_dx_kernel(int32_t n, float inv_n, int rd_mean, const T *__restrict__ dy, const T *__restrict__ x,
                                                                const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                                const T *__restrict__ w, T *__restrict__ dx) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * n, *dyr = dy + row * n;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < n; i += kLnThreads) {
        const float g = to_f32(dyr[i]) * to_f32(w[i]);
        s1 += g;
        s2 = fmaf(g, (to_f32(xr[i]) - mean) * rstd, s2);
    }
    const float c1 = rd_mean ? block_sum(s1, red) * inv_n : 0.f;
    const float c2 = block_sum(s2, red) * inv_n;
    for (int i = threadIdx.x; i < n; i += kLnThreads) {
        const float g = to_f32(dyr[i]) * to_f32(w[i]), xh = (to_f32(xr[i]) - mean) * rstd;
        dx[row * n + i] = from_f32<T>(rstd * (g - c1 - xh * c2));
    }
}

// One thread per column: the sums over the rows in order.
template <typename T>
__global__ void __launch_bounds__(32) ln_rows_dw_kernel(int32_t rows, int32_t n, const T *__restrict__ dy, const T *__restrict__ x,
                                                        const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                        T *__restrict__ dw, T *__restrict__ db) {
    const int c = blockIdx.x * 32 + threadIdx.x;
    if (c >= n) return;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = 0; r < rows; ++r) {
        const float d = to_f32(dy[r * n + c]);
        sw = fmaf(d, (to_f32(x[r * n + c]) - mean_in[r]) * rstd_in[r], sw);
        sb += d;
    }
    if (dw) dw[c] = from_f32<T>(sw);
    if (db) db[c] = from_f32<T>(sb);
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
int32_t forward(int32_t rows, int32_t n, const void *x, float eps, int rd_mean, const void *w, const void *b, void *y, float *mean, float *rstd,
                cudaStream_t stream) {
    ln_rows_forward_kernel<T><<<rows, kLnThreads, 0, stream>>>(n, 1.f / (float)n, eps, rd_mean, static_cast<const T *>(x), static_cast<const T *>(w),
                                                               static_cast<const T *>(b), static_cast<T *>(y), mean, rstd);
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

template <typename T>
int32_t backward(int32_t rows, int32_t n, const void *dy, const void *x, int rd_mean, const void *w, const float *mean, const float *rstd, void *dx,
                 void *dw, void *db, cudaStream_t stream) {
    if (dx) {
        ln_rows_dx_kernel<T><<<rows, kLnThreads, 0, stream>>>(n, 1.f / (float)n, rd_mean, static_cast<const T *>(dy), static_cast<const T *>(x), mean, rstd,
                                                              static_cast<const T *>(w), static_cast<T *>(dx));
        CPMK_LAUNCH_CHECK();
    }
    if (dw || db) {
        ln_rows_dw_kernel<T><<<(n + 31) / 32, 32, 0, stream>>>(rows, n, static_cast<const T *>(dy), static_cast<const T *>(x), mean, rstd,
                                                               static_cast<T *>(dw), static_cast<T *>(db));
        CPMK_LAUNCH_CHECK();
    }
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
    *bytes = 0;
    return CPMK_OK;
}

int32_t cpmk_layernorm_rows_backward(int32_t rows, int32_t n, int32_t dtype, const void *dy, const void *x, int32_t rd_mean, const void *weight,
                                     const void *mean, const void *rstd, void *dx, void *dweight, void *dbias, void *scratch, cpmk_stream_t stream) {
    const int32_t rc = check_common(rows, n, dtype);
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
    const float *m = static_cast<const float *>(mean), *r = static_cast<const float *>(rstd);
    if (dtype == CPMK_F16) return backward<__half>(rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, s);
    if (dtype == CPMK_BF16) return backward<__nv_bfloat16>(rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, s);
    return backward<float>(rows, n, dy, x, rd_mean != 0, weight, m, r, dx, dweight, dbias, s);
}

}  // extern "C"
