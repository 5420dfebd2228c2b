// What the kernel files of the gated feed-forward block share: the activations, one call's constants, and the launchers of the
// tensor-core kernels.
#pragma once

#include "cpmk_common.cuh"
#include "cpmk_types.cuh"

namespace cpmk {

// ------------------------------------------------------------------------------------------------
// the activation
// ------------------------------------------------------------------------------------------------
// Both activations are v s(z(v)) with the logistic function s: z = v (silu), z = 2 c (v + 0.044715 v^3), c = sqrt(2 / pi) (gelu:
// (1 + tanh t) / 2 = s(2 t)).  Derivative: s + v s (1 - s) z'(v).  Beyond |v| = 30 the logistic is 0 or 1 in fp32 (|z| > 1900), so z
// and z' are taken of the clamped value: the cube cannot overflow and 0 * inf does not arise.
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_value(float v) {
    if (ACT == CPMK_ACT_SILU) return v * logistic(v);
    const float c = fminf(fmaxf(v, -30.f), 30.f);
    return v * logistic(1.5957691216057308f * fmaf(0.044715f * c * c, c, c));
}

template <int ACT>
__device__ __forceinline__ void act_value_slope(float v, float &value, float &slope) {
    if (ACT == CPMK_ACT_SILU) {
        const float s = logistic(v);
        value = v * s;
        slope = fmaf(value, 1.f - s, s);
    } else {
        const float c = fminf(fmaxf(v, -30.f), 30.f), c2 = c * c;
        const float s = logistic(1.5957691216057308f * fmaf(0.044715f * c2, c, c));
        value = v * s;
        slope = fmaf(value * (1.f - s), 1.5957691216057308f * fmaf(3.f * 0.044715f, c2, 1.f), s);
    }
}

// What becomes of a finished sum: stored; with its partner (gate and up) through the activation; as dh through the activation's slope.
enum { kEpiStore = 0, kEpiGated = 1, kEpiDact = 2 };

struct Call {
    DeviceInfo info;
    int32_t dtype, act;
    cudaStream_t stream;
};

// Tensor-core products on 256 x 256 tiles (cpmk_gated_tc.cu): extents multiples of 8, pointers 16-byte aligned, scratch as many bytes as
// the _scratch function of the product says.
// tc_products: up to three products out (R, C) = P Q^T of the same K in one launch, operands stored (rows, K), or (K, rows) when
// `transposed`.  tc_sum: out = P0 Q0^T + P1 Q1^T with P stored (R, K), Q stored (K, C).
struct Product {
    int32_t R, C;
    const void *p, *q;
    void *out;
};
int32_t tc_products(const Call &call, int32_t K, bool transposed, const Product *products, int count, void *scratch);
int32_t tc_sum(const Call &call, int32_t R, int32_t C, int32_t K, const void *p0, const void *q0, const void *p1, const void *q1, void *out, void *scratch);
int32_t tc_gated(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u,
                 void *scratch);
int32_t tc_dact(const Call &call, int32_t tokens, int32_t n, int32_t m, const void *dy, const void *wd, const void *g, const void *u, void *dg, void *du,
                void *scratch);
int64_t tc_products_scratch(const DeviceInfo &info, int32_t K, const Product *products, int count);
int64_t tc_sum_scratch(const DeviceInfo &info, int32_t R, int32_t C, int32_t K);
int64_t tc_gated_scratch(const DeviceInfo &info, int32_t tokens, int32_t k, int32_t n);
int64_t tc_dact_scratch(const DeviceInfo &info, int32_t tokens, int32_t n, int32_t m);

// Products for few tokens (cpmk_gated_few.cu), the same requirements; few_down follows few_gated of the same call.  few_scratch: bytes
// for both (m = 0: the first alone).
constexpr int32_t kFewTokens = 256;
int64_t few_scratch(const DeviceInfo &info, int32_t tokens, int32_t k, int32_t n, int32_t m);
int32_t few_gated(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u,
                  void *scratch);
int32_t few_down(const Call &call, int32_t tokens, int32_t k, int32_t n, int32_t m, const void *h, const void *wd, void *y, void *scratch);

}  // namespace cpmk
