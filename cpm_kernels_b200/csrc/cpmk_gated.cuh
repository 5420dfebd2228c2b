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
// (1 + tanh t) / 2 = s(2 t)).  Derivative: s + v s (1 - s) z'(v).  Beyond |v| = 30 gelu's logistic is 0 or 1 in fp32 (|z| > 1900), so z
// and z' are taken of the clamped value: the cube cannot overflow and 0 * inf does not arise.
//
// Two values at a time in packed fp32 arithmetic: the epilogue of a product is bound by the instructions it issues (scalar, the epilogue
// of dy Wd took 12 us a tile, more than half of what its products take at k = 4096).  s = 1 / (1 + 2^(-z log2 e)) with the hardware's
// approximate exponential and reciprocal (2^-22 each; the exponential's argument is rounded, 2^-24 of at most 128).
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 both(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
// s(z) from -z log2 e
__device__ __forceinline__ F2 logistic2(F2 minus_z_log2e) {
    const float2 t = both(minus_z_log2e);
    float e0, e1, s0, s1;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t.y));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s0) : "f"(1.f + e0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s1) : "f"(1.f + e1));
    return f2(s0, s1);
}

constexpr float kLog2e = 1.4426950408889634f, kGeluTwoC = 1.5957691216057308f, kGeluCube = 0.044715f;

// the larger and the smaller of two values, NaN if one is
__device__ __forceinline__ float larger_of(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float smaller_of(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// act(v); SLOPE: and act'(v), of a v that was stored in 16 bits: beyond 65504 an fp16 one is infinite, though it was not when h was worked
// out.  Both have their limits there (0 and 0, infinity and 1), not the NaN of 0 times infinity: v is held above -L, where s is 0 already
// (L = 30, silu 128), and the v of the slope's second term below L, where 1 - s is.
template <int ACT, bool SLOPE>
__device__ __forceinline__ void act2(F2 v, F2 &value, F2 &slope) {
    constexpr float kLimit = ACT == CPMK_ACT_SILU ? 128.f : 30.f;
    float2 x = both(v);
    if (SLOPE) {
        x = make_float2(larger_of(x.x, -kLimit), larger_of(x.y, -kLimit));
        v = f2(x.x, x.y);
    }
    F2 s, c = v, dz = f2(1.f);
    if (ACT == CPMK_ACT_SILU) {
        s = logistic2(v * f2(-kLog2e));
    } else {
        c = f2(smaller_of(larger_of(x.x, -kLimit), kLimit), smaller_of(larger_of(x.y, -kLimit), kLimit));
        const F2 c2 = c * c;
        s = logistic2(c * fma2(c2, f2(-kLog2e * kGeluTwoC * kGeluCube), f2(-kLog2e * kGeluTwoC)));
        if (SLOPE) dz = fma2(c2, f2(3.f * kGeluTwoC * kGeluCube), f2(kGeluTwoC));
    }
    value = v * s;
    if (SLOPE) {
        if (ACT == CPMK_ACT_SILU) c = f2(smaller_of(x.x, kLimit), smaller_of(x.y, kLimit));
        const F2 rest = c * s * fma2(s, f2(-1.f), f2(1.f));          // v s (1 - s)
        slope = ACT == CPMK_ACT_SILU ? rest + s : fma2(rest, dz, s);
    }
}
template <int ACT>
__device__ __forceinline__ F2 act_value2(F2 v) {
    F2 value, slope;
    act2<ACT, false>(v, value, slope);
    return value;
}

// What becomes of a finished sum: stored; with its partner (gate and up) through the activation; as dh through the activation's slope.
enum { kEpiStore = 0, kEpiGated = 1, kEpiDact = 2 };

struct Call {
    DeviceInfo info;
    int32_t dtype, act;
    cudaStream_t stream;
    // A tile kernel (or its join) of this call is the stream's last: the next starts while it drains, and waits for it.  Block of 1467
    // tokens, 832 / 2136: 35.4 -> 33.8 us, its backward pass 65.9 -> 64.5; 4096 tokens, 4096 / 10240: 1419 -> 1412.
    mutable bool launched = false;
    mutable uint32_t *status = nullptr;  // the word of the call's stream, once a kernel that waits is launched (status_of)
};
inline int32_t status_of(const Call &call, uint32_t **word) {
    const int32_t rc = call.status ? CPMK_OK : get_status_word(call.stream, &call.status);
    *word = call.status;
    return rc;
}

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
