// Gated feed-forward block: h = act(x Wg^T) * (x Wu^T), y = h Wd^T, and its backward pass, in fp16 and bf16 with fp32 sums.
//
//   backward   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
// Rounded to 16 bits on the way, once each: h, dg and du, because they are operands of the 16-bit products behind them (an operand in fp32
// would be two of them, and twice the products); g and u for the backward pass, because fp32 would double what a step keeps.  dh never
// leaves the chip.  Measured against 64 bits, in roundings of the result: y 1.4, gradients up to 1.9 (independent errors of as many
// roundings as each has behind it: sqrt 2 for y; g, u, dg and its own for dw_gate).
#include "cpmk_gated.cuh"

namespace cpmk {
namespace {

// ------------------------------------------------------------------------------------------------
// Generic product: out[r, c] = sum_k P[r, k] Q[c, k] with any strides, 64 x 64 outputs per block of 256 threads, 4 x 4 per thread.
// ------------------------------------------------------------------------------------------------
struct SimtParams {
    int32_t R, C, K;
    int64_t tiles_c;
    int64_t p_rs, p_ks, q_rs, q_ks;      // element strides of the rows and of k
    const void *p[2], *q[2];             // kEpiStore: sum over both pairs when p[1] is given; kEpiGated: q[0] gate, q[1] up
    void *out[3];                        // kEpiStore: out; kEpiGated: h, g, u (g, u may be null); kEpiDact: dg, du
    const void *in[2];                   // kEpiDact: g, u
};
constexpr int kSimtTile = 64, kSimtK = 16;

template <typename T, int EPI, int ACT>
__global__ void __launch_bounds__(256) gated_simt_kernel(const SimtParams prm) {
    __shared__ float sp[kSimtK][kSimtTile + 1], sq[EPI == kEpiGated ? 2 : 1][kSimtK][kSimtTile + 1];
    const int r0 = (int)(blockIdx.x / prm.tiles_c) * kSimtTile, c0 = (int)(blockIdx.x % prm.tiles_c) * kSimtTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {}, acc2[4][4] = {};
    const int pairs = EPI == kEpiStore && prm.p[1] ? 2 : 1;
    for (int pair = 0; pair < pairs; ++pair) {
        const T *P = static_cast<const T *>(prm.p[pair]), *Q = static_cast<const T *>(prm.q[pair]), *Q1 = static_cast<const T *>(prm.q[1]);
        for (int k0 = 0; k0 < prm.K; k0 += kSimtK) {
            for (int e = threadIdx.x; e < kSimtK * kSimtTile; e += 256) {
                // the thread index runs along the contiguous axis
                const int lp = prm.p_ks == 1 ? e % kSimtK : e / kSimtTile, i = prm.p_ks == 1 ? e / kSimtK : e % kSimtTile;
                sp[lp][i] = k0 + lp < prm.K && r0 + i < prm.R ? to_f32(P[(r0 + i) * prm.p_rs + (k0 + lp) * prm.p_ks]) : 0.f;
                const int lq = prm.q_ks == 1 ? e % kSimtK : e / kSimtTile, j = prm.q_ks == 1 ? e / kSimtK : e % kSimtTile;
                const bool in = k0 + lq < prm.K && c0 + j < prm.C;
                const int64_t at = (c0 + j) * prm.q_rs + (k0 + lq) * prm.q_ks;
                sq[0][lq][j] = in ? to_f32(Q[at]) : 0.f;
                if (EPI == kEpiGated) sq[EPI == kEpiGated ? 1 : 0][lq][j] = in ? to_f32(Q1[at]) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int l = 0; l < kSimtK; ++l) {
                float pv[4], qv[4], qw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pv[i] = sp[l][ty + 16 * i];
                    qv[i] = sq[0][l][tx + 16 * i];
                    if (EPI == kEpiGated) qw[i] = sq[EPI == kEpiGated ? 1 : 0][l][tx + 16 * i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        acc[i][j] = fmaf(pv[i], qv[j], acc[i][j]);
                        if (EPI == kEpiGated) acc2[i][j] = fmaf(pv[i], qw[j], acc2[i][j]);
                    }
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + ty + 16 * i, c = c0 + tx + 16 * j;
            if (r >= prm.R || c >= prm.C) continue;
            const int64_t at = (int64_t)r * prm.C + c;
            if (EPI == kEpiStore) {
                static_cast<T *>(prm.out[0])[at] = from_f32<T>(acc[i][j]);
            } else if (EPI == kEpiGated) {
                static_cast<T *>(prm.out[0])[at] = from_f32<T>(both(act_value2<ACT>(f2(acc[i][j]))).x * acc2[i][j]);
                if (prm.out[1]) {
                    static_cast<T *>(prm.out[1])[at] = from_f32<T>(acc[i][j]);
                    static_cast<T *>(prm.out[2])[at] = from_f32<T>(acc2[i][j]);
                }
            } else {
                F2 value, slope;
                act2<ACT, true>(f2(to_f32(static_cast<const T *>(prm.in[0])[at])), value, slope);
                static_cast<T *>(prm.out[0])[at] = from_f32<T>(acc[i][j] * to_f32(static_cast<const T *>(prm.in[1])[at]) * both(slope).x);
                static_cast<T *>(prm.out[1])[at] = from_f32<T>(acc[i][j] * both(value).x);
            }
        }
}

// dg = dh u act'(g), du = dh act(g) for a dh that lies in memory (the backward pass of the gated linear on its own): 16 bytes of each
// tensor per thread where their addresses and the count allow it (VEC = 8), single elements otherwise.
template <typename T, int ACT, int VEC>
__global__ void __launch_bounds__(256) gated_dact_kernel(int64_t count, const T *__restrict__ dh, const T *__restrict__ g, const T *__restrict__ u,
                                                         T *__restrict__ dg, T *__restrict__ du) {
    struct alignas(VEC * sizeof(T)) Vector {
        T v[VEC];
    };
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC; i < count; i += (int64_t)gridDim.x * 256 * VEC) {
        const Vector d = *reinterpret_cast<const Vector *>(dh + i), vg = *reinterpret_cast<const Vector *>(g + i), vu = *reinterpret_cast<const Vector *>(u + i);
        Vector og, ou;
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            constexpr int kNext = VEC > 1 ? 1 : 0;
            const F2 d2 = f2(to_f32(d.v[e]), to_f32(d.v[e + kNext]));
            F2 value, slope;
            act2<ACT, true>(f2(to_f32(vg.v[e]), to_f32(vg.v[e + kNext])), value, slope);
            const float2 a = both(d2 * f2(to_f32(vu.v[e]), to_f32(vu.v[e + kNext])) * slope), b = both(d2 * value);
            og.v[e] = from_f32<T>(a.x);
            ou.v[e] = from_f32<T>(b.x);
            if (VEC > 1) {
                og.v[e + kNext] = from_f32<T>(a.y);
                ou.v[e + kNext] = from_f32<T>(b.y);
            }
        }
        *reinterpret_cast<Vector *>(dg + i) = og;
        *reinterpret_cast<Vector *>(du + i) = ou;
    }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
template <int EPI>
int32_t launch_simt(const Call &call, SimtParams prm) {
    prm.tiles_c = ceil_div64(prm.C, kSimtTile);
    const int64_t tiles = prm.tiles_c * ceil_div64(prm.R, kSimtTile);
    CPMK_REQUIRE(tiles < (int64_t(1) << 31), "too many output tiles");
    const dim3 grid((unsigned)tiles);
    constexpr int kSilu = EPI == kEpiStore ? CPMK_ACT_GELU : CPMK_ACT_SILU;              // a plain product has no activation
    const bool silu = call.act == kSilu;
    if (call.dtype == CPMK_F16) {
        if (silu) gated_simt_kernel<__half, EPI, kSilu><<<grid, 256, 0, call.stream>>>(prm);
        else gated_simt_kernel<__half, EPI, CPMK_ACT_GELU><<<grid, 256, 0, call.stream>>>(prm);
    } else {
        if (silu) gated_simt_kernel<__nv_bfloat16, EPI, kSilu><<<grid, 256, 0, call.stream>>>(prm);
        else gated_simt_kernel<__nv_bfloat16, EPI, CPMK_ACT_GELU><<<grid, 256, 0, call.stream>>>(prm);
    }
    CPMK_LAUNCH_CHECK();
    call.launched = false;                               // (nothing waits for it early)
    return CPMK_OK;
}

bool tensor_core_size(int32_t extent) { return extent % 8 == 0; }

// The tensor cores' loads and stores want 16-byte rows and addresses; everything else runs generic.
bool on_tensor_cores(const Product &p, int32_t K, bool transposed) {
    return tensor_core_size(transposed ? p.R : K) && tensor_core_size(p.C) && aligned16(p.p) && aligned16(p.q) && aligned16(p.out);
}

// Up to three products out (R, C) = P Q^T of the same K; operands stored (rows, K), or (K, rows) when `transposed`.
int32_t products_of(const Call &call, int32_t K, bool transposed, const Product *products, int count, void *scratch) {
    bool all = true;
    for (int i = 0; i < count; ++i) all = all && on_tensor_cores(products[i], K, transposed);
    if (all) return tc_products(call, K, transposed, products, count, scratch);
    for (int i = 0; i < count; ++i) {
        const Product &p = products[i];
        int32_t rc;
        if (on_tensor_cores(p, K, transposed)) {
            rc = tc_products(call, K, transposed, &p, 1, scratch);
        } else {
            SimtParams prm = {};
            prm.R = p.R; prm.C = p.C; prm.K = K;
            prm.p_rs = transposed ? 1 : K; prm.p_ks = transposed ? p.R : 1;
            prm.q_rs = transposed ? 1 : K; prm.q_ks = transposed ? p.C : 1;
            prm.p[0] = p.p; prm.q[0] = p.q;
            prm.out[0] = p.out;
            rc = launch_simt<kEpiStore>(call, prm);
        }
        if (rc) return rc;
    }
    return CPMK_OK;
}

// out (R, C) = P0 Q0^T + P1 Q1^T, P stored (R, K), Q stored (K, C)
int32_t sum_of(const Call &call, int32_t R, int32_t C, int32_t K, const void *p0, const void *q0, const void *p1, const void *q1, void *out, void *scratch) {
    if (tensor_core_size(K) && tensor_core_size(C) && aligned16(p0) && aligned16(q0) && aligned16(p1) && aligned16(q1) && aligned16(out))
        return tc_sum(call, R, C, K, p0, q0, p1, q1, out, scratch);
    SimtParams prm = {};
    prm.R = R; prm.C = C; prm.K = K;
    prm.p_rs = K; prm.p_ks = 1; prm.q_rs = 1; prm.q_ks = C;
    prm.p[0] = p0; prm.p[1] = p1; prm.q[0] = q0; prm.q[1] = q1;
    prm.out[0] = out;
    return launch_simt<kEpiStore>(call, prm);
}

bool few_tokens(int32_t tokens) { return tokens <= kFewTokens; }

bool gated_on_tensor_cores(int32_t k, int32_t n, const void *x, const void *wg, const void *wu, const void *h, const void *g, const void *u) {
    return tensor_core_size(k) && tensor_core_size(n) && aligned16(x) && aligned16(wg) && aligned16(wu) && aligned16(h) && aligned16(g) && aligned16(u);
}

int32_t gated_product(const Call &call, int32_t tokens, int32_t k, int32_t n, const void *x, const void *wg, const void *wu, void *h, void *g, void *u,
                      void *scratch) {
    if (gated_on_tensor_cores(k, n, x, wg, wu, h, g, u))
        return few_tokens(tokens) ? few_gated(call, tokens, k, n, x, wg, wu, h, g, u, scratch) : tc_gated(call, tokens, k, n, x, wg, wu, h, g, u, scratch);
    SimtParams prm = {};
    prm.R = tokens; prm.C = n; prm.K = k;
    prm.p_rs = k; prm.p_ks = 1; prm.q_rs = k; prm.q_ks = 1;
    prm.p[0] = x; prm.q[0] = wg; prm.q[1] = wu;
    prm.out[0] = h; prm.out[1] = g; prm.out[2] = u;
    return launch_simt<kEpiGated>(call, prm);
}

// dg, du from dh = dy Wd, which is not stored; Wd is (m, n)
int32_t dact_product(const Call &call, int32_t tokens, int32_t n, int32_t m, const void *dy, const void *wd, const void *g, const void *u, void *dg,
                     void *du, void *scratch) {
    if (tensor_core_size(n) && tensor_core_size(m) && aligned16(dy) && aligned16(wd) && aligned16(g) && aligned16(u) && aligned16(dg) && aligned16(du))
        return tc_dact(call, tokens, n, m, dy, wd, g, u, dg, du, scratch);
    SimtParams prm = {};
    prm.R = tokens; prm.C = n; prm.K = m;
    prm.p_rs = m; prm.p_ks = 1; prm.q_rs = 1; prm.q_ks = n;
    prm.p[0] = dy; prm.q[0] = wd;
    prm.in[0] = g; prm.in[1] = u;
    prm.out[0] = dg; prm.out[1] = du;
    return launch_simt<kEpiDact>(call, prm);
}

template <typename T, int ACT>
void launch_dact(const Call &call, int64_t count, const void *dh, const void *g, const void *u, void *dg, void *du) {
    const bool wide = count % 8 == 0 && aligned16(dh) && aligned16(g) && aligned16(u) && aligned16(dg) && aligned16(du);
    const int64_t blocks = ceil_div64(count, wide ? 2048 : 256), most = 8 * call.info.sm_count;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    const T *d = static_cast<const T *>(dh), *a = static_cast<const T *>(g), *b = static_cast<const T *>(u);
    if (wide) gated_dact_kernel<T, ACT, 8><<<grid, 256, 0, call.stream>>>(count, d, a, b, static_cast<T *>(dg), static_cast<T *>(du));
    else gated_dact_kernel<T, ACT, 1><<<grid, 256, 0, call.stream>>>(count, d, a, b, static_cast<T *>(dg), static_cast<T *>(du));
}

int32_t dact(const Call &call, int64_t count, const void *dh, const void *g, const void *u, void *dg, void *du) {
    const bool silu = call.act == CPMK_ACT_SILU;
    if (call.dtype == CPMK_F16) silu ? launch_dact<__half, CPMK_ACT_SILU>(call, count, dh, g, u, dg, du) : launch_dact<__half, CPMK_ACT_GELU>(call, count, dh, g, u, dg, du);
    else silu ? launch_dact<__nv_bfloat16, CPMK_ACT_SILU>(call, count, dh, g, u, dg, du) : launch_dact<__nv_bfloat16, CPMK_ACT_GELU>(call, count, dh, g, u, dg, du);
    CPMK_LAUNCH_CHECK();
    return CPMK_OK;
}

bool even_address(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }

// Every extent fits an int with room for a tile beside it.
int32_t check_sizes(int32_t tokens, int32_t k, int32_t n, int32_t m) {
    constexpr int32_t kMost = 1 << 30;
    CPMK_REQUIRE(tokens >= 0 && tokens <= kMost && k >= 1 && k <= kMost && n >= 1 && n <= kMost && m >= 1 && m <= kMost,
                 "bad size: tokens=%d k=%d n=%d m=%d (at most 2^30)", tokens, k, n, m);
    return CPMK_OK;
}

int32_t begin(Call *call, int32_t tokens, int32_t k, int32_t n, int32_t m, int32_t dtype, int32_t act, cpmk_stream_t stream) {
    const int32_t rc = current_device_info(&call->info);
    if (rc) return rc;
    // a thread whose first CUDA call this is (autograd's) has no context yet, and encoding a tensor map fails without one
    CPMK_CUDA_TRY(cudaSetDevice(call->info.device));
    const int32_t rc_sizes = check_sizes(tokens, k, n, m);
    if (rc_sizes) return rc_sizes;
    CPMK_REQUIRE(dtype == CPMK_F16 || dtype == CPMK_BF16, "the gated block takes fp16 and bf16 (dtype %d)", dtype);
    CPMK_REQUIRE(act == CPMK_ACT_GELU || act == CPMK_ACT_SILU, "unknown activation %d", act);
    call->dtype = dtype;
    call->act = act;
    call->stream = as_stream(stream);
    return CPMK_OK;
}

// dx, dWg, dWu from dg, du, and dWd from dy, h
int32_t gradients(const Call &call, int32_t tokens, int32_t k, int32_t n, int32_t m, const void *x, const void *wg, const void *wu, const void *dg,
                  const void *du, const void *dy, const void *h, void *dx, void *dwg, void *dwu, void *dwd, void *scratch) {
    if (dx) {
        const int32_t rc = sum_of(call, tokens, k, n, dg, wg, du, wu, dx, scratch);
        if (rc) return rc;
    }
    Product wanted[3];
    int count = 0;
    if (dwg) wanted[count++] = {n, k, dg, x, dwg};
    if (dwu) wanted[count++] = {n, k, du, x, dwu};
    if (dwd) wanted[count++] = {m, n, dy, h, dwd};
    return count ? products_of(call, tokens, true, wanted, count, scratch) : CPMK_OK;
}

// without tokens the weights' gradients are zero
int32_t clear_gradients(const Call &call, void *dwg, void *dwu, void *dwd, int64_t nk, int64_t mn) {
    if (dwg) CPMK_CUDA_TRY(cudaMemsetAsync(dwg, 0, (size_t)nk * 2, call.stream));
    if (dwu) CPMK_CUDA_TRY(cudaMemsetAsync(dwu, 0, (size_t)nk * 2, call.stream));
    if (dwd) CPMK_CUDA_TRY(cudaMemsetAsync(dwd, 0, (size_t)mn * 2, call.stream));
    return CPMK_OK;
}

// scratch is there where the sizes ask for it, and aligned
int32_t check_scratch(const void *scratch, int32_t (*bytes_of)(int32_t, int32_t, int32_t, int32_t, int64_t *), int32_t tokens, int32_t k, int32_t n, int32_t m) {
    int64_t bytes = 0;
    const int32_t rc = bytes_of(tokens, k, n, m, &bytes);
    if (rc) return rc;
    CPMK_REQUIRE(aligned16(scratch) && (scratch || !bytes), "scratch of %lld bytes, 16-byte aligned, is needed", (long long)bytes);
    return CPMK_OK;
}

int64_t larger(int64_t a, int64_t b) { return a > b ? a : b; }

}  // namespace
}  // namespace cpmk

using namespace cpmk;

extern "C" {

int32_t cpmk_gated_scratch(int32_t tokens, int32_t k, int32_t n, int32_t m, int64_t *bytes) {
    DeviceInfo info;
    int32_t rc = current_device_info(&info);
    if (rc) return rc;
    rc = check_sizes(tokens, k, n, m > 0 ? m : 1);
    if (rc) return rc;
    CPMK_REQUIRE(m >= 0 && bytes, "bad arguments: m=%d", m);
    int64_t need = 0;
    if (tokens > 0 && tensor_core_size(n)) {
        const bool down = m > 0 && tensor_core_size(m), first = tensor_core_size(k);
        // pointers are not known here: room for the few-token pair of products, and for those of the tiles
        if (few_tokens(tokens) && first) need = few_scratch(info, tokens, k, n, down ? m : 0);
        if (!few_tokens(tokens) && first) need = tc_gated_scratch(info, tokens, k, n);
        const Product y = {tokens, m, nullptr, nullptr, nullptr};
        if (down) need = larger(need, tc_products_scratch(info, n, &y, 1));
    }
    *bytes = need;
    return CPMK_OK;
}

int32_t cpmk_gated_backward_scratch(int32_t tokens, int32_t k, int32_t n, int32_t m, int64_t *bytes) {
    DeviceInfo info;
    int32_t rc = current_device_info(&info);
    if (rc) return rc;
    rc = check_sizes(tokens, k, n, m > 0 ? m : 1);
    if (rc) return rc;
    CPMK_REQUIRE(m >= 0 && bytes, "bad arguments: m=%d", m);
    int64_t need = 0;
    if (tokens > 0 && tensor_core_size(n)) {
        const bool down = m > 0 && tensor_core_size(m);
        if (tensor_core_size(k)) need = larger(need, tc_sum_scratch(info, tokens, k, n));
        if (down) need = larger(need, tc_dact_scratch(info, tokens, n, m));
        // the weights' gradients that are wanted are not known here: any of them, alone or together
        const Product up = {n, k, nullptr, nullptr, nullptr}, last = {m, n, nullptr, nullptr, nullptr};
        const Product ups[3] = {up, up, last}, one[2] = {up, last};
        for (int count = 1; tensor_core_size(k) && count <= (down ? 3 : 2); ++count) need = larger(need, tc_products_scratch(info, tokens, ups, count));
        if (down && tensor_core_size(k)) need = larger(need, tc_products_scratch(info, tokens, one, 2));
        if (down) need = larger(need, tc_products_scratch(info, tokens, &last, 1));
    }
    *bytes = need;
    return CPMK_OK;
}

int32_t cpmk_gated_linear_forward(int32_t tokens, int32_t k, int32_t n, int32_t dtype, int32_t activation, const void *x, const void *w_gate,
                                  const void *w_up, void *h, void *g, void *u, void *scratch, cpmk_stream_t stream) {
    Call call;
    int32_t rc = begin(&call, tokens, k, n, 1, dtype, activation, stream);
    if (rc) return rc;
    if (tokens == 0) return CPMK_OK;
    CPMK_REQUIRE(x && w_gate && w_up && h, "null pointer");
    CPMK_REQUIRE((g == nullptr) == (u == nullptr), "g and u are wanted together or not at all");
    CPMK_REQUIRE(even_address(x) && even_address(w_gate) && even_address(w_up) && even_address(h) && even_address(g) && even_address(u),
                 "tensors must be 2-byte aligned");
    rc = check_scratch(scratch, cpmk_gated_scratch, tokens, k, n, 0);
    if (rc) return rc;
    return gated_product(call, tokens, k, n, x, w_gate, w_up, h, g, u, scratch);
}

int32_t cpmk_gated_linear_backward(int32_t tokens, int32_t k, int32_t n, int32_t dtype, int32_t activation, const void *dh, const void *x,
                                   const void *w_gate, const void *w_up, const void *g, const void *u, void *dg, void *du, void *dx, void *dw_gate,
                                   void *dw_up, void *scratch, cpmk_stream_t stream) {
    Call call;
    int32_t rc = begin(&call, tokens, k, n, 1, dtype, activation, stream);
    if (rc) return rc;
    if (tokens == 0) return clear_gradients(call, dw_gate, dw_up, nullptr, (int64_t)n * k, 0);
    CPMK_REQUIRE(dh && x && w_gate && w_up && g && u && dg && du, "null pointer");
    CPMK_REQUIRE(even_address(dh) && even_address(x) && even_address(w_gate) && even_address(w_up) && even_address(g) && even_address(u) &&
                     even_address(dg) && even_address(du) && even_address(dx) && even_address(dw_gate) && even_address(dw_up),
                 "tensors must be 2-byte aligned");
    rc = check_scratch(scratch, cpmk_gated_backward_scratch, tokens, k, n, 0);
    if (rc) return rc;
    rc = dact(call, (int64_t)tokens * n, dh, g, u, dg, du);
    if (rc) return rc;
    return gradients(call, tokens, k, n, 0, x, w_gate, w_up, dg, du, nullptr, nullptr, dx, dw_gate, dw_up, nullptr, scratch);
}

int32_t cpmk_gated_feed_forward_forward(int32_t tokens, int32_t k, int32_t n, int32_t m, int32_t dtype, int32_t activation, const void *x,
                                        const void *w_gate, const void *w_up, const void *w_down, void *h, void *g, void *u, void *y, void *scratch,
                                        cpmk_stream_t stream) {
    Call call;
    int32_t rc = begin(&call, tokens, k, n, m, dtype, activation, stream);
    if (rc) return rc;
    if (tokens == 0) return CPMK_OK;
    CPMK_REQUIRE(x && w_gate && w_up && w_down && h && y, "null pointer");
    CPMK_REQUIRE((g == nullptr) == (u == nullptr), "g and u are wanted together or not at all");
    CPMK_REQUIRE(even_address(x) && even_address(w_gate) && even_address(w_up) && even_address(w_down) && even_address(h) && even_address(g) &&
                     even_address(u) && even_address(y),
                 "tensors must be 2-byte aligned");
    rc = check_scratch(scratch, cpmk_gated_scratch, tokens, k, n, m);
    if (rc) return rc;
    rc = gated_product(call, tokens, k, n, x, w_gate, w_up, h, g, u, scratch);
    if (rc) return rc;
    if (few_tokens(tokens) && tensor_core_size(m) && gated_on_tensor_cores(k, n, x, w_gate, w_up, h, g, u) && aligned16(w_down) && aligned16(y))
        return few_down(call, tokens, k, n, m, h, w_down, y, scratch);
    const Product down = {tokens, m, h, w_down, y};
    return products_of(call, n, false, &down, 1, scratch);
}

int32_t cpmk_gated_feed_forward_backward(int32_t tokens, int32_t k, int32_t n, int32_t m, int32_t dtype, int32_t activation, const void *dy,
                                         const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *g, const void *u,
                                         const void *h, void *dg, void *du, void *dx, void *dw_gate, void *dw_up, void *dw_down, void *scratch,
                                         cpmk_stream_t stream) {
    Call call;
    int32_t rc = begin(&call, tokens, k, n, m, dtype, activation, stream);
    if (rc) return rc;
    if (tokens == 0) return clear_gradients(call, dw_gate, dw_up, dw_down, (int64_t)n * k, (int64_t)m * n);
    CPMK_REQUIRE(dy && x && w_gate && w_up && w_down && g && u && dg && du && (h || !dw_down), "null pointer");
    CPMK_REQUIRE(even_address(dy) && even_address(x) && even_address(w_gate) && even_address(w_up) && even_address(w_down) && even_address(g) &&
                     even_address(u) && even_address(h) && even_address(dg) && even_address(du) && even_address(dx) && even_address(dw_gate) &&
                     even_address(dw_up) && even_address(dw_down),
                 "tensors must be 2-byte aligned");
    rc = check_scratch(scratch, cpmk_gated_backward_scratch, tokens, k, n, m);
    if (rc) return rc;
    if (dx || dw_gate || dw_up) {
        rc = dact_product(call, tokens, n, m, dy, w_down, g, u, dg, du, scratch);
        if (rc) return rc;
    }
    return gradients(call, tokens, k, n, m, x, w_gate, w_up, dg, du, dy, h, dx, dw_gate, dw_up, dw_down, scratch);
}

}  // extern "C"
