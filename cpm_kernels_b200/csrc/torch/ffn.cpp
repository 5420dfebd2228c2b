// Autograd of the row layer norm and the gated feed-forward block: checks of arguments, allocation of outputs and scratch, the current
// stream and what the backward pass keeps, as C++ functions of PyTorch's autograd.  All arithmetic happens behind the C interface (include/cpmk_b200.h), whose
// entry points are handed over by address (bind), from the library that the ctypes layer has loaded.
//
// In C++ because a training step of a small layer is bound by the host: a forward and backward pass of the layer norm of 64 x 512 took 109
// us as Python functions, and takes 68 here (PyTorch's layer norm: 71; a step that only doubles: 51), where the calls need neither the
// interpreter nor its lock.  A forward pass alone: 16 x 512 layer norm 5.1 us, block of 16 tokens 13.6 (checks in Python: 2 us more).
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <string>

#include "../../../include/cpmk_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&cpmk_last_error) last_error;
    decltype(&cpmk_layernorm_rows_forward) layernorm_rows_forward;
    decltype(&cpmk_layernorm_rows_backward_scratch) layernorm_rows_backward_scratch;
    decltype(&cpmk_layernorm_rows_backward) layernorm_rows_backward;
    decltype(&cpmk_gated_scratch) gated_scratch;
    decltype(&cpmk_gated_backward_scratch) gated_backward_scratch;
    decltype(&cpmk_gated_linear_forward) gated_linear_forward;
    decltype(&cpmk_gated_linear_backward) gated_linear_backward;
    decltype(&cpmk_gated_feed_forward_forward) gated_feed_forward_forward;
    decltype(&cpmk_gated_feed_forward_backward) gated_feed_forward_backward;
} api;

void bind(const std::vector<uintptr_t> &addresses) {
    if (addresses.size() * sizeof(uintptr_t) != sizeof(Api)) throw std::runtime_error("bind: as many addresses as entry points are wanted");
    memcpy(&api, addresses.data(), sizeof(Api));
}

// the error the ctypes layer raises for a non-zero status
void check(int32_t status, const char *what) {
    if (status != CPMK_OK) throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(status) + "): " + api.last_error());
}

// an argument that the documentation does not allow; an AssertionError in Python, as from the other operators
struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void want(bool ok, const char *what) {
    if (!ok) throw Refused(what);
}
// contiguous, and what its memory holds (a view such as z.conj().imag is to be read negated)
bool as_it_lies(const Tensor &t) { return t.is_contiguous() && !t.is_neg(); }
Tensor laid_out(const Tensor &t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }
// of the type and on the device of x, as it lies, with these extents
bool goes_with(const Tensor &t, const Tensor &x, at::IntArrayRef sizes) {
    return t.defined() && t.device() == x.device() && t.scalar_type() == x.scalar_type() && t.sizes() == sizes && as_it_lies(t);
}
constexpr int64_t kMost = int64_t{1} << 30;

int32_t dtype_of(const Tensor &t) { return t.scalar_type() == at::kHalf ? CPMK_F16 : t.scalar_type() == at::kBFloat16 ? CPMK_BF16 : CPMK_F32; }

void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
char *part(const Tensor &t, int64_t i) { return static_cast<char *>(t.data_ptr()) + i * (t.numel() / t.size(0)) * t.element_size(); }

// uninitialised, contiguous, of the type and on the device of t; straight from the allocator (0.5 us each less than through the dispatcher:
// 97 -> 93 us for a step of the block)
Tensor fresh(at::IntArrayRef sizes, const Tensor &t) { return at::detail::empty_cuda(sizes, t.scalar_type(), t.device(), std::nullopt); }

Tensor bytes_like(const Tensor &t, int64_t bytes) { return bytes ? at::Tensor(at::detail::empty_cuda({bytes}, at::kByte, t.device(), std::nullopt)) : Tensor(); }

// The tensors' device made current, and its current stream.
struct Place {
    c10::cuda::CUDAGuard guard;
    cpmk_stream_t stream;
    explicit Place(const Tensor &t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// Forward-mode differentiation would lose its tangents on the direct path, silently: refused whether or not gradients are recorded.
template <typename... T>
void refuse_tangents(const T &...t) {
    if ((... || (t.defined() && t._fw_grad(/*level=*/0).defined())))
        throw std::runtime_error("forward-mode differentiation (torch.autograd.forward_ad) is not available for this operator");
}

// Whether anything is to be differentiated.
template <typename... T>
bool tracked(const T &...t) {
    return at::GradMode::is_enabled() && (... || (t.defined() && t.requires_grad()));
}

// A gradient that is returned while a graph of the gradients is asked for (create_graph) raises when it is differentiated again: once is all
// there is.  `on`: the tensors that it is computed from.  Where none of them requires a gradient it is a constant, and stays one; the
// incoming gradient alone does not tell (that of y.sum() requires none, but dx depends on x and the weights all the same).
struct Once : torch::autograd::Function<Once> {
    static Tensor forward(AutogradContext *, const Tensor &g) { return g.view_as(g); }
    static variable_list backward(AutogradContext *, variable_list) {
        throw std::runtime_error("trying to differentiate twice a function that is differentiable once");
    }
};
template <typename... T>
Tensor once(const Tensor &g, const T &...on) {
    return g.defined() && tracked(on...) ? Once::apply(g.detach().requires_grad_(true)) : g;
}

// ------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------
// stats: the rows' means, then their reciprocal deviations, when they are wanted
Tensor layernorm_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, double eps, bool rd_mean, Tensor *stats) {
    const int64_t n = weight.numel(), rows = x.numel() / n;
    const Place place(x);
    Tensor y = fresh(x.sizes(), x);
    if (stats) *stats = at::detail::empty_cuda({2 * rows}, at::kFloat, x.device(), std::nullopt);
    float *mean = stats ? static_cast<float *>(stats->data_ptr()) : nullptr;
    check(api.layernorm_rows_forward((int32_t)rows, (int32_t)n, dtype_of(x), x.data_ptr(), (float)eps, rd_mean, weight.data_ptr(), address(bias), y.data_ptr(),
                                     mean, stats && rows ? mean + rows : mean, place.stream),
          "cpmk_layernorm_rows_forward");
    return y;
}

struct LayerNormRows : torch::autograd::Function<LayerNormRows> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const std::optional<Tensor> &bias, double eps, bool rd_mean) {
        Tensor stats;
        Tensor y = layernorm_forward(x, weight, bias ? *bias : Tensor(), eps, rd_mean, &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["rd_mean"] = rd_mean;
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
        const int64_t n = weight.numel(), rows = x.numel() / n;
        const Tensor dy = laid_out(grads[0]);
        const Place place(x);
        Tensor dx, dweight, dbias, scratch;
        if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x);
        if (ctx->needs_input_grad(1)) dweight = fresh(weight.sizes(), weight);
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)) dbias = fresh(weight.sizes(), weight);
        if (dweight.defined() || dbias.defined()) {
            int64_t bytes = 0;
            check(api.layernorm_rows_backward_scratch((int32_t)rows, (int32_t)n, &bytes), "cpmk_layernorm_rows_backward_scratch");
            scratch = bytes_like(x, bytes);
        }
        float *mean = static_cast<float *>(stats.data_ptr());
        check(api.layernorm_rows_backward((int32_t)rows, (int32_t)n, dtype_of(x), dy.data_ptr(), x.data_ptr(), ctx->saved_data["rd_mean"].toBool(),
                                          weight.data_ptr(), mean, mean + rows, address(dx), address(dweight), address(dbias), address(scratch), place.stream),
              "cpmk_layernorm_rows_backward");
        return {once(dx, grads[0], x, weight), once(dweight, grads[0], x), once(dbias, grads[0]), Tensor(), Tensor()};
    }
};

Tensor layernorm_rows(const Tensor &x, double eps, const Tensor &weight, const std::optional<Tensor> &bias, bool rd_mean) {
    want(x.is_cuda() && x.dim() >= 1 && as_it_lies(x), "layernorm_rows: x must be a contiguous CUDA tensor of one axis or more");
    const at::ScalarType type = x.scalar_type();
    want(type == at::kHalf || type == at::kBFloat16 || type == at::kFloat, "layernorm_rows: x must be fp16, bf16 or fp32");
    const int64_t n = x.size(-1);
    want(n >= 1 && n <= kMost && x.numel() / n < 2 * kMost, "layernorm_rows: 1 to 2^30 elements a row, fewer than 2^31 rows");
    want(eps >= 0, "layernorm_rows: eps must not be negative");
    want(goes_with(weight, x, {n}), "layernorm_rows: weight must be contiguous, (n), of x's type and on its device");
    want(!bias || goes_with(*bias, x, {n}), "layernorm_rows: bias must be contiguous, (n), of x's type and on its device");
    const Tensor b = bias ? *bias : Tensor();
    refuse_tangents(x, weight, b);
    if (tracked(x, weight, b)) return LayerNormRows::apply(x, weight, bias, eps, rd_mean);
    return layernorm_forward(x, weight, b, eps, rd_mean, nullptr);
}

// ------------------------------------------------------------------------------------------------
// gated feed-forward block
// ------------------------------------------------------------------------------------------------
void check_gated(const Tensor &x, const Tensor &w_gate, const Tensor &w_up) {
    want(x.is_cuda() && x.dim() >= 1 && as_it_lies(x), "gated block: x must be a contiguous CUDA tensor of one axis or more");
    want(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "gated block: x must be fp16 or bf16");
    want(w_gate.dim() == 2, "gated block: w_gate must be a matrix");
    const int64_t n = w_gate.size(0), k = w_gate.size(1);
    // the C entry points take 32-bit extents
    want(n >= 1 && k >= 1 && n <= kMost && k <= kMost && x.size(-1) == k && x.numel() / k <= kMost,
         "gated block: w_gate must be (N, K) for x (..., K), with N, K and the rows of x at most 2^30");
    want(goes_with(w_gate, x, {n, k}) && goes_with(w_up, x, {n, k}), "gated block: w_gate and w_up must be contiguous, alike, of x's type and on its device");
}

std::vector<int64_t> with_last(const Tensor &x, int64_t last) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = last;
    return shape;
}

// gu: the two projections (2, tokens, n), when they are wanted
Tensor gated_forward(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, int64_t activation, Tensor *gu) {
    const int64_t n = w_gate.size(0), k = w_gate.size(1), tokens = x.numel() / k;
    const Place place(x);
    Tensor h = fresh(with_last(x, n), x);
    if (gu) *gu = fresh({2, tokens, n}, x);
    int64_t bytes = 0;
    check(api.gated_scratch((int32_t)tokens, (int32_t)k, (int32_t)n, 0, &bytes), "cpmk_gated_scratch");
    const Tensor scratch = bytes_like(x, bytes);
    check(api.gated_linear_forward((int32_t)tokens, (int32_t)k, (int32_t)n, dtype_of(x), (int32_t)activation, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
                                   h.data_ptr(), gu ? part(*gu, 0) : nullptr, gu ? part(*gu, 1) : nullptr, address(scratch), place.stream),
          "cpmk_gated_linear_forward");
    return h;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, int64_t activation) {
        Tensor gu;
        Tensor h = gated_forward(x, w_gate, w_up, activation, &gu);
        ctx->save_for_backward({x, w_gate, w_up, gu});
        ctx->saved_data["activation"] = activation;
        return h;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w_gate = saved[1], &w_up = saved[2], &gu = saved[3];
        const int64_t n = w_gate.size(0), k = w_gate.size(1), tokens = x.numel() / k;
        const Tensor dh = laid_out(grads[0]);
        const Place place(x);
        const Tensor dgu = fresh(gu.sizes(), gu);
        Tensor dx, dw_gate, dw_up;
        if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x);
        if (ctx->needs_input_grad(1)) dw_gate = fresh(w_gate.sizes(), w_gate);
        if (ctx->needs_input_grad(2)) dw_up = fresh(w_up.sizes(), w_up);
        int64_t bytes = 0;
        check(api.gated_backward_scratch((int32_t)tokens, (int32_t)k, (int32_t)n, 0, &bytes), "cpmk_gated_backward_scratch");
        const Tensor scratch = bytes_like(x, bytes);
        check(api.gated_linear_backward((int32_t)tokens, (int32_t)k, (int32_t)n, dtype_of(x), (int32_t)ctx->saved_data["activation"].toInt(), dh.data_ptr(),
                                        x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), part(gu, 0), part(gu, 1), part(dgu, 0), part(dgu, 1), address(dx),
                                        address(dw_gate), address(dw_up), address(scratch), place.stream),
              "cpmk_gated_linear_backward");
        return {once(dx, grads[0], x, w_gate, w_up), once(dw_gate, grads[0], x, w_gate, w_up), once(dw_up, grads[0], x, w_gate), Tensor()};
    }
};

Tensor gated_linear(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, int64_t activation) {
    check_gated(x, w_gate, w_up);
    refuse_tangents(x, w_gate, w_up);
    if (tracked(x, w_gate, w_up)) return GatedLinear::apply(x, w_gate, w_up, activation);
    return gated_forward(x, w_gate, w_up, activation, nullptr);
}

// hgu: the hidden activations, and with `keep` the two projections behind them
Tensor block_forward(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, int64_t activation, bool keep, Tensor *hgu) {
    const int64_t n = w_gate.size(0), k = w_gate.size(1), m = w_down.size(0), tokens = x.numel() / k;
    const Place place(x);
    Tensor y = fresh(with_last(x, m), x);
    *hgu = fresh({keep ? 3 : 1, tokens, n}, x);
    int64_t bytes = 0;
    check(api.gated_scratch((int32_t)tokens, (int32_t)k, (int32_t)n, (int32_t)m, &bytes), "cpmk_gated_scratch");
    const Tensor scratch = bytes_like(x, bytes);
    check(api.gated_feed_forward_forward((int32_t)tokens, (int32_t)k, (int32_t)n, (int32_t)m, dtype_of(x), (int32_t)activation, x.data_ptr(), w_gate.data_ptr(),
                                         w_up.data_ptr(), w_down.data_ptr(), part(*hgu, 0), keep ? part(*hgu, 1) : nullptr, keep ? part(*hgu, 2) : nullptr,
                                         y.data_ptr(), address(scratch), place.stream),
          "cpmk_gated_feed_forward_forward");
    return y;
}

struct GatedFeedForward : torch::autograd::Function<GatedFeedForward> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, int64_t activation) {
        Tensor hgu;
        Tensor y = block_forward(x, w_gate, w_up, w_down, activation, true, &hgu);
        ctx->save_for_backward({x, w_gate, w_up, w_down, hgu});
        ctx->saved_data["activation"] = activation;
        return y;
    }

    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w_gate = saved[1], &w_up = saved[2], &w_down = saved[3], &hgu = saved[4];
        const int64_t n = w_gate.size(0), k = w_gate.size(1), m = w_down.size(0), tokens = x.numel() / k;
        const Tensor dy = laid_out(grads[0]);
        const Place place(x);
        const Tensor dgu = fresh({2, tokens, n}, x);
        Tensor dx, dw_gate, dw_up, dw_down;
        if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x);
        if (ctx->needs_input_grad(1)) dw_gate = fresh(w_gate.sizes(), w_gate);
        if (ctx->needs_input_grad(2)) dw_up = fresh(w_up.sizes(), w_up);
        if (ctx->needs_input_grad(3)) dw_down = fresh(w_down.sizes(), w_down);
        int64_t bytes = 0;
        check(api.gated_backward_scratch((int32_t)tokens, (int32_t)k, (int32_t)n, (int32_t)m, &bytes), "cpmk_gated_backward_scratch");
        const Tensor scratch = bytes_like(x, bytes);
        check(api.gated_feed_forward_backward((int32_t)tokens, (int32_t)k, (int32_t)n, (int32_t)m, dtype_of(x), (int32_t)ctx->saved_data["activation"].toInt(),
                                              dy.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), part(hgu, 1), part(hgu, 2),
                                              part(hgu, 0), part(dgu, 0), part(dgu, 1), address(dx), address(dw_gate), address(dw_up), address(dw_down),
                                              address(scratch), place.stream),
              "cpmk_gated_feed_forward_backward");
        return {once(dx, grads[0], x, w_gate, w_up, w_down), once(dw_gate, grads[0], x, w_gate, w_up, w_down), once(dw_up, grads[0], x, w_gate, w_down),
                once(dw_down, grads[0], x, w_gate, w_up), Tensor()};
    }
};

Tensor gated_feed_forward(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, int64_t activation) {
    check_gated(x, w_gate, w_up);
    want(w_down.dim() == 2 && w_down.size(0) >= 1 && w_down.size(0) <= kMost && goes_with(w_down, x, {w_down.size(0), w_gate.size(0)}),
         "gated_feed_forward: w_down must be (M, N), M at most 2^30, contiguous, of x's type and on its device");
    refuse_tangents(x, w_gate, w_up, w_down);
    if (tracked(x, w_gate, w_up, w_down)) return GatedFeedForward::apply(x, w_gate, w_up, w_down, activation);
    Tensor h;
    return block_forward(x, w_gate, w_up, w_down, activation, false, &h);
}

}  // namespace

PYBIND11_MODULE(cpmk_torch, m) {
    const auto unlocked = py::call_guard<py::gil_scoped_release>();
    py::register_local_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused &e) {
            PyErr_SetString(PyExc_AssertionError, e.what());
        }
    });
    m.def("bind", &bind);
    m.def("layernorm_rows", &layernorm_rows, unlocked);
    m.def("gated_linear", &gated_linear, unlocked);
    m.def("gated_feed_forward", &gated_feed_forward, unlocked);
}
