"""``gated_linear`` and ``gated_feed_forward``: the gated feed-forward block act(x Wg^T) * (x Wu^T), times Wd^T, with autograd.

What a caller of cpm_kernels composes from ``bmm`` (torch/gemm.py:233-239), ``gelu`` (torch/gelu.py:46-47) and a product of tensors,
with both projections, the activation and the product in one pass, and the activation's derivative in the epilogue of the product
before it on the way back.  fp16 and bf16, fp32 sums."""
import torch

from ..kernels import gated_linear_forward, gated_linear_backward, gated_feed_forward_forward, gated_feed_forward_backward, gated_scratch, gated_backward_scratch
from ..library import cpmk
from ._launch import address, launch, once

_DTYPES = {torch.float16: cpmk.F16, torch.bfloat16: cpmk.BF16}


def _check(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str) -> None:
    dtype, device = x.dtype, x.device
    assert x.is_cuda and x.is_contiguous() and x.ndim >= 1 and dtype in _DTYPES
    k, n = x.size(-1), w_gate.size(0)
    assert k >= 1 and n >= 1 and x.numel() // k <= 2 ** 30
    assert w_gate.device == device and w_gate.dtype == dtype and w_gate.shape == (n, k) and w_gate.is_contiguous()
    assert w_up.device == device and w_up.dtype == dtype and w_up.shape == (n, k) and w_up.is_contiguous()
    assert activation in cpmk.ACTIVATIONS


def _scratch(size: int, x: torch.Tensor):
    return x.new_empty(size, dtype=torch.uint8) if size else None


def _launch_linear(x, w_gate, w_up, activation, h, gu, stream):
    n, k = w_gate.shape
    tokens = x.numel() // k
    scratch = _scratch(gated_scratch(tokens, k, n), x)
    g = address(gu)
    gated_linear_forward(tokens, k, n, _DTYPES[x.dtype], cpmk.ACTIVATIONS[activation], x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), h.data_ptr(),
                         g, g + 2 * tokens * n if g else 0, address(scratch), stream)


def _linear_forward(x, w_gate, w_up, activation: str, save: bool):
    n, k = w_gate.shape
    h = x.new_empty((*x.shape[:-1], n))
    gu = x.new_empty((2, x.numel() // k, n)) if save else None
    launch(x.get_device(), _launch_linear, x, w_gate, w_up, activation, h, gu)
    return h, gu


def _launch_linear_backward(x, w_gate, w_up, activation, gu, dh, dgu, dx, dw_gate, dw_up, stream):
    n, k = w_gate.shape
    tokens = x.numel() // k
    scratch = _scratch(gated_backward_scratch(tokens, k, n), x)
    g, dg, each = gu.data_ptr(), dgu.data_ptr(), 2 * tokens * n
    gated_linear_backward(tokens, k, n, _DTYPES[x.dtype], cpmk.ACTIVATIONS[activation], dh.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
                          g, g + each, dg, dg + each, address(dx), address(dw_gate), address(dw_up), address(scratch), stream)


class OpGatedLinear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str):
        h, gu = _linear_forward(x, w_gate, w_up, activation, True)
        ctx.save_for_backward(x, w_gate, w_up, gu)
        ctx.activation = activation
        return h

    @once
    def backward(ctx, grad_output: torch.Tensor):
        x, w_gate, w_up, gu = ctx.saved_tensors
        dgu = torch.empty_like(gu)
        dx, dw_gate, dw_up = (torch.empty_like(t) if need else None for t, need in zip((x, w_gate, w_up), ctx.needs_input_grad))
        launch(x.get_device(), _launch_linear_backward, x, w_gate, w_up, ctx.activation, gu, grad_output.contiguous(), dgu, dx, dw_gate, dw_up)
        return dx, dw_gate, dw_up, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``act(x w_gate^T) * (x w_up^T)`` for x (..., K) and weights (N, K): (..., N).  ``activation``: "gelu" (the tanh form of ``gelu``)
    or "silu", applied to the fp32 sums.  fp16 or bf16.  Differentiable (once) in x and both weights; a call that is differentiated
    keeps the two projections, in the tensors' type."""
    _check(x, w_gate, w_up, activation)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        return OpGatedLinear.apply(x, w_gate, w_up, activation)
    return _linear_forward(x, w_gate, w_up, activation, False)[0]


def _launch_block(x, w_gate, w_up, w_down, activation, hgu, y, stream):
    n, k = w_gate.shape
    m = w_down.size(0)
    tokens = x.numel() // k
    scratch = _scratch(gated_scratch(tokens, k, n, m), x)
    h, each = hgu.data_ptr(), 2 * tokens * n
    save = hgu.size(0) == 3
    gated_feed_forward_forward(tokens, k, n, m, _DTYPES[x.dtype], cpmk.ACTIVATIONS[activation], x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
                               w_down.data_ptr(), h, h + each if save else 0, h + 2 * each if save else 0, y.data_ptr(),
                               address(scratch), stream)


def _block_forward(x, w_gate, w_up, w_down, activation: str, save: bool):
    n, k = w_gate.shape
    y = x.new_empty((*x.shape[:-1], w_down.size(0)))
    hgu = x.new_empty((3 if save else 1, x.numel() // k, n))      # h, and g, u for the backward pass
    launch(x.get_device(), _launch_block, x, w_gate, w_up, w_down, activation, hgu, y)
    return y, hgu


def _launch_block_backward(x, w_gate, w_up, w_down, activation, hgu, dy, dx, dw_gate, dw_up, dw_down, stream):
    n, k = w_gate.shape
    m = w_down.size(0)
    tokens = x.numel() // k
    dgu = x.new_empty((2, tokens, n))
    scratch = _scratch(gated_backward_scratch(tokens, k, n, m), x)
    h, dg, each = hgu.data_ptr(), dgu.data_ptr(), 2 * tokens * n
    gated_feed_forward_backward(tokens, k, n, m, _DTYPES[x.dtype], cpmk.ACTIVATIONS[activation], dy.data_ptr(), x.data_ptr(), w_gate.data_ptr(),
                                w_up.data_ptr(), w_down.data_ptr(), h + each, h + 2 * each, h, dg, dg + each,
                                address(dx), address(dw_gate), address(dw_up), address(dw_down), address(scratch), stream)


class OpGatedFeedForward(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str):
        y, hgu = _block_forward(x, w_gate, w_up, w_down, activation, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, hgu)
        ctx.activation = activation
        return y

    @once
    def backward(ctx, grad_output: torch.Tensor):
        x, w_gate, w_up, w_down, hgu = ctx.saved_tensors
        dx, dw_gate, dw_up, dw_down = (torch.empty_like(t) if need else None for t, need in zip((x, w_gate, w_up, w_down), ctx.needs_input_grad))
        launch(x.get_device(), _launch_block_backward, x, w_gate, w_up, w_down, ctx.activation, hgu, grad_output.contiguous(), dx, dw_gate, dw_up, dw_down)
        return dx, dw_gate, dw_up, dw_down, None


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``gated_linear(x, w_gate, w_up, activation)`` times ``w_down^T``: x (..., K), w_gate and w_up (N, K), w_down (M, N) -> (..., M).
    The hidden activations between the two are rounded to the tensors' type.  Differentiable (once) in x and the three weights; a call
    that is differentiated keeps the two projections and the hidden activations."""
    _check(x, w_gate, w_up, activation)
    assert w_down.device == x.device and w_down.dtype == x.dtype and w_down.ndim == 2 and w_down.is_contiguous()
    assert w_down.size(0) >= 1 and w_down.size(1) == w_gate.size(0)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad):
        return OpGatedFeedForward.apply(x, w_gate, w_up, w_down, activation)
    return _block_forward(x, w_gate, w_up, w_down, activation, False)[0]
