"""``gated_linear`` and ``gated_feed_forward``: the gated feed-forward block act(x Wg^T) * (x Wu^T), times Wd^T, with autograd.

What a caller of cpm_kernels composes from ``bmm`` (torch/gemm.py:233-239), ``gelu`` (torch/gelu.py:46-47) and a product of tensors,
with both projections, the activation and the product in one pass, and the activation's derivative in the epilogue of the product
before it on the way back.  fp16 and bf16, fp32 sums.

The first call on a device is made outside a CUDA-graph capture (it allocates the library's status word); after that calls may be
captured, the backward pass too.  As with PyTorch's own operators, a backward pass is captured only while no graph of an earlier,
uncaptured call on the same leaves is alive: PyTorch ties a leaf's gradient to the stream of that call."""
import torch

from ..library import cpmk
from ._ext import ext


def _check(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str) -> None:
    dtype, device = x.dtype, x.device
    assert x.is_cuda and x.is_contiguous() and x.ndim >= 1 and (dtype == torch.float16 or dtype == torch.bfloat16)
    assert w_gate.ndim == 2
    n, k = w_gate.shape
    assert k >= 1 and n >= 1 and x.size(-1) == k and x.numel() // k <= 2 ** 30
    assert w_gate.device == device and w_gate.dtype == dtype and w_gate.is_contiguous()
    assert w_up.device == device and w_up.dtype == dtype and w_up.shape == (n, k) and w_up.is_contiguous()
    assert activation in cpmk.ACTIVATIONS


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``act(x w_gate^T) * (x w_up^T)`` for x (..., K) and weights (N, K): (..., N).  ``activation``: "gelu" (the tanh form of ``gelu``)
    or "silu", applied to the fp32 sums.  fp16 or bf16.  Differentiable (once) in x and both weights; a call that is differentiated
    keeps the two projections, in the tensors' type."""
    _check(x, w_gate, w_up, activation)
    return ext.gated_linear(x, w_gate, w_up, cpmk.ACTIVATIONS[activation])


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``gated_linear(x, w_gate, w_up, activation)`` times ``w_down^T``: x (..., K), w_gate and w_up (N, K), w_down (M, N) -> (..., M).
    The hidden activations between the two are rounded to the tensors' type.  Differentiable (once) in x and the three weights; a call
    that is differentiated keeps the two projections and the hidden activations."""
    _check(x, w_gate, w_up, activation)
    assert w_down.device == x.device and w_down.dtype == x.dtype and w_down.ndim == 2 and w_down.is_contiguous()
    assert w_down.size(0) >= 1 and w_down.size(1) == w_gate.size(0)
    return ext.gated_feed_forward(x, w_gate, w_up, w_down, cpmk.ACTIVATIONS[activation])
