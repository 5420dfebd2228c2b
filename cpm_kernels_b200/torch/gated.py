"""``gated_linear`` and ``gated_feed_forward``: the gated feed-forward block act(x Wg^T) * (x Wu^T), times Wd^T, with autograd.

What a caller of cpm_kernels composes from ``bmm`` (torch/gemm.py:233-239), ``gelu`` (torch/gelu.py:46-47) and a product of tensors,
with both projections, the activation and the product in one pass, and the activation's derivative in the epilogue of the product
before it on the way back.  fp16 and bf16, fp32 sums.

What is handed from one product to the next, or kept for the backward pass, has the tensors' type, its precision and its range: in fp16,
hidden activations beyond 65504 are infinite, kept projections too (for the gate's, the activation's limits are taken: 0, or infinity with
slope 1), and the gradients of the projections are zero below 2^-25, as between operators of their own.  bf16 has the range of fp32.

N, K, M and the rows of x are at most 2^30 each.  Extents that are multiples of 8, in tensors that start on 16-byte boundaries, run on the
tensor cores; others on a generic kernel that is far slower (1000 tokens, 1024 -> 2730: 1.1 ms, 2736: 0.04), so a model's widths are
best padded.  Forward-mode differentiation raises a RuntimeError.

The first call on a device is made outside a CUDA-graph capture (it allocates the library's status words); after that calls may be
captured, the backward pass too.  As with PyTorch's own operators, a backward pass is captured only while no graph of an earlier,
uncaptured call on the same leaves is alive: PyTorch ties a leaf's gradient to the stream of that call."""
import torch

from ..library import cpmk
from . import _ext


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``act(x w_gate^T) * (x w_up^T)`` for x (..., K) and weights (N, K): (..., N).  ``activation``: "gelu" (the tanh form of ``gelu``)
    or "silu", applied to the fp32 sums.  fp16 or bf16.  Differentiable (once) in x and both weights; a call that is differentiated
    keeps the two projections, in the tensors' type."""
    assert activation in cpmk.ACTIVATIONS
    return _ext.ext.gated_linear(x, w_gate, w_up, cpmk.ACTIVATIONS[activation])


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "gelu") -> torch.Tensor:
    """``gated_linear(x, w_gate, w_up, activation)`` times ``w_down^T``: x (..., K), w_gate and w_up (N, K), w_down (M, N) -> (..., M).
    The hidden activations between the two are rounded to the tensors' type.  Differentiable (once) in x and the three weights; a call
    that is differentiated keeps the two projections and the hidden activations."""
    assert activation in cpmk.ACTIVATIONS
    return _ext.ext.gated_feed_forward(x, w_gate, w_up, w_down, cpmk.ACTIVATIONS[activation])
