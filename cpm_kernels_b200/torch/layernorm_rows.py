"""``layernorm_rows``: layer norm of every row of token-major activations, with autograd.  cpm_kernels/torch/layernorm.py:8-66
normalises the middle axis of (batch, hidden, seq) and applies the affine step separately; this is the form in front of a linear whose
activations are (tokens, hidden), the layout ``bmm(x, False, w, True)`` takes."""
from typing import Optional

import torch

from ..kernels import layernorm_rows_forward, layernorm_rows_backward, layernorm_rows_backward_scratch
from ..library import cpmk
from ._launch import address, launch, once

_DTYPES = {torch.float16: cpmk.F16, torch.bfloat16: cpmk.BF16, torch.float32: cpmk.F32}


def _forward(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor], rd_mean: bool, statistics: bool):
    """(y, stats): stats holds the rows' means, then their reciprocal deviations, when they are wanted."""
    n = weight.numel()
    rows = x.numel() // n
    y = torch.empty_like(x)
    stats = x.new_empty(2 * rows, dtype=torch.float32) if statistics else None
    mean = address(stats)
    launch(x.get_device(), layernorm_rows_forward, rows, n, _DTYPES[x.dtype], x.data_ptr(), eps, rd_mean, weight.data_ptr(), address(bias), y.data_ptr(),
           mean, mean + 4 * rows if statistics else 0)
    return y, stats


def _launch_backward(rows, n, dtype, dy, x, rd_mean, weight, stats, dx, dweight, dbias, stream):
    scratch = None
    if dweight is not None or dbias is not None:
        scratch = x.new_empty(layernorm_rows_backward_scratch(rows, n), dtype=torch.uint8)
    mean = stats.data_ptr()
    layernorm_rows_backward(rows, n, dtype, dy.data_ptr(), x.data_ptr(), rd_mean, weight.data_ptr(), mean, mean + 4 * rows, address(dx), address(dweight),
                            address(dbias), address(scratch), stream)


class OpLayerNormRows(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor], rd_mean: bool):
        y, stats = _forward(x, eps, weight, bias, rd_mean, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.rd_mean = rd_mean
        return y

    @once
    def backward(ctx, grad_output: torch.Tensor):
        x, weight, stats = ctx.saved_tensors
        n = weight.numel()
        want_x, _, want_weight, want_bias, _ = ctx.needs_input_grad
        dx = torch.empty_like(x) if want_x else None
        dweight = torch.empty_like(weight) if want_weight else None
        dbias = torch.empty_like(weight) if want_bias else None
        launch(x.get_device(), _launch_backward, x.numel() // n, n, _DTYPES[x.dtype], grad_output.contiguous(), x, ctx.rd_mean, weight, stats, dx, dweight,
               dbias)
        return dx, None, dweight, dbias, None


def layernorm_rows(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, rd_mean: bool = True) -> torch.Tensor:
    """Layer norm of ``x`` (..., n) over its last axis, times ``weight`` (n), plus ``bias`` (n) if given; ``rd_mean`` False leaves the
    mean in (the RMS form).  fp16, bf16 or fp32, the same type for all three; statistics in fp32.  Differentiable in x, weight and bias
    (once).  Any n >= 1 and any number of rows, none included."""
    dtype, device = x.dtype, x.device
    assert x.is_cuda and x.is_contiguous() and x.ndim >= 1 and dtype in _DTYPES
    n = x.size(-1)
    assert 1 <= n <= 2 ** 30 and x.numel() // n < 2 ** 31
    assert eps >= 0
    assert weight.device == device and weight.dtype == dtype and weight.shape == (n,) and weight.is_contiguous()
    assert bias is None or (bias.device == device and bias.dtype == dtype and bias.shape == (n,) and bias.is_contiguous())
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return OpLayerNormRows.apply(x, eps, weight, bias, rd_mean)
    return _forward(x, eps, weight, bias, rd_mean, False)[0]
