"""Launchers of the gated feed-forward block.  The reference's callers run it as ``bmm``, ``bmm``, ``gelu``, a product and ``bmm``
(cpm_kernels/torch/gemm.py:233-239, torch/gelu.py:46-47); there is no counterpart of the fused form."""
import ctypes

from .base import DevicePointer, CUDAStream, stream_arg
from ..library import cpmk


def gated_scratch(tokens: int, k: int, n: int, m: int = 0) -> int:
    """Bytes of scratch the two forward launchers want on the current device; ``m`` = 0: ``gated_linear_forward``."""
    out = ctypes.c_int64(0)
    cpmk.call("cpmk_gated_scratch", tokens, k, n, m, ctypes.byref(out))
    return out.value


def gated_backward_scratch(tokens: int, k: int, n: int, m: int = 0) -> int:
    """The same for the two backward launchers."""
    out = ctypes.c_int64(0)
    cpmk.call("cpmk_gated_backward_scratch", tokens, k, n, m, ctypes.byref(out))
    return out.value


def gated_linear_forward(tokens: int, k: int, n: int, dtype: int, activation: int,
                         x: DevicePointer,         # (tokens, k)
                         w_gate: DevicePointer,    # (n, k)
                         w_up: DevicePointer,      # (n, k)
                         h: DevicePointer,         # (tokens, n), written
                         g: DevicePointer,         # (tokens, n), written, or 0
                         u: DevicePointer,         # (tokens, n), written, or 0 with g
                         scratch: DevicePointer,   # gated_scratch(tokens, k, n) bytes
                         stream: CUDAStream):
    """h = act(x w_gate^T) * (x w_up^T)."""
    assert tokens >= 0 and k >= 1 and n >= 1
    cpmk.call("cpmk_gated_linear_forward", tokens, k, n, dtype, activation, x, w_gate, w_up, h, g, u, scratch,
              stream_arg(stream))


def gated_linear_backward(tokens: int, k: int, n: int, dtype: int, activation: int,
                          dh: DevicePointer,        # (tokens, n)
                          x: DevicePointer, w_gate: DevicePointer, w_up: DevicePointer,
                          g: DevicePointer, u: DevicePointer,      # (tokens, n): what the forward pass wrote
                          dg: DevicePointer, du: DevicePointer,    # (tokens, n), written
                          dx: DevicePointer,        # (tokens, k), written, or 0
                          dw_gate: DevicePointer,   # (n, k), written, or 0
                          dw_up: DevicePointer,     # (n, k), written, or 0
                          scratch: DevicePointer,   # gated_backward_scratch(tokens, k, n) bytes
                          stream: CUDAStream):
    assert tokens >= 0 and k >= 1 and n >= 1
    cpmk.call("cpmk_gated_linear_backward", tokens, k, n, dtype, activation, dh, x, w_gate, w_up, g, u, dg, du, dx, dw_gate,
              dw_up, scratch, stream_arg(stream))


def gated_feed_forward_forward(tokens: int, k: int, n: int, m: int, dtype: int, activation: int,
                               x: DevicePointer, w_gate: DevicePointer, w_up: DevicePointer,
                               w_down: DevicePointer,    # (m, n)
                               h: DevicePointer,         # (tokens, n), written
                               g: DevicePointer, u: DevicePointer,      # (tokens, n), written, or 0
                               y: DevicePointer,         # (tokens, m), written
                               scratch: DevicePointer,   # gated_scratch(tokens, k, n, m) bytes
                               stream: CUDAStream):
    """h as gated_linear_forward, y = h w_down^T."""
    assert tokens >= 0 and k >= 1 and n >= 1 and m >= 1
    cpmk.call("cpmk_gated_feed_forward_forward", tokens, k, n, m, dtype, activation, x, w_gate, w_up, w_down, h, g, u, y,
              scratch, stream_arg(stream))


def gated_feed_forward_backward(tokens: int, k: int, n: int, m: int, dtype: int, activation: int,
                                dy: DevicePointer,        # (tokens, m)
                                x: DevicePointer, w_gate: DevicePointer, w_up: DevicePointer, w_down: DevicePointer,
                                g: DevicePointer, u: DevicePointer,
                                h: DevicePointer,         # (tokens, n): what the forward pass wrote, or 0 when dw_down is
                                dg: DevicePointer, du: DevicePointer,    # (tokens, n), written when dx, dw_gate or dw_up is wanted
                                dx: DevicePointer, dw_gate: DevicePointer, dw_up: DevicePointer,
                                dw_down: DevicePointer,   # (m, n), written, or 0
                                scratch: DevicePointer,   # gated_backward_scratch(tokens, k, n, m) bytes
                                stream: CUDAStream):
    assert tokens >= 0 and k >= 1 and n >= 1 and m >= 1
    cpmk.call("cpmk_gated_feed_forward_backward", tokens, k, n, m, dtype, activation, dy, x, w_gate, w_up, w_down, g, u, h, dg, du, dx,
              dw_gate, dw_up, dw_down, scratch, stream_arg(stream))
