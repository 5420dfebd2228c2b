"""Launchers of the layer norm over rows (token-major activations), forward and backward.  cpm_kernels/kernels/layernorm.py:18-120
normalises the middle axis of (batch, n, m); here every row of (rows, n) is normalised."""
import ctypes

from .base import DevicePointer, CUDAStream, stream_arg
from ..library import cpmk


def layernorm_rows_forward(rows: int, n: int, dtype: int,
                           x: DevicePointer,         # (rows, n)
                           eps: float, rd_mean: bool,
                           weight: DevicePointer,    # (n)
                           bias: DevicePointer,      # (n), or 0
                           y: DevicePointer,         # (rows, n), written
                           mean: DevicePointer,      # (rows) fp32, written, or 0
                           rstd: DevicePointer,      # (rows) fp32, written, or 0 with mean
                           stream: CUDAStream):
    """y = (x - mean) * rstd * weight + bias per row; ``rd_mean`` False: mean = 0 (the RMS form)."""
    assert rows >= 0 and n >= 1
    cpmk.call("cpmk_layernorm_rows_forward", rows, n, dtype, x, float(eps), 1 if rd_mean else 0, weight, bias, y, mean, rstd, stream_arg(stream))


def layernorm_rows_backward_scratch(rows: int, n: int) -> int:
    """Bytes of scratch ``layernorm_rows_backward`` wants on the current device."""
    out = ctypes.c_int64(0)
    cpmk.call("cpmk_layernorm_rows_backward_scratch", rows, n, ctypes.byref(out))
    return out.value


def layernorm_rows_backward(rows: int, n: int, dtype: int,
                            dy: DevicePointer,         # (rows, n)
                            x: DevicePointer,          # (rows, n): the forward pass's input
                            rd_mean: bool,
                            weight: DevicePointer,     # (n)
                            mean: DevicePointer, rstd: DevicePointer,    # (rows) fp32: what the forward pass wrote
                            dx: DevicePointer,         # (rows, n), written, or 0
                            dweight: DevicePointer,    # (n), written, or 0
                            dbias: DevicePointer,      # (n), written, or 0
                            scratch: DevicePointer,    # layernorm_rows_backward_scratch(rows, n) bytes
                            stream: CUDAStream):
    assert rows >= 0 and n >= 1
    cpmk.call("cpmk_layernorm_rows_backward", rows, n, dtype, dy, x, 1 if rd_mean else 0, weight, mean, rstd, dx, dweight, dbias, scratch,
              stream_arg(stream))
