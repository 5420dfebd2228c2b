"""Argument checks of the row layer norm and the gated block that need no GPU: they refuse before any CUDA call."""
import pytest
import torch

import cpm_kernels_b200.kernels as ck
import cpm_kernels_b200.torch as ct
from cpm_kernels_b200.library import cpmk


def test_host_tensors_are_refused():
    x, w = torch.ones((4, 16), dtype=torch.half), torch.ones((8, 16), dtype=torch.half)
    with pytest.raises(AssertionError):
        ct.layernorm_rows(x, 1e-5, torch.ones(16, dtype=torch.half))
    with pytest.raises(AssertionError):
        ct.gated_linear(x, w, w)
    with pytest.raises(AssertionError):
        ct.gated_feed_forward(x, w, w, torch.ones((16, 8), dtype=torch.half))


def test_launchers_check_sizes():
    with pytest.raises(AssertionError):
        ck.layernorm_rows_forward(1, 0, cpmk.F16, 0, 1e-5, True, 0, 0, 0, 0, 0, 0)
    with pytest.raises(AssertionError):
        ck.layernorm_rows_backward(-1, 8, cpmk.F16, 0, 0, True, 0, 0, 0, 0, 0, 0, 0, 0)
    with pytest.raises(AssertionError):
        ck.gated_linear_forward(1, 0, 8, cpmk.F16, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    with pytest.raises(AssertionError):
        ck.gated_linear_backward(1, 8, 0, cpmk.F16, 0, *([0] * 12), 0)
    with pytest.raises(AssertionError):
        ck.gated_feed_forward_forward(1, 8, 8, 0, cpmk.F16, 0, *([0] * 9), 0)
    with pytest.raises(AssertionError):
        ck.gated_feed_forward_backward(-1, 8, 8, 8, cpmk.F16, 0, *([0] * 15), 0)


def test_the_launch_follows_the_tensors_device(monkeypatch):
    """``launch`` makes the tensors' device current for the call when another one is, and hands on that device's stream."""
    from cpm_kernels_b200.torch import _launch
    entered = []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *a):
            entered.append(None)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(_launch, "_raw_stream", lambda device: 1000 + device)
    body = lambda *a: (a, list(entered))
    assert _launch.launch(0, body, 5) == ((5, 1000), [])
    assert _launch.launch(1, body, 5, 6) == ((5, 6, 1001), [1])
    assert entered == [1, None]
