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


def test_refusals_say_what_is_wanted():
    x, w = torch.ones((4, 16), dtype=torch.half), torch.ones((8, 16), dtype=torch.half)
    with pytest.raises(AssertionError, match="contiguous CUDA tensor"):
        ct.layernorm_rows(x, 1e-5, x[0])
    with pytest.raises(AssertionError, match="contiguous CUDA tensor"):
        ct.gated_linear(x, w, w)
    with pytest.raises(AssertionError):
        ct.gated_linear(x, w, w, "tanh")
    with pytest.raises(TypeError):
        ct.layernorm_rows(None, 1e-5, x[0])


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


def test_the_autograd_module_is_built_and_takes_every_entry_point(built_library):
    from cpm_kernels_b200 import build
    from cpm_kernels_b200.torch import _ext
    import os
    assert os.path.getsize(build.EXT_PATH) > 0
    with pytest.raises(RuntimeError):
        _ext.ext.bind([0])
    for name in _ext._ENTRY_POINTS[1:]:
        assert name in cpmk.SIGNATURES


def test_a_missing_autograd_module_fails_loudly(monkeypatch, tmp_path):
    from cpm_kernels_b200.torch import _ext
    monkeypatch.setattr(_ext, "EXT_PATH", str(tmp_path / "nope.so"))
    with pytest.raises(RuntimeError, match="no fallback"):
        _ext._load()


def test_another_pytorch_asks_for_another_autograd_module(built_library, monkeypatch):
    from cpm_kernels_b200 import build
    assert build.EXT_PATH == build.ext_path() and not build._ext_is_stale()
    monkeypatch.setattr(build, "_torch_version", lambda: "0.0.1")
    assert build.ext_path() != build.EXT_PATH
    monkeypatch.setattr(build, "EXT_PATH", build.ext_path())
    assert build._ext_is_stale() and build.is_stale()
    monkeypatch.setattr(build, "_torch_version", lambda: None)
    assert not build._ext_is_stale()                     # no PyTorch: the library alone


def test_the_other_operators_do_not_need_the_autograd_module(built_library, tmp_path):
    import os
    import subprocess
    import sys
    script = """
import cpm_kernels_b200.build as build
build.EXT_PATH = %r
import cpm_kernels_b200.torch as ct
assert ct.bmm and ct.gelu and ct.transpose
import torch
for call in (lambda: ct.layernorm_rows(torch.ones(4), 1e-5, torch.ones(4)), lambda: ct.gated_linear(torch.ones(4), torch.ones(4, 4), torch.ones(4, 4))):
    try:
        call()
    except %s as e:
        continue
    raise SystemExit("the call went through without its module")
"""
    broken = tmp_path / "broken.so"
    broken.write_bytes(b"not a shared library")
    for path, error in ((str(tmp_path / "nope.so"), "RuntimeError"), (str(broken), "ImportError")):
        done = subprocess.run([sys.executable, "-c", script % (path, error)], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                              capture_output=True, text=True)
        assert done.returncode == 0, done.stderr
