"""Which stream a given-up wait of the gated feed-forward block is reported for.  The wait is the library's own self-test: a 1 ms limit, on a
barrier on which nothing arrives."""
import pytest
import torch

import cpm_kernels_b200.torch as ct
from cpm_kernels_b200.library import cpmk

pytestmark = pytest.mark.gpu


def give_up(stream):
    cpmk.call("cpmk_selftest_bounded_wait_gated", 1000, stream.cuda_stream)


@pytest.fixture(autouse=True)
def clean():
    assert cpmk.read_status() == 0
    yield
    assert cpmk.read_status() == 0


def test_a_failure_is_its_stream_s():
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    give_up(a)
    cpmk.check_stream(b.cuda_stream)                      # not b's, and not taken from a
    cpmk.check_stream(torch.cuda.current_stream().cuda_stream)
    with pytest.raises(RuntimeError, match=r"status 4.*0x901"):
        cpmk.check_stream(a.cuda_stream)
    cpmk.check_stream(a.cuda_stream)                      # once


def test_read_status_finds_it_on_any_stream():
    streams = [torch.cuda.Stream() for _ in range(5)]
    give_up(streams[3])
    assert cpmk.read_status() == 0x901
    for s in streams:
        cpmk.check_stream(s.cuda_stream)


def test_a_captured_call_s_failure_is_reported_until_it_is_read():
    x, w = torch.ones((4, 64), device="cuda", dtype=torch.half), torch.ones((64, 64), device="cuda", dtype=torch.half)
    want = ct.gated_linear(x, w, w)
    graph, replaying, other = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        give_up(torch.cuda.current_stream())
        h = ct.gated_linear(x, w, w)
    cpmk.check_stream(replaying.cuda_stream)              # captured, not run
    with torch.cuda.stream(replaying):
        graph.replay()
    for s in (replaying, other, replaying):
        with pytest.raises(RuntimeError, match="captured"):
            cpmk.check_stream(s.cuda_stream)
    assert cpmk.read_status() == 0x901
    cpmk.check_stream(replaying.cuda_stream)
    assert torch.equal(h, want)


def test_a_released_stream_starts_clean():
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    give_up(a)
    cpmk.release_workspace(a.cuda_stream)
    cpmk.release_workspace(a.cuda_stream)                # twice is harmless
    x, w = torch.ones((4, 64), device="cuda", dtype=torch.half), torch.ones((64, 64), device="cuda", dtype=torch.half)
    with torch.cuda.stream(b):                           # takes the word that a gave back
        ct.gated_linear(x, w, w)
    cpmk.check_stream(b.cuda_stream)
    cpmk.check_stream(a.cuda_stream)


def test_the_limit_is_checked():
    for limit in (0, 10_000_000):
        with pytest.raises(RuntimeError, match="limit_us"):
            cpmk.call("cpmk_selftest_bounded_wait_gated", limit, None)


def test_a_first_call_without_waits_may_be_captured():
    """Sizes of the generic kernel, and the layer norm: no status words are allocated, so that even a process's first call may be captured."""
    import os
    import subprocess
    import sys
    script = """
import torch
import cpm_kernels_b200.torch as ct
x, w, n = (torch.ones(s, device="cuda", dtype=torch.half) for s in ((4, 7), (5, 7), (7,)))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    h = ct.gated_linear(ct.layernorm_rows(x, 1e-5, n, rd_mean=False), w, w)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(h, ct.gated_linear(ct.layernorm_rows(x, 1e-5, n, rd_mean=False), w, w)) and h.any()
"""
    done = subprocess.run([sys.executable, "-c", script], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
