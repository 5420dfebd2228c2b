"""The gated feed-forward block, forward and backward, against the definition in 64 bits.

Tolerances, derived from the arithmetic (eps: the type's, u = 2^-24):
* a product of K terms in fp32 is off by at most K u times the sum of the terms' magnitudes (S), whatever the order of the additions;
* the activations are off by 2^-17 of the value (the exponential's argument is rounded: 88 / ln 2 times 2^-24) and change by at most
  1.13 per unit of their argument, their slopes by at most 1 per unit; the slopes are off by 2^-18;
* every tensor that is stored is rounded once: eps / 2 of the value (half the smallest subnormal below the normal range).
These bounds are carried through the products with magnitudes in place of values.  They hold for every element but are wide for long
sums, so the relative error in the Frobenius norm is held to half a step per rounding on the way as well (a rounding's error is at most
half a step of each value, and a product with independent operands keeps the relative size of such errors)."""
import math

import pytest
import torch

import cpm_kernels_b200.kernels as ck
import cpm_kernels_b200.torch as ct
from cpm_kernels_b200.library import cpmk

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = 2.0 ** -24
# tokens, k, n, m: one token, few, ragged counts around the tile edges, extents that are multiples of 8 only, and extents that are not
SIZES = [(1, 8, 8, 8), (1, 512, 1368, 512), (2, 64, 64, 64), (3, 72, 40, 24), (8, 256, 520, 264), (17, 128, 136, 64), (33, 1000, 264, 120), (64, 64, 200, 72),
         (65, 320, 64, 128), (100, 512, 512, 512), (128, 256, 256, 256), (129, 72, 328, 136), (200, 136, 1032, 40), (255, 64, 128, 256), (256, 192, 384, 64),
         (257, 520, 264, 1032), (513, 256, 640, 264), (1000, 128, 72, 320),
         (1, 5, 3, 1), (5, 33, 7, 9), (70, 130, 67, 31), (130, 12, 129, 20), (9, 64, 64, 63)]


def make(tokens, k, n, m, t, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return ((r(tokens, k)).to(t), (r(n, k) * (2.0 / k ** 0.5)).to(t), (r(n, k) / k ** 0.5).to(t), (r(m, n) / n ** 0.5).to(t),
            r(tokens, m).to(t), r(tokens, n).to(t))


def act_and_slope(v, act):
    if act == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)


class Exact:
    """Values and bounds of everything the block computes; dh is given (gated_linear) or comes from dy and w_down."""

    def __init__(self, x, wg, wu, act, wd=None, dy=None, dh=None):
        t = x.dtype
        half, tiny = torch.finfo(t).eps / 2, TINY[t]
        self.half = half
        x, wg, wu = x.double(), wg.double(), wu.double()
        tokens, k = x.shape
        n = wg.shape[0]
        g, u = x @ wg.T, x @ wu.T
        eg, eu = k * U * (x.abs() @ wg.abs().T), k * U * (x.abs() @ wu.abs().T)
        a, s = act_and_slope(g, act)
        h = a * u
        eh = 1.13 * eg * (u.abs() + eu) + a.abs() * eu + 2.0 ** -17 * h.abs()
        self.h, self.eh = h, eh + half * (h.abs() + eh) + tiny
        if wd is not None:
            wd, dy = wd.double(), dy.double()
            m = wd.shape[0]
            self.y = h @ wd.T
            ey = self.eh @ wd.abs().T + n * U * (h.abs() @ wd.abs().T)
            self.ey = ey + half * (self.y.abs() + ey) + tiny
            dh, edh = dy @ wd, m * U * (dy.abs() @ wd.abs())
            self.dwd = dy.T @ h
            e = dy.abs().T @ self.eh + tokens * U * (dy.abs().T @ h.abs())
            self.edwd = e + half * (self.dwd.abs() + e) + tiny
        else:
            dh, edh = dh.double(), 0.0
        eg, eu = eg + half * (g.abs() + eg) + tiny, eu + half * (u.abs() + eu) + tiny           # g and u are stored
        du, dg = dh * a, dh * u * s
        edu = a.abs() * edh + (dh.abs() + edh) * 1.13 * eg + 2.0 ** -17 * du.abs()
        edg = (u * s).abs() * edh + (dh.abs() + edh) * (s.abs() * eu + (u.abs() + eu) * (eg + 2.0 ** -18)) + 2.0 ** -17 * dg.abs()
        edu, edg = edu + half * (du.abs() + edu) + tiny, edg + half * (dg.abs() + edg) + tiny
        self.dx = dg @ wg + du @ wu
        e = edg @ wg.abs() + edu @ wu.abs() + 2 * n * U * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
        self.edx = e + half * (self.dx.abs() + e) + tiny
        for name, d, ed in (("dwg", dg, edg), ("dwu", du, edu)):
            v = d.T @ x
            e = ed.T @ x.abs() + tokens * U * (d.abs().T @ x.abs())
            setattr(self, name, v)
            setattr(self, "e" + name, e + half * (v.abs() + e) + tiny)

    def check(self, got, name, roundings):
        want, bound = getattr(self, name), getattr(self, "e" + name)
        assert got.shape == want.shape and torch.isfinite(got).all(), name
        off = (got.double() - want).abs()
        assert (off <= bound).all(), "%s: off by %.3g where %.3g is allowed" % (name, off.max(), bound.flatten()[(off - bound).argmax()])
        if want.numel() >= 4096:                          # the norm's bound speaks of many independent errors
            rel = (off.norm() / want.norm()).item()
            assert rel <= roundings * self.half, "%s: relative error %.3g, %d roundings allow %.3g" % (name, rel, roundings, roundings * self.half)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,n,m", SIZES)
def test_gated_linear(tokens, k, n, m, name):
    for act in ("gelu", "silu"):
        x, wg, wu, _, _, dh = make(tokens, k, n, m, TYPES[name], tokens + k)
        ts = [t.clone().requires_grad_() for t in (x, wg, wu)]
        h = ct.gated_linear(*ts, activation=act)
        grads = torch.autograd.grad(h, ts, dh)
        want = Exact(x, wg, wu, act, dh=dh)
        want.check(h, "h", 1)
        for got, what in zip(grads, ("dx", "dwg", "dwu")):
            want.check(got, what, 4)
        assert torch.equal(ct.gated_linear(x, wg, wu, activation=act), h)      # with and without autograd: the same bits


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,k,n,m", SIZES)
def test_gated_feed_forward(tokens, k, n, m, name):
    for act in ("gelu", "silu"):
        x, wg, wu, wd, dy, _ = make(tokens, k, n, m, TYPES[name], tokens + n)
        ts = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
        y = ct.gated_feed_forward(*ts, activation=act)
        grads = torch.autograd.grad(y, ts, dy)
        want = Exact(x, wg, wu, act, wd, dy)
        want.check(y, "y", 2)
        for got, what in zip(grads, ("dx", "dwg", "dwu", "dwd")):
            want.check(got, what, 4)
        assert torch.equal(ct.gated_feed_forward(x, wg, wu, wd, activation=act), y)
    torch.cuda.synchronize()
    assert cpmk.read_status() == 0


# whole layers; sums that are cut along k: of every product (600 tokens), of left-over tiles behind whole waves (2304), of the three weight
# gradients together (5000, 3001)
@pytest.mark.parametrize("tokens,k,n,m,name", [(1, 4096, 10240, 4096, "fp16"), (48, 4096, 10240, 4096, "bf16"), (700, 4096, 1024, 2048, "bf16"),
                                               (1500, 1024, 4096, 1024, "fp16"), (600, 4096, 512, 4096, "fp16"), (2304, 64, 4096, 2560, "bf16"),
                                               (5000, 256, 264, 520, "bf16"), (3001, 64, 136, 72, "fp16"), (256, 2048, 1368, 2048, "fp16"),
                                               (257, 2048, 1368, 2048, "fp16")])
def test_wide_layers(tokens, k, n, m, name):
    x, wg, wu, wd, dy, _ = make(tokens, k, n, m, TYPES[name], 5)
    ts = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    y = ct.gated_feed_forward(*ts)
    grads = torch.autograd.grad(y, ts, dy)
    want = Exact(x, wg, wu, "gelu", wd, dy)
    want.check(y, "y", 2)
    for got, what in zip(grads, ("dx", "dwg", "dwu", "dwd")):
        want.check(got, what, 4)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k,n", [(8, 64), (7, 5)])
def test_activation_over_its_range(act, name, k, n):
    """x = (v, 0, ...), w_gate and w_up rows (1, 0, ...): g = u = v for v over the whole range of both signs, then dh = 1."""
    t = TYPES[name]
    v = torch.cat([torch.linspace(-12, 12, 4001), torch.tensor([0.0, -0.0, 30.0, -30.0, 89.0, -89.0, 200.0, -200.0, 1e-7, -1e-7])]).cuda().to(t)
    x = torch.zeros((v.numel(), k), device="cuda", dtype=t)
    x[:, 0] = v
    w = torch.zeros((n, k), device="cuda", dtype=t)
    w[:, 0] = 1
    ts = [z.clone().requires_grad_() for z in (x, w, w)]
    h = ct.gated_linear(*ts, activation=act)
    dh = torch.zeros_like(h)
    dh[:, 0] = 1
    grads = torch.autograd.grad(h, ts, dh)
    want = Exact(x, w, w, act, dh=dh)
    want.check(h, "h", 1)
    want.check(grads[0], "dx", 4)


def test_values_that_are_not_numbers_stay_in_their_row():
    for tokens, k, n, m in ((6, 64, 64, 64), (300, 128, 256, 128), (6, 9, 11, 7)):
        x, wg, wu, wd, _, _ = make(tokens, k, n, m, torch.bfloat16, 3)
        clean = ct.gated_feed_forward(x, wg, wu, wd)
        x[2, 1] = float("nan")
        y = ct.gated_feed_forward(x, wg, wu, wd)
        assert torch.isnan(y[2]).all()
        keep = [r for r in range(tokens) if r != 2]
        assert torch.equal(y[keep], clean[keep])


def test_no_tokens():
    for k, n, m in ((64, 64, 64), (3, 5, 7)):
        _, wg, wu, wd, _, _ = make(1, k, n, m, torch.half)
        ts = [torch.empty((0, k), device="cuda", dtype=torch.half).requires_grad_(), *(w.requires_grad_() for w in (wg, wu, wd))]
        y = ct.gated_feed_forward(*ts)
        assert y.shape == (0, m)
        grads = torch.autograd.grad(y, ts, torch.empty_like(y))
        assert grads[0].shape == (0, k) and not any(g.any() for g in grads[1:])
        h = ct.gated_linear(*ts[:3])
        assert h.shape == (0, n)
        assert not any(g.any() for g in torch.autograd.grad(h, ts[:3], torch.empty_like(h)))


@pytest.mark.parametrize("tokens", [3, 300])
def test_leading_axes_views_and_expanded_gradients(tokens):
    x, wg, wu, wd, _, _ = make(2 * tokens, 64, 136, 64, torch.half, 2)
    big = torch.stack([x, x * 0.5]).view(2, 2, tokens, 64)
    xs = big[1].requires_grad_()
    ts = [xs, *(w.requires_grad_() for w in (wg, wu, wd))]
    y = ct.gated_feed_forward(*ts)
    assert y.shape == (2, tokens, 64)
    got = torch.autograd.grad(y.sum(), ts)
    want = torch.autograd.grad(ct.gated_feed_forward(*ts), ts, torch.ones_like(y))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("tokens,k,n,m", [(5, 64, 72, 64), (300, 136, 256, 64)])
def test_pointers_that_are_not_aligned_to_16_bytes(tokens, k, n, m):
    x, wg, wu, wd, dy, _ = make(tokens, k, n, m, torch.bfloat16, 4)

    def moved(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    for which in range(5):
        ts = [moved(t) if i == which else t.clone() for i, t in enumerate((x, wg, wu, wd))]
        ts = [t.requires_grad_() for t in ts]
        y = ct.gated_feed_forward(*ts)
        grads = torch.autograd.grad(y, ts, moved(dy) if which == 4 else dy)
        want = Exact(x, wg, wu, "gelu", wd, dy)
        want.check(y, "y", 2)
        for got, what in zip(grads, ("dx", "dwg", "dwu", "dwd")):
            want.check(got, what, 4)


@pytest.mark.parametrize("tokens,k,n,m", [(19, 64, 72, 40), (300, 136, 256, 64), (7, 5, 3, 2)])
def test_some_gradients_only(tokens, k, n, m):
    x, wg, wu, wd, dy, dh = make(tokens, k, n, m, torch.half, 6)
    full = None
    for mask in (15, 1, 2, 4, 8, 9, 6, 7):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, wg, wu, wd))]
        got = torch.autograd.grad(ct.gated_feed_forward(*ts), [t for t in ts if t.requires_grad], dy)
        full = got if mask == 15 else full
        for i, v in zip([i for i in range(4) if mask >> i & 1], got):
            assert torch.equal(v, full[i])
    full = None
    for mask in (7, 1, 2, 4, 6):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, wg, wu))]
        got = torch.autograd.grad(ct.gated_linear(*ts), [t for t in ts if t.requires_grad], dh)
        full = got if mask == 7 else full
        for i, v in zip([i for i in range(3) if mask >> i & 1], got):
            assert torch.equal(v, full[i])


@pytest.mark.parametrize("tokens", [4, 300])
def test_a_thread_that_has_not_used_the_device(tokens):
    """The first CUDA call of a thread: no context is current on it, and PyTorch serves the outputs from its cache."""
    import threading
    x, wg, wu, wd, _, _ = make(tokens, 64, 64, 64, torch.half, 14)
    want = ct.gated_feed_forward(x, wg, wu, wd)
    torch.cuda.synchronize()
    got = []
    thread = threading.Thread(target=lambda: got.append(ct.gated_feed_forward(x, wg, wu, wd)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_offsets_beyond_32_bits():
    """2.2e9 hidden activations: rows at both ends and around the 2^31st element against the same rows among 300 of their own."""
    tokens, k, n, m = 262_200, 64, 8200, 64
    x, wg, wu, wd, dy, _ = make(tokens, k, n, m, torch.half, 15)
    x.requires_grad_()
    y = ct.gated_feed_forward(x, wg, wu, wd)
    (dx,) = torch.autograd.grad(y, x, dy)
    h = ct.gated_linear(x.detach(), wg, wu)
    for at in (0, 2 ** 31 // n - 150, tokens - 300):
        part = x.detach()[at:at + 300].clone().requires_grad_()
        z = ct.gated_feed_forward(part, wg, wu, wd)
        (dpart,) = torch.autograd.grad(z, part, dy[at:at + 300].clone())
        # other tiles are cut along k than in the large call: a step of fp16 apart, 2^-8 below 8 and 2^-6 below 32
        assert torch.equal(ct.gated_linear(part.detach(), wg, wu), h[at:at + 300])
        assert (z - y[at:at + 300]).abs().max() <= 2.0 ** -8 and (dpart - dx[at:at + 300]).abs().max() <= 2.0 ** -6
    Exact(x.detach()[-40:], wg, wu, "gelu", wd, dy[-40:]).check(y[-40:], "y", 2)


def test_the_same_tensor_as_both_weights():
    x, wg, _, _, _, dh = make(40, 64, 64, 64, torch.half, 7)
    a, b = wg.clone().requires_grad_(), wg.clone().requires_grad_()
    one = torch.autograd.grad(ct.gated_linear(x, a, a), a, dh)[0]
    two = torch.autograd.grad(ct.gated_linear(x, a, b), (a, b), dh)
    assert torch.equal(one, two[0] + two[1])


@pytest.mark.parametrize("tokens,k,n,m", [(1, 64, 72, 40), (20, 72, 136, 200), (130, 64, 72, 264), (300, 136, 256, 64), (7, 5, 3, 2)])
def test_nothing_is_written_outside_the_outputs(tokens, k, n, m):
    x, wg, wu, wd, dy, _ = make(tokens, k, n, m, torch.half, 8)
    s = torch.cuda.current_stream().cuda_stream
    pad = 64
    guard = lambda count: torch.full((count + 2 * pad,), 7.0, dtype=torch.half, device="cuda")
    h, g, u, dg, du = (guard(tokens * n) for _ in range(5))
    y, dx, dwg, dwu, dwd = guard(tokens * m), guard(tokens * k), guard(n * k), guard(n * k), guard(m * n)
    at = lambda t: t.data_ptr() + 2 * pad
    need = max(ck.gated_scratch(tokens, k, n, m), ck.gated_backward_scratch(tokens, k, n, m))
    scratch = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
    p = lambda t: t.data_ptr()
    ck.gated_feed_forward_forward(tokens, k, n, m, cpmk.F16, 0, p(x), p(wg), p(wu), p(wd), at(h), at(g), at(u), at(y), p(scratch), s)
    ck.gated_feed_forward_backward(tokens, k, n, m, cpmk.F16, 0, p(dy), p(x), p(wg), p(wu), p(wd), at(g), at(u), at(h), at(dg), at(du), at(dx), at(dwg),
                                   at(dwu), at(dwd), p(scratch), s)
    for t in (h, g, u, dg, du, y, dx, dwg, dwu, dwd):
        assert (t[:pad] == 7).all() and (t[-pad:] == 7).all()
    assert (scratch[need:] == 77).all()
    want = Exact(x, wg, wu, "gelu", wd, dy)
    inner = lambda t, *shape: t[pad:-pad].view(*shape)
    want.check(inner(h, tokens, n), "h", 1)
    want.check(inner(y, tokens, m), "y", 2)
    want.check(inner(dx, tokens, k), "dx", 4)
    want.check(inner(dwg, n, k), "dwg", 4)
    want.check(inner(dwu, n, k), "dwu", 4)
    want.check(inner(dwd, m, n), "dwd", 4)


@pytest.mark.parametrize("tokens,k,n,m", [(5, 512, 1024, 512), (700, 256, 512, 256), (40, 30, 50, 20)])
def test_same_bits_on_every_run_and_stream(tokens, k, n, m):
    x, wg, wu, wd, dy, _ = make(tokens, k, n, m, torch.bfloat16, 9)
    results = []
    for s in [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ts = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
            y = ct.gated_feed_forward(*ts)
            results.append((y.detach(), *torch.autograd.grad(y, ts, dy)))
    torch.cuda.synchronize()
    for r in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], r))


@pytest.mark.parametrize("tokens,k,n,m", [(4, 256, 520, 256), (300, 256, 512, 256), (4, 25, 52, 25)])
def test_two_captured_graphs_replayed_side_by_side(tokens, k, n, m):
    """Two graphs captured from calls on the same stream, replayed at the same time on two streams with new inputs."""
    graphs, outs, inputs = [], [], []
    for seed in (1, 2):
        x, wg, wu, wd, dy, _ = make(tokens, k, n, m, torch.half, seed)
        ts = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]

        def step(ts=ts, dy=dy):
            y = ct.gated_feed_forward(*ts)
            return (y.detach(), *torch.autograd.grad(y, ts, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
        inputs.append((ts, step))
    for seed, (ts, _) in enumerate(inputs):
        with torch.no_grad():
            ts[0].copy_(make(tokens, k, n, m, torch.half, 50 + seed)[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out, (_, step) in zip(outs, inputs):
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
    assert cpmk.read_status() == 0


def test_refusals():
    x, wg, wu, wd, _, _ = make(4, 16, 24, 8, torch.half)
    for bad in (lambda: ct.gated_linear(x, wg, wu, activation="tanh"), lambda: ct.gated_linear(x.float(), wg.float(), wu.float()),
                lambda: ct.gated_linear(x, wg, wu.bfloat16()), lambda: ct.gated_linear(x, wg, wu[:8]), lambda: ct.gated_linear(x[:, :8], wg, wu),
                lambda: ct.gated_linear(x, wg.t().contiguous().t(), wu), lambda: ct.gated_linear(x.cpu(), wg, wu), lambda: ct.gated_linear(x, wg.cpu(), wu),
                lambda: ct.gated_linear(x[:, ::2], wg[:, :8].contiguous(), wu[:, :8].contiguous()),
                lambda: ct.gated_feed_forward(x, wg, wu, wd[:, :16].contiguous()), lambda: ct.gated_feed_forward(x, wg, wu, wd[0]),
                lambda: ct.gated_feed_forward(x, wg[:0], wu[:0], wd[:, :0].contiguous())):
        with pytest.raises(AssertionError):
            bad()
    s = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    h = torch.empty((4, 24), device="cuda", dtype=torch.half)
    for args in ((4, 16, 24, cpmk.F32, 0, p(x), p(wg), p(wu), p(h), 0, 0, 0, s), (4, 16, 24, 0, 5, p(x), p(wg), p(wu), p(h), 0, 0, 0, s),
                 (4, 16, 24, 0, 0, 0, p(wg), p(wu), p(h), 0, 0, 0, s), (4, 16, 24, 0, 0, p(x), p(wg), p(wu), p(h), p(h), 0, 0, s),
                 (4, 16, 24, 0, 0, p(x) + 1, p(wg), p(wu), p(h), 0, 0, 0, s), (2 ** 30 + 1, 16, 24, 0, 0, p(x), p(wg), p(wu), p(h), 0, 0, 0, s),
                 (4, 16, 24, 0, 0, p(x), p(wg), p(wu), p(h), 0, 0, 0, s), (4, 16, 24, 0, 0, p(x), p(wg), p(wu), p(h), 0, 0, p(x) + 8, s)):
        with pytest.raises(RuntimeError):
            ck.gated_linear_forward(*args)


@pytest.mark.parametrize("tokens,k,n", [(6, 64, 136), (300, 256, 512)])
def test_layer_norm_block_and_residual_together(tokens, k, n):
    """The second half of a layer: x + gated_feed_forward(layernorm_rows(x)).  The relative errors in the norm: half a step per rounding
    (layer norm, hidden activations, block, sum; on the way back those of the projections, dg and du, dx of the block, the layer norm's
    gradient and the residual's sum)."""
    t = torch.bfloat16
    x, wg, wu, wd, dy, _ = make(tokens, k, n, k, t, 11)
    w = (1 + 0.1 * torch.randn(k, generator=torch.Generator("cuda").manual_seed(1), device="cuda")).to(t)
    ts = [v.clone().requires_grad_() for v in (x, w, wg, wu, wd)]
    y = ts[0] + ct.gated_feed_forward(ct.layernorm_rows(ts[0], 1e-5, ts[1], rd_mean=False), *ts[2:], activation="silu")
    grads = torch.autograd.grad(y, ts, dy)
    ds = [v.double().requires_grad_() for v in (x, w, wg, wu, wd)]
    z = ds[0] / torch.sqrt(ds[0].square().mean(-1, keepdim=True) + 1e-5) * ds[1]
    a, _ = act_and_slope(z @ ds[2].T, "silu")
    want = ds[0] + (a * (z @ ds[3].T)) @ ds[4].T
    wanted = torch.autograd.grad(want, ds, dy.double())
    half = torch.finfo(t).eps / 2
    for got, v, roundings in zip((y, *grads), (want, *wanted), (4, 8, 8, 6, 6, 4)):
        assert ((got.double() - v).norm() / v.norm()).item() <= roundings * half


def test_int8_linear_after_the_gated_linear():
    """The gated linear's result as the operand of the framework's int8 linear: its quantiser takes it as it is."""
    x, wg, wu, wd, _, _ = make(64, 256, 512, 256, torch.half, 13)
    h = ct.gated_linear(x, wg, wu)
    y = ct.bmm(h[None], False, wd[None], True, int8=True)[0]
    want = Exact(x, wg, wu, "gelu", wd, torch.zeros((64, 256), device="cuda")).y
    # codes are off by half a step of absmax / 127, absmax about 4 standard deviations: 1 / 110 of a value's size per operand, RMS / sqrt 3
    assert ((y.double() - want).norm() / want.norm()).item() <= 2 / 60
