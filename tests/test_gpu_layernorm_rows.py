"""Layer norm over rows, forward and backward, against the definition in 64 bits.

Tolerances, derived from the arithmetic: an output of type t is one rounding (half a step, eps(t) / 2 of the value; half of the smallest
subnormal below the normal range) of an fp32 result.  The fp32 result is off by its sums: a sum over n terms that 32 or more threads
share adds at most n / 32 + 10 numbers one after another, each addition off by 2^-24 of a partial sum that is no larger than the sum
of magnitudes; a further 8 roundings of 2^-24 happen on the way to the output.  Column sums add at most all rows one after another."""
import numpy as np
import pytest
import torch

import cpm_kernels_b200.kernels as ck
import cpm_kernels_b200.torch as ct
from cpm_kernels_b200.library import cpmk

pytestmark = pytest.mark.gpu
EPS = 1e-5
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TINY = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 2.0 ** -150}
SIZES = [(1, 1), (1, 4096), (3, 8), (5, 7), (2, 31), (33, 32), (7, 33), (130, 129), (64, 256), (9, 1000), (300, 1024), (257, 1032), (31, 4096),
         (1000, 64), (5, 8192), (4, 16384), (3, 16392), (2, 20001), (12, 5001), (2, 33000), (700, 520), (37, 16385), (300, 9000), (9, 3),
         (4000, 77), (5000, 515), (2500, 1003), (1300, 4099), (400, 9003), (600, 2050), (20, 1001), (150, 16367), (450, 16369),
         (130, 16400), (90, 33001), (45, 66000),
         (5000, 1024), (4800, 1000), (6001, 300), (5003, 769), (4737, 333), (1300, 2048), (1200, 3584)]


def make(rows, n, t, seed=0, offset=0.25):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return ((r(rows, n) * 1.5 + offset).to(t), (1 + 0.2 * r(n)).to(t), (0.3 * r(n)).to(t), r(rows, n).to(t))


def exact(x, w, b, dy, eps, rd_mean):
    """(y, dx, dw, db) in 64 bits and the error bounds of the fp32 results before their last rounding."""
    x, w, dy = x.double(), w.double(), dy.double()
    rows, n = x.shape
    mean = x.mean(-1, keepdim=True) if rd_mean else torch.zeros_like(x[:, :1])
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w + (b.double() if b is not None else 0)
    g = dy * w
    c1 = g.mean(-1, keepdim=True) if rd_mean else torch.zeros_like(mean)
    c2 = (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    u, k = 2.0 ** -24, n / 32 + 18
    size = x.abs().mean(-1, keepdim=True) * rstd if rd_mean else torch.zeros_like(mean)      # how far the mean can be off, in units of the row
    e_xh = k * u * (xh.abs() + size + x.abs() * rstd * (1 if rd_mean else 0) * 0.1)
    e_y = e_xh * w.abs() + 2 * u * (y.abs() + (xh * w).abs())
    e_c2 = k * u * (g * xh).abs().mean(-1, keepdim=True) + (g.abs() * e_xh).mean(-1, keepdim=True)
    e_dx = rstd * (k * u * (g.abs() + g.abs().mean(-1, keepdim=True) + (xh * c2).abs()) + xh.abs() * e_c2 + e_xh * c2.abs()) + k * u * dx.abs()
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = (rows + 8) * u * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    e_db = (rows + 8) * u * dy.abs().sum(0)
    return (y, dx, dw, db), (e_y, e_dx, e_dw, e_db)


def check(got, want, bound, name, what=""):
    t = got.dtype
    tol = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + TINY[name]
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), "%s: off by %.3g where %.3g is allowed" % (what, off.max(), tol.flatten()[off.argmax()])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward_and_backward(rows, n, name):
    for rd_mean, bias in ((True, True), (False, False), (True, False), (False, True)):
        x, w, b, dy = make(rows, n, TYPES[name], rows + n)
        if n == 1 and rd_mean:
            continue                                     # one value less its own mean: see test_constant_rows
        b = b if bias else None
        leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
        y = ct.layernorm_rows(leaves[0], EPS, leaves[1], leaves[2] if bias else None, rd_mean=rd_mean)
        grads = torch.autograd.grad(y, leaves, dy)
        want, bound = exact(x, w, b, dy, EPS, rd_mean)
        check(y, want[0], bound[0], name, "y")
        check(grads[0], want[1], bound[1], name, "dx")
        check(grads[1], want[2], bound[2], name, "dweight")
        if bias:
            check(grads[2], want[3], bound[3], name, "dbias")
        plain = ct.layernorm_rows(x, EPS, w, b, rd_mean=rd_mean)
        assert torch.equal(plain, y)                     # with and without autograd: the same bits


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n", [1, 8, 129, 4096, 20001])
def test_constant_rows(n, name):
    """The deviations of a constant row are zero: y is the bias, and with eps = 0 still no matter of the mean's size (0 / 0 is NaN)."""
    t = TYPES[name]
    x = torch.full((3, n), 2.0, device="cuda").to(t)
    w, b = torch.ones(n, device="cuda").to(t), torch.full((n,), 0.5, device="cuda").to(t)
    assert torch.equal(ct.layernorm_rows(x, EPS, w, b), b.expand(3, n))
    assert torch.equal(ct.layernorm_rows(torch.zeros_like(x), EPS, w, b, rd_mean=False), b.expand(3, n))


@pytest.mark.parametrize("name", TYPES)
def test_a_large_mean_does_not_drown_the_deviations(name):
    """Mean 64 times the spread: the deviations are taken before they are squared."""
    x, w, b, dy = make(40, 2048, TYPES[name], 3, offset=96.0)
    want, bound = exact(x, w, b, dy, EPS, True)
    check(ct.layernorm_rows(x, EPS, w, b), want[0], bound[0], name, "y")


@pytest.mark.parametrize("n", [40, 1024, 5001, 17000])
def test_values_that_are_not_numbers_stay_in_their_row(n):
    x, w, b, dy = make(6, n, torch.float16, 1)
    clean = ct.layernorm_rows(x, EPS, w, b)
    x[2, n // 2] = float("nan")
    x[4, 0] = float("inf")
    y = ct.layernorm_rows(x, EPS, w, b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).any()
    for r in (0, 1, 3, 5):
        assert torch.equal(y[r], clean[r])


def test_no_rows():
    w = torch.ones(16, device="cuda", dtype=torch.half, requires_grad=True)
    b = torch.ones(16, device="cuda", dtype=torch.half, requires_grad=True)
    x = torch.empty((0, 16), device="cuda", dtype=torch.half, requires_grad=True)
    y = ct.layernorm_rows(x, EPS, w, b)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()


def test_leading_axes_views_and_expanded_gradients():
    g = torch.Generator(device="cuda").manual_seed(9)
    big = torch.randn((4, 7, 25, 48), generator=g, device="cuda").half()
    w = torch.randn(48, generator=g, device="cuda").half().requires_grad_()
    x = big[1].requires_grad_()                           # contiguous, an offset into a larger tensor
    y = ct.layernorm_rows(x, EPS, w, rd_mean=False)
    assert y.shape == (7, 25, 48)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))         # an expanded output gradient
    ones = torch.ones_like(y)
    dx2, dw2 = torch.autograd.grad(ct.layernorm_rows(x, EPS, w, rd_mean=False), (x, w), ones)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,n,shift", [(9, 64, 1), (5, 1000, 3), (4, 4096, 1), (3, 129, 1)])
def test_pointers_that_are_not_aligned_to_16_bytes(rows, n, shift, name):
    x, w, b, dy = make(rows, n, TYPES[name], 5)

    def moved(t):
        out = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:].view(t.shape)
        return out.copy_(t)

    leaves = [moved(t).requires_grad_() for t in (x, w, b)]
    y = ct.layernorm_rows(leaves[0], EPS, leaves[1], leaves[2])
    grads = torch.autograd.grad(y, leaves, moved(dy))
    want, bound = exact(x, w, b, dy, EPS, True)
    for got, v, e, what in zip((y, *grads), want, bound, ("y", "dx", "dweight", "dbias")):
        check(got, v, e, name, what)


def test_some_gradients_only():
    x, w, b, dy = make(37, 520, torch.bfloat16, 2)
    everything = None
    for mask in (7, 1, 2, 4, 3, 6, 5):
        ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        y = ct.layernorm_rows(ts[0], EPS, ts[1], ts[2])
        got = torch.autograd.grad(y, [t for t in ts if t.requires_grad], dy)
        if mask == 7:
            everything = got
        for i, v in zip([i for i in range(3) if mask >> i & 1], got):
            assert torch.equal(v, everything[i])


@pytest.mark.parametrize("rows,n", [(5, 33), (6, 1024), (300, 4096), (3, 17000)])
def test_nothing_is_written_outside_the_outputs(rows, n):
    x, w, b, dy = make(rows, n, torch.half, 4)
    s = torch.cuda.current_stream().cuda_stream
    pad = 64
    y = torch.full((rows * n + 2 * pad,), 7.0, dtype=torch.half, device="cuda")
    dx, dw, db = y.clone(), torch.full((n + 2 * pad,), 7.0, dtype=torch.half, device="cuda"), torch.full((n + 2 * pad,), 7.0, dtype=torch.half, device="cuda")
    stats = torch.full((2, rows + 2 * pad), 7.0, device="cuda")
    need = ck.layernorm_rows_backward_scratch(rows, n)
    scratch = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
    at = lambda t: t.data_ptr() + pad * t.element_size()
    ck.layernorm_rows_forward(rows, n, cpmk.F16, x.data_ptr(), EPS, True, w.data_ptr(), b.data_ptr(), at(y), at(stats[0]), at(stats[1]), s)
    ck.layernorm_rows_backward(rows, n, cpmk.F16, dy.data_ptr(), x.data_ptr(), True, w.data_ptr(), at(stats[0]), at(stats[1]), at(dx), at(dw), at(db),
                               scratch.data_ptr(), s)
    for t in (y, dx, dw, db, stats[0], stats[1]):
        assert (t[:pad] == 7).all() and (t[-pad:] == 7).all()
    assert (scratch[need:] == 77).all()
    want, bound = exact(x, w, b, dy, EPS, True)
    for got, v, e, what in zip((y[pad:-pad].view(rows, n), dx[pad:-pad].view(rows, n), dw[pad:-pad], db[pad:-pad]), want, bound, "yxwb"):
        check(got, v, e, "fp16", what)


def test_offsets_beyond_32_bits():
    """2.2e9 elements per tensor: the rows at both ends and around the 2^31st element against the same rows on their own."""
    rows, n = 1_050_000, 2056
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dy = torch.empty_like(x).normal_(generator=g)
    w = torch.ones(n, dtype=torch.bfloat16, device="cuda") * 1.5
    x.requires_grad_()
    y = ct.layernorm_rows(x, EPS, w)
    (dx,) = torch.autograd.grad(y, x, dy)
    middle = 2 ** 31 // n
    for at in (0, middle - 2, rows - 4):
        part = x.detach()[at:at + 4].clone().requires_grad_()
        z = ct.layernorm_rows(part, EPS, w)
        assert torch.equal(z, y[at:at + 4])
        assert torch.equal(torch.autograd.grad(z, part, dy[at:at + 4].clone())[0], dx[at:at + 4])


def test_same_bits_on_every_run_and_stream():
    x, w, b, dy = make(3000, 1024, torch.bfloat16, 8)
    results = []
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ts = [t.clone().requires_grad_() for t in (x, w, b)]
            y = ct.layernorm_rows(ts[0], EPS, ts[1], ts[2])
            results.append((y.detach(), *torch.autograd.grad(y, ts, dy)))
    torch.cuda.synchronize()
    for r in results[1:]:
        assert all(torch.equal(p, q) for p, q in zip(results[0], r))


def test_captured_and_replayed_on_new_values():
    x, w, b, dy = make(130, 1024, torch.half, 6)
    ts = [t.clone().requires_grad_() for t in (x, w, b)]
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, ts, dy)))(ct.layernorm_rows(ts[0], EPS, ts[1], ts[2]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    other = make(130, 1024, torch.half, 60)[0]
    with torch.no_grad():
        ts[0].copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    again = step()
    assert all(torch.equal(p, q) for p, q in zip(captured, again))


def test_refusals():
    w = torch.ones(16, device="cuda", dtype=torch.half)
    x = torch.ones((4, 16), device="cuda", dtype=torch.half)
    for bad in (lambda: ct.layernorm_rows(x.t().contiguous().t(), EPS, w), lambda: ct.layernorm_rows(x.double(), EPS, w.double()),
                lambda: ct.layernorm_rows(x, EPS, w.float()), lambda: ct.layernorm_rows(x, EPS, w[:8]), lambda: ct.layernorm_rows(x, -1.0, w),
                lambda: ct.layernorm_rows(x, float("nan"), w), lambda: ct.layernorm_rows(x, EPS, w, w[::2]), lambda: ct.layernorm_rows(x.cpu(), EPS, w),
                lambda: ct.layernorm_rows(torch.empty((4, 0), device="cuda", dtype=torch.half), EPS, w[:0])):
        with pytest.raises(AssertionError):
            bad()
    s = torch.cuda.current_stream().cuda_stream
    for args in ((4, 16, 9, x.data_ptr(), EPS, True, w.data_ptr(), 0, x.data_ptr(), 0, 0, s), (4, 16, 0, 0, EPS, True, w.data_ptr(), 0, x.data_ptr(), 0, 0, s),
                 (4, 16, 0, x.data_ptr() + 1, EPS, True, w.data_ptr(), 0, x.data_ptr(), 0, 0, s),
                 (4, 16, 0, x.data_ptr(), EPS, True, w.data_ptr(), 0, x.data_ptr(), x.data_ptr(), 0, s),
                 (1, 2 ** 30 + 8, 0, x.data_ptr(), EPS, True, w.data_ptr(), 0, x.data_ptr(), 0, 0, s)):
        with pytest.raises(RuntimeError):
            ck.layernorm_rows_forward(*args)
    y = ct.layernorm_rows(x.requires_grad_(), EPS, w)
    with pytest.raises(RuntimeError):                     # differentiable once
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
        dx.sum().backward()


def test_gradients_against_differences():
    """Central differences of the 64-bit loss <y(x), dy>, y computed by the kernel in fp32: step 2^-6, the third derivative of a layer
    norm of unit spread is O(1), so the truncation is O(2^-12); the fp32 rounding of y divided by the step adds n 2^-24 2^6."""
    x, w, b, dy = make(3, 24, torch.float32, 12)
    ts = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ct.layernorm_rows(ts[0], EPS, ts[1], ts[2]), ts, dy)
    loss = lambda a, c, d: (ct.layernorm_rows(a, EPS, c, d).double() * dy.double()).sum().item()
    h = 2.0 ** -6
    for i, g in enumerate(grads):
        for j in range(0, g.numel(), 5):
            args = [t.clone() for t in (x, w, b)]
            args[i].view(-1)[j] += h
            up = loss(*args)
            args[i].view(-1)[j] -= 2 * h
            assert abs((up - loss(*args)) / (2 * h) - g.view(-1)[j].item()) <= 2.0 ** -8


@pytest.mark.parametrize("name", ["fp16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1300, 4099), (700, 1031), (9, 5001), (300, 12289), (200, 16365)])
def test_rows_that_share_a_vector_keep_to_themselves(rows, n, name):
    """Odd widths: a 16-byte vector holds the end of one row and the start of the next; a third of the rows is NaN or infinite.  Weight
    and bias at an odd address."""
    x, w, b, dy = make(rows, n, TYPES[name], 9)
    w, b = (torch.cat([t[:1], t])[1:] for t in (w, b))
    assert w.data_ptr() % 16 and x.data_ptr() % 16 == 0
    y = ct.layernorm_rows(x, EPS, w, b)
    want, bound = exact(x, w, b, dy, EPS, True)
    check(y, want[0], bound[0], name, "y")
    bad = x.clone()
    bad[1::3] = float("nan")
    bad[4::9] = float("inf")
    z = ct.layernorm_rows(bad, EPS, w, b)
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[1::3] = False
    assert torch.equal(z[keep], y[keep])
    assert torch.isnan(z[~keep]).all()


@pytest.mark.parametrize("name", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,n", [(1300, 4099), (90, 20000), (50, 33001), (9, 66000)])
def test_long_and_odd_rows_write_their_outputs_only(rows, n, name):
    t, code = TYPES[name], cpmk.F16 if name == "fp16" else cpmk.F32
    x, w, b, dy = make(rows, n, t, 6)
    s = torch.cuda.current_stream().cuda_stream
    pad = 64
    y = torch.full((rows * n + 2 * pad,), 7.0, dtype=t, device="cuda")
    dx, dw, db = y.clone(), torch.full((n + 2 * pad,), 7.0, dtype=t, device="cuda"), torch.full((n + 2 * pad,), 7.0, dtype=t, device="cuda")
    stats = torch.empty((2, rows), device="cuda")
    need = ck.layernorm_rows_backward_scratch(rows, n)
    scratch = torch.full((need + 256,), 77, dtype=torch.uint8, device="cuda")
    at = lambda v: v.data_ptr() + pad * v.element_size()
    ck.layernorm_rows_forward(rows, n, code, x.data_ptr(), EPS, True, w.data_ptr(), b.data_ptr(), at(y), stats[0].data_ptr(), stats[1].data_ptr(), s)
    ck.layernorm_rows_backward(rows, n, code, dy.data_ptr(), x.data_ptr(), True, w.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), at(dx), at(dw),
                               at(db), scratch.data_ptr(), s)
    for v in (y, dx, dw, db):
        assert (v[:pad] == 7).all() and (v[-pad:] == 7).all()
    assert (scratch[need:] == 77).all()
    want, bound = exact(x, w, b, dy, EPS, True)
    for got, v, e, what in zip((y[pad:-pad].view(rows, n), dx[pad:-pad].view(rows, n), dw[pad:-pad], db[pad:-pad]), want, bound, "yxwb"):
        check(got, v, e, name, what)


@pytest.mark.parametrize("n", [2051, 20000])
def test_offsets_beyond_32_bits_of_odd_and_long_rows(n):
    """2.2e9 elements per tensor, as above; the gradient is zero but in one row behind the 2^31st element, so that the sums over the rows
    are that row's."""
    rows = 2_200_000_000 // n
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dy = torch.zeros_like(x)
    dy[rows - 3].normal_(generator=g)
    w = (torch.ones(n, dtype=torch.bfloat16, device="cuda") * 1.5).requires_grad_()
    x.requires_grad_()
    y = ct.layernorm_rows(x, EPS, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    middle = 2 ** 31 // n
    for at in (0, middle - 4, rows - 3):
        at = at // 8 * 8                                 # rows 8 apart start at the same place of a vector: the same sums
        part = x.detach()[at:at + 8].clone().requires_grad_()
        z = ct.layernorm_rows(part, EPS, w)
        assert torch.equal(z, y[at:at + 8])
        ex, ew = torch.autograd.grad(z, (part, w), dy[at:at + 8].clone())
        assert torch.equal(ex, dx[at:at + 8])
        if at <= rows - 3 < at + 8:
            assert torch.equal(ew, dw)
