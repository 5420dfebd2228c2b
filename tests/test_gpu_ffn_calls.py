"""Calls of the row layer norm and the gated feed-forward block at the edges of what their documentation allows."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import cpm_kernels_b200.kernels as ck
import cpm_kernels_b200.torch as ct
from cpm_kernels_b200.library import cpmk

pytestmark = pytest.mark.gpu
OPERATORS = ["layernorm_rows", "gated_linear", "gated_feed_forward"]


def operands_of(name, tokens=6):
    """Small fp16 operands of an operator, and the call that takes them."""
    g = torch.Generator(device="cuda").manual_seed(21)
    r = lambda *s: (torch.randn(*s, generator=g, device="cuda") * 0.3).half()
    if name == "layernorm_rows":
        return [r(tokens, 64), 1 + r(64), r(64)], lambda x, w, b: ct.layernorm_rows(x, 1e-5, w, b)
    operands = [r(tokens, 64), r(72, 64), r(72, 64), r(40, 72)]
    return (operands[:3], ct.gated_linear) if name == "gated_linear" else (operands, ct.gated_feed_forward)


@pytest.mark.parametrize("which", ["k", "n", "m"])
def test_extents_beyond_32_bits_are_refused(which):
    """2^32 + 8 must not arrive as 8.  (Refused before anything of these tensors is read.)"""
    k, n, m = (2 ** 32 + 8 if which == w else 1 for w in "knm")
    x, w, w_down = (torch.empty(shape, device="cuda", dtype=torch.half) for shape in ((1, k), (n, k), (m, n)))
    with pytest.raises(AssertionError):
        ct.gated_feed_forward(x, w, w, w_down)
    if which != "m":
        with pytest.raises(AssertionError):
            ct.gated_linear(x, w, w)


@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode_differentiation_is_refused(name):
    """A tangent on any one operand: an error, not an output without a tangent."""
    operands, call = operands_of(name)
    want = call(*operands)
    for i in range(len(operands)):
        with forward_ad.dual_level():
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(operands)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            assert torch.equal(call(*operands), want)    # others are not concerned


@pytest.mark.parametrize("name", OPERATORS)
@pytest.mark.parametrize("dy_requires_grad", [False, True])
def test_a_gradient_is_not_differentiated_again(name, dy_requires_grad):
    """A penalty on a gradient raises, beside another loss too; it must not count as a constant."""
    operands, call = operands_of(name)
    operands = [t.requires_grad_() for t in operands]
    y = call(*operands)
    dy = torch.ones_like(y).requires_grad_(dy_requires_grad)
    plain = torch.autograd.grad(y, operands, dy.detach(), retain_graph=True)
    for i, (g, p) in enumerate(zip(torch.autograd.grad(y, operands, dy, create_graph=True), plain)):
        assert torch.equal(g, p)
        if name == "layernorm_rows" and i == 2 and not dy_requires_grad:
            assert not g.requires_grad                   # dbias is the sum of dy: a constant
            continue
        with pytest.raises(RuntimeError, match="differentiable once"):
            (y.sum() + g.square().sum()).backward(retain_graph=True)


@pytest.mark.parametrize("name", OPERATORS)
def test_gradients_of_some_operands_with_a_graph_of_them(name):
    """Only one operand requires a gradient: its gradient depends on itself, or on constants only (then it is one)."""
    constants = {"layernorm_rows": (1, 2), "gated_linear": (2,), "gated_feed_forward": (2, 3)}[name]
    for i in range(len(operands_of(name)[0])):
        operands, call = operands_of(name)
        y = call(*[t.requires_grad_(j == i) for j, t in enumerate(operands)])
        (g,) = torch.autograd.grad(y, operands[i], torch.ones_like(y), create_graph=True)
        assert g.requires_grad == (i not in constants)


def alike(n, t, kind):
    """Rows of values that are alike: constant ones, and constant ones but for a few values a step of their type away."""
    rows = []
    for c in (1000.0, 2.0, 0.1, -777.7, 1025.0, 3.0e-5):
        row = torch.full((n,), c, device="cuda", dtype=torch.float64).to(t)
        if kind == "steps":
            row[:: max(1, n // 3)] = (row[0].double() * (1 + torch.finfo(t).eps)).to(t)
        rows.append(row)
    return torch.stack(rows)


@pytest.mark.parametrize("kind", ["constant", "steps"])
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [3, 41, 47, 256, 511, 1000, 1024, 1032, 2047, 2560, 4095, 4096, 5000, 5001, 8191, 8192, 12289, 16384, 20000, 20001, 32768, 33001, 66000])
def test_rows_of_values_that_are_alike(n, t, kind):
    """The rounding of the mean must not show.  With K = (n / 32 + 18) 2^-24 the relative error of a sum (32 or more threads share it, a tree
    joins them) and o = K mean|x| r what the mean may be off by in units of the spread: what it is off by is known to K (1 + o), the spread
    to K (1 + o^2), and three more roundings of 2^-24 follow; then y is rounded once.  Without that o itself would be the error.  Many
    rows and few, so that all forms of the kernel are met; with and without a mean to take off; weight and bias."""
    x = alike(n, t, kind)
    g = torch.Generator(device="cuda").manual_seed(n)
    w, b = ((1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(t), torch.randn(n, generator=g, device="cuda").to(t))
    d = x.double()
    mean = d.mean(-1, keepdim=True)
    r = 1 / ((d - mean).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    xh, u = (d - mean) * r, 2.0 ** -24
    want = xh * w.double() + b.double()
    k = (n / 32 + 18) * u
    o = k * d.abs().mean(-1, keepdim=True) * r
    bound = w.double().abs() * (k * (1 + o) + (k * (1 + o * o) + 4 * u) * xh.abs() + 4 * u * o) + 2 * u * (want.abs() + (xh * w.double()).abs())
    tol = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + 2.0 ** -25
    for copies in (1, 250):
        many = x.repeat(copies, 1) if copies * n < 5_000_000 else x
        y = ct.layernorm_rows(many, 1e-5, w, b)
        off = (y.double().view(-1, *x.shape) - want).abs()
        assert (off <= tol).all(), "off by %.3g where %.3g is allowed" % (off.max(), tol.expand_as(off).flatten()[(off - tol).argmax()])


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [41, 1000, 4095, 5000, 12289, 20001, 33001])
def test_gradients_of_constant_rows(n, t):
    """xh = 0: dweight is zero, dx = r (g - mean g) with K as above for the sum of g."""
    x = alike(n, t, "constant").requires_grad_()
    g = torch.Generator(device="cuda").manual_seed(n)
    w = (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(t).requires_grad_()
    dy = torch.randn(x.shape, generator=g, device="cuda").to(t)
    dx, dw = torch.autograd.grad(ct.layernorm_rows(x, 1e-5, w), (x, w), dy)
    assert not dw.any()
    gw = dy.double() * w.detach().double()
    r, k = 1e-5 ** -0.5, (n / 32 + 18) * 2.0 ** -24
    want = r * (gw - gw.mean(-1, keepdim=True))
    bound = r * k * (gw.abs() + gw.abs().mean(-1, keepdim=True))
    assert ((dx.double() - want).abs() <= bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + 2.0 ** -25).all()


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("tokens,k,n,m", [(5, 64, 72, 40), (300, 64, 72, 40), (300, 64, 136, 4096), (700, 64, 512, 64), (7, 5, 3, 2)])
def test_gate_projections_beyond_the_range_of_fp16(tokens, k, n, m, act):
    """A gate projection of -120000 is kept as minus infinity.  The activation and its slope are zero there as they are at -60000, so
    the hidden activations and all gradients are those of a call whose projection is -60000; at +120000 the slope is 1 as at +60000."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    wg, wu, wd = ((r(n, k) / k ** 0.5).half(), (r(n, k) / k ** 0.5).half(), (r(m, n) / n ** 0.5).half())
    wg[:, 0] = -2.0
    wu[:, 0] = 2.0 ** -6
    dy, dh, x = r(tokens, m).half(), r(tokens, n).half(), r(tokens, k).half()
    x[1] = 0

    def step(size):
        inputs = x.clone()
        inputs[1, 0] = size
        ts = [t.clone().requires_grad_() for t in (inputs, wg, wu, wd)]
        y, h = ct.gated_feed_forward(*ts, activation=act), ct.gated_linear(*ts[:3], activation=act)
        return (y.detach(), h.detach(), *torch.autograd.grad(y, ts, dy), *torch.autograd.grad(h, ts[:3], dh))

    for got, want in zip(step(60000.0), step(30000.0)):
        assert torch.isfinite(want).all() and torch.equal(got, want)

    # g = 120000: dg = dh u (du is infinite), seen in the gradient of w_gate, dg^T x
    ts = [t.clone().requires_grad_() for t in (-60000.0 * torch.eye(1, k, device="cuda").half(), wg, wu * 2.0 ** -8)]
    (dwg,) = torch.autograd.grad(ct.gated_linear(*ts, activation=act), ts[1], dh[:1] * 2.0 ** -8)
    u = (ts[0].detach().double() @ ts[2].detach().double().T).half().double()
    dg = ((dh[:1] * 2.0 ** -8).double() * u).half().double()
    assert torch.equal(dwg.double(), (dg.T @ ts[0].detach().double()).half().double())


@pytest.mark.parametrize("tokens", [3, 300])
def test_hidden_activations_have_the_range_of_their_type(tokens):
    """act(g) u = 260 * 260 is beyond fp16 and infinite there, and not in bf16."""
    for t, infinite in ((torch.float16, True), (torch.bfloat16, False)):
        x = torch.ones((tokens, 8), device="cuda", dtype=t)
        w, w_down = torch.full((16, 8), 32.5, device="cuda", dtype=t), torch.full((8, 16), 2.0 ** -10, device="cuda", dtype=t)
        assert torch.isinf(ct.gated_linear(x, w, w)).all() == infinite
        y = ct.gated_feed_forward(x, w, w, w_down)
        assert torch.isinf(y).all() if infinite else (y - 260.0 * 260 * 16 / 1024).abs().max() <= 1056 * 2.0 ** -7


@pytest.mark.parametrize("rows,n", [(3000, 60000), (600, 20_000_000), (40, 100_000_000)])
def test_scratch_of_long_rows_stays_small(rows, n):
    """Partial sums for as many rows as fill the device with strips of columns, one at least: not one per block (24 GB at 600 x 20 million)."""
    assert ck.layernorm_rows_backward_scratch(rows, n) <= 8 * (n + 64) + 16 * 2 ** 20


@pytest.mark.parametrize("t,code", [(torch.float16, cpmk.F16), (torch.float32, cpmk.F32)])
@pytest.mark.parametrize("rows,n", [(700, 16400), (700, 33000), (300, 66004), (5, 9000), (400, 9000)])
def test_scratch_suffices_whatever_the_alignment(rows, n, t, code):
    """Each tensor at an odd address in turn, so that every layout meets the same scratch; nothing behind it is written."""
    g = torch.Generator(device="cuda").manual_seed(n)
    s, need = torch.cuda.current_stream().cuda_stream, ck.layernorm_rows_backward_scratch(rows, n)
    make = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(t)
    plain = {"dy": make(rows, n), "x": make(rows, n), "w": make(n), "dx": make(rows, n)}
    moved = {k: torch.empty(v.numel() + 1, device="cuda", dtype=t)[1:].view(v.shape).copy_(v) for k, v in plain.items()}
    mean, rstd = plain["x"].double().mean(-1), 1 / (plain["x"].double().var(-1, unbiased=False) + 1e-5).sqrt()
    stats = torch.stack([mean, rstd]).float()
    want = (plain["dy"].double() * (plain["x"].double() - mean[:, None]) * rstd[:, None]).sum(0)
    size = (plain["dy"].double() * (plain["x"].double() - mean[:, None]) * rstd[:, None]).abs().sum(0)
    for odd in ((), ("x",), ("dy",), ("x", "dy"), ("w",), ("dx",), ("x", "dy", "w", "dx")):
        at = {k: moved[k] if k in odd else plain[k] for k in plain}
        scratch = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
        dw, db = torch.empty(n, device="cuda", dtype=t), torch.empty(n, device="cuda", dtype=t)
        ck.layernorm_rows_backward(rows, n, code, at["dy"].data_ptr(), at["x"].data_ptr(), True, at["w"].data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
                                   at["dx"].data_ptr(), dw.data_ptr(), db.data_ptr(), scratch.data_ptr(), s)
        assert (scratch[need:] == 77).all()
        # at most rows + 8 roundings of 2^-24 of the sum of magnitudes, the statistics' among them, and that of the output
        assert ((dw.double() - want).abs() <= (rows + 8) * 2.0 ** -24 * size * 2 + torch.finfo(t).eps / 2 * want.abs() * 1.01 + 2.0 ** -25).all()


def test_the_same_bits_at_every_address_of_the_same_alignment():
    """The order of the sums depends on sizes, type, device and alignment: copies elsewhere, aligned alike, give the same bits."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for rows, n in ((700, 1000), (300, 4099), (90, 20000)):
        x, w, dy = (torch.randn(s, generator=g, device="cuda").half() for s in ((rows, n), (n,), (rows, n)))
        for odd in (0, 1):
            results = []
            for lead in (0, 8, 4096):
                moved = [torch.empty(t.numel() + lead + odd, device="cuda", dtype=t.dtype)[lead + odd:].view(t.shape).copy_(t) for t in (x, w, dy)]
                leaves = [t.requires_grad_() for t in moved[:2]]
                y = ct.layernorm_rows(leaves[0], 1e-5, leaves[1])
                results.append((y.detach(), *torch.autograd.grad(y, leaves, moved[2])))
            assert all(torch.equal(p, q) for r in results[1:] for p, q in zip(results[0], r))


def test_negated_views():
    """The imaginary part of a conjugate is read negated; where it counts as contiguous, operands are refused and an output gradient is
    taken as what it stands for."""
    lazy = torch.tensor([[1 + 2j]], device="cuda").conj().imag
    assert lazy.is_neg() and lazy.is_contiguous() and lazy.item() == -2
    w = torch.ones(1, device="cuda", requires_grad=True)
    x = torch.full((1, 1), 3.0, device="cuda", requires_grad=True)
    with pytest.raises(AssertionError):
        ct.layernorm_rows(lazy, 1e-5, w)
    with pytest.raises(AssertionError):
        ct.layernorm_rows(x, 1e-5, lazy[0])
    step = lambda dy: torch.autograd.grad(ct.layernorm_rows(x, 1e-5, w, w, rd_mean=False), (x, w), dy)
    for got, want in zip(step(lazy), step(torch.full((1, 1), -2.0, device="cuda"))):
        assert torch.equal(got, want)
