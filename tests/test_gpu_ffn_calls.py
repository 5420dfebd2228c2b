"""Calls of the row layer norm and the gated feed-forward block at the edges of what their documentation allows."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import cpm_kernels_b200.torch as ct

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
