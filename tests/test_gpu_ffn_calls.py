"""Calls of the row layer norm and the gated feed-forward block at the edges of what their documentation allows."""
import pytest
import torch

import cpm_kernels_b200.torch as ct

pytestmark = pytest.mark.gpu


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
