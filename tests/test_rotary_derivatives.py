"""What apply_rotary does with derivatives that it does not compute: it says so (the attention calls, Python autograd
functions without a forward-mode rule, raise in the same place)."""
import pytest
import torch

import pallas_flexattn as pf
from torch.autograd import forward_ad


@pytest.mark.parametrize("which", ["query", "key", "key alone", "inv_freq"])
def test_forward_mode_is_refused(which):
    """A dual tensor does not require grad: without a check its tangent would be dropped.  (The device is looked at last,
    so CPU tensors reach the check.)"""
    rot = pf.rotary_embedding(32, device="cpu")
    q, k = torch.ones(1, 2, 3, 64), torch.ones(1, 1, 3, 64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        if which == "query":
            q = dual(q)
        elif which == "inv_freq":
            rot = rot._replace(inv_freq=dual(rot.inv_freq))
        else:
            k = dual(k)
        if which == "key alone":
            q, k = k, None
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pf.apply_rotary(q, k, rot)


@pytest.mark.gpu
@pytest.mark.parametrize("create_graph", [False, True])
def test_forward_mode_over_the_gradient_is_refused(create_graph):
    rot = pf.rotary_embedding(32)
    q = torch.randn(1, 2, 3, 64, device="cuda", requires_grad=True)
    y = pf.apply_rotary(q, None, rot)
    g = torch.randn_like(y)
    want, = torch.autograd.grad(y, q, g, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, q, forward_ad.make_dual(g, torch.ones_like(g)), retain_graph=True, create_graph=create_graph)
        # (an ordinary gradient inside a dual level is one)
        assert torch.equal(torch.autograd.grad(y, q, g, retain_graph=True, create_graph=create_graph)[0], want)


def test_frequencies_that_require_grad_are_refused():
    """They would get no gradient.  (Without grad mode, or detached, they are numbers like any other: the next check, of the
    device, is reached.)"""
    rot = pf.rotary_embedding(32, device="cpu")
    rot.inv_freq.requires_grad_()
    q = torch.ones(1, 2, 3, 64)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(NotImplementedError, match="inv_freq"):
            pf.apply_rotary(x, None, rot)
        with pytest.raises(ValueError, match="GPU"):
            pf.apply_rotary(x, None, rot._replace(inv_freq=rot.inv_freq.detach()))
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        pf.apply_rotary(q, None, rot)
