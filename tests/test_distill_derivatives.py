"""Derivatives that the distillation loss does not have are refused, never left out: forward mode, second ones."""

import pytest
import torch
from torch.autograd import forward_ad

from mlxturbo_b200 import ops


def arguments(device):
    g = torch.Generator().manual_seed(1)
    x = torch.randn((4, 600), generator=g).to(device)
    tv, ti = torch.randn((4, 600), generator=g).to(device).topk(5, dim=-1)
    return x, tv, ti, torch.logsumexp(tv, -1) + 0.1


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode(device):
    x, tv, ti, lse = arguments(device)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda l: ops.distill_loss(l, tv, ti), (x,), (torch.ones_like(x),))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda l: ops.distill_loss_and_grad(l, tv, ti)[0], (x,), (torch.ones_like(x),))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.distill_loss(dual(x), tv, ti), lambda: ops.distill_loss(x, dual(tv), ti),
                     lambda: ops.distill_loss(x, tv, ti, teacher_logsumexp=dual(lse)),
                     lambda: ops.distill_loss(dual(x.clone().requires_grad_()), tv, ti),
                     lambda: ops.distill_loss_and_grad(dual(x), tv, ti),
                     lambda: ops.distill_loss_and_grad(x, tv, ti, dual(lse))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        if device == "cuda":  # without a tangent nothing is refused
            assert ops.distill_loss(x, tv, ti).shape == (4,)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [False, True])
def test_second_derivatives(tail):
    """A graph of the gradient may be asked for; what differentiates it again is told so."""
    x, tv, ti, lse = arguments("cuda")
    kw = dict(teacher_logsumexp=lse if tail else None)
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(ops.distill_loss(leaf, tv, ti, **kw).sum(), leaf)
    (grad,) = torch.autograd.grad(ops.distill_loss(leaf, tv, ti, **kw).sum(), leaf, create_graph=True)
    assert grad.requires_grad and torch.equal(grad.detach(), want)
    with pytest.raises(NotImplementedError, match="second derivative"):
        ((grad ** 2).sum() + (leaf ** 2).sum()).backward()
    # a graph for another term's sake
    (ops.distill_loss(leaf * 1.0, tv, ti, **kw).sum() + 0.0 * leaf.sum()).backward(create_graph=True)
    assert torch.equal(leaf.grad.detach(), want)
    leaf.grad = None
    with forward_ad.dual_level():  # forward over reverse
        loss = ops.distill_loss(leaf, tv, ti, **kw)
        with pytest.raises(NotImplementedError, match="second derivative"):
            torch.autograd.grad(loss, leaf, forward_ad.make_dual(torch.ones(4, device="cuda"), torch.ones(4, device="cuda")))
    with torch.no_grad():
        assert not ops.distill_loss(leaf, tv, ti, **kw).requires_grad
