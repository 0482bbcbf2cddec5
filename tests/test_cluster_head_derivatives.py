"""Cluster head: derivatives that it does not have are refused, not dropped (CPU
only: the launches are replaced by the formula in plain torch)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import flash_kmeans as fk
from flash_kmeans import cluster_head as ch


class _Formula:
    """Stands in for a call's launches: float64 on the CPU, cut off from autograd
    as results of kernels are."""

    def __init__(self, x, centroids, labels, scale, ignore_index, reduction, name):
        self.args = x.detach(), centroids.detach(), labels, scale, reduction
        self.none = reduction == "none"

    def _grads(self, grad_loss):
        x, c, y, scale, reduction = self.args
        with torch.enable_grad():
            x, c = x.clone().requires_grad_(), c.clone().requires_grad_()
            loss = torch.nn.functional.cross_entropy(scale * x @ c.T, y.long(), reduction=reduction)
            gx, gc = torch.autograd.grad(loss, (x, c), grad_loss)
        return loss.detach(), gx, gc

    def forward(self, keep):
        ones = torch.ones(self.args[2].shape if self.none else (), dtype=self.args[0].dtype)
        return self._grads(ones)[0], object() if keep else None

    def backward(self, kept, grad_loss, want_x, want_c):
        _, gx, gc = self._grads(grad_loss.detach())
        return gx if want_x else None, gc if want_c else None

    def loss_grad(self, grad_loss):
        return self._grads(torch.ones(()) if grad_loss is None else grad_loss)


@pytest.fixture(autouse=True)
def _no_launch(monkeypatch):
    monkeypatch.setattr(ch, "_Xent", _Formula)


def _case():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 8, generator=g, dtype=torch.float64)
    c = torch.randn(4, 8, generator=g, dtype=torch.float64)
    return x, c, torch.tensor([0, 3, 1, 2, 2, 0])


@pytest.mark.parametrize("fn", [fk.cluster_cross_entropy, fk.cluster_cross_entropy_grad])
@pytest.mark.parametrize("which", ["x", "centroids", "both"])
def test_forward_mode_is_refused(fn, which):
    """A dual tensor made from an ordinary one does not require grad."""
    x, c, y = _case()
    with fwAD.dual_level():
        xd = fwAD.make_dual(x, torch.ones_like(x)) if which != "centroids" else x
        cd = fwAD.make_dual(c, torch.ones_like(c)) if which != "x" else c
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(xd, cd, y)
        fn(x, c, y)     # no tangent: as outside


def test_forward_mode_through_torch_func_is_refused():
    x, c, y = _case()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda a: fk.cluster_cross_entropy(a, c, y), (x,), (torch.ones_like(x),))


def test_forward_mode_of_the_upstream_gradient_is_refused():
    x, c, y = _case()
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones(()), torch.ones(()))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fk.cluster_cross_entropy_grad(x, c, y, grad_loss=g)
