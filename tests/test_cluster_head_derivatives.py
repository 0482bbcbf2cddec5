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


# ------------------------------------------------------------- second order
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("which", ["x", "centroids", "both"])
def test_a_penalty_on_the_gradient_is_refused(which, reduction):
    """The loss has a graph of its own, so dropping the penalty's would not show."""
    x, c, y = _case()
    x.requires_grad_(which != "centroids")
    c.requires_grad_(which != "x")
    of = [t for t in (x, c) if t.requires_grad]
    loss = fk.cluster_cross_entropy(x, c, y, reduction=reduction).sum()
    grads = torch.autograd.grad(loss, of, create_graph=True)
    total = loss + sum(g.square().sum() for g in grads)
    with pytest.raises(RuntimeError, match="differentiable once"):
        total.backward()
    for g in grads:     # and each of them alone
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), of, allow_unused=True, retain_graph=True)


def test_a_second_derivative_by_the_upstream_gradient_is_refused():
    x, c, y = _case()
    x.requires_grad_()
    w = torch.ones((), dtype=torch.float64, requires_grad=True)
    g, = torch.autograd.grad(w * fk.cluster_cross_entropy(x, c, y), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), w)


def test_gradients_with_a_graph_can_still_be_used_as_values():
    x, c, y = _case()
    x.requires_grad_()
    c.requires_grad_()
    loss = fk.cluster_cross_entropy(x, c, y)
    gx, gc = torch.autograd.grad(loss, (x, c), create_graph=True)
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(x @ c.T, y), (x, c))
    assert torch.allclose(gx, want[0]) and torch.allclose(gc, want[1])
    (loss * gx.detach().norm()).backward()      # a weight that is taken as a constant
    assert torch.allclose(x.grad, want[0] * want[0].norm())
    # a plain backward pass gives gradients without a graph
    x.grad = None
    fk.cluster_cross_entropy(x, c, y).backward()
    assert not x.grad.requires_grad


# ---------------------------------------------------------- scale and ignore_index
@pytest.mark.parametrize("fn", [fk.cluster_cross_entropy, fk.cluster_cross_entropy_grad])
def test_a_learnable_scale_is_refused(fn):
    """Its gradient would be dropped: a temperature multiplies x."""
    x, c, y = _case()
    for s in (torch.tensor(2.0, requires_grad=True), torch.nn.Parameter(torch.ones(1))):
        with pytest.raises(TypeError, match="scale"):
            fn(x, c, y, scale=s)
        with pytest.raises(TypeError, match="scale"):
            fn(x.requires_grad_(), c, y, scale=s)
        x = x.detach()
    with fwAD.dual_level(), pytest.raises(TypeError, match="scale"):
        fn(x, c, y, scale=fwAD.make_dual(torch.tensor(2.0), torch.tensor(1.0)))


# ---------------------------------------------------------------- mixed precision
@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
def test_autocast_takes_16_bit_points_with_float32_centroids(low, monkeypatch):
    """Activations of an autocast layer against a head kept in float32."""
    seen = []

    class Seen(_Formula):
        def __init__(self, x, centroids, *rest):
            seen.append((x.dtype, centroids.dtype))
            if x.dtype != centroids.dtype:
                raise TypeError("refused")
            super().__init__(x, centroids, *rest)

    monkeypatch.setattr(ch, "_Xent", Seen)
    x, c, y = _case()
    x, c = x.to(low).requires_grad_(), c.float().requires_grad_()
    # (torch.autocast("cuda") turns itself off where there is no GPU)
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: device == "cuda")
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: low)
    loss = fk.cluster_cross_entropy(x, c, y)
    assert seen[-1] == (low, low)
    with torch.no_grad():
        fk.cluster_cross_entropy(x, c, y)
    assert seen[-1] == (low, low)
    fk.cluster_cross_entropy(c.detach(), c, torch.tensor([0, 1, 2, 3]))
    assert seen[-1] == (torch.float32, torch.float32)      # equal types stay
    with pytest.raises(TypeError):                         # no type of the head's
        fk.cluster_cross_entropy(x.detach().double(), c, y)
    with pytest.raises(TypeError):                         # its gradients have their inputs' types
        fk.cluster_cross_entropy_grad(x, c, y)
    loss.backward()
    assert x.grad.dtype == low and c.grad.dtype == torch.float32
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(x @ c.to(low).T, y), (x, c))
    assert torch.equal(x.grad, want[0]) and torch.equal(c.grad, want[1])
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: False)
    with pytest.raises(TypeError):                             # outside of autocast
        fk.cluster_cross_entropy(x, c, y)
