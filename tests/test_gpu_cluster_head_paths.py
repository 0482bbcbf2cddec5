"""Cluster head on the GPU: paths that the sizes, types and weights of a call choose."""
import pytest
import torch

import flash_kmeans as fk
from test_gpu_cluster_head import BF, FP, HF, close, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("N,K,D", [(40000, 3000, 600), (70001, 1000, 1000)])
@pytest.mark.parametrize("live", ["most", "few", "ends", "one segment"])
def test_rows_gathered_in_the_backward_pass_alone(live, N, K, D, dtype):
    """Few centroids: the loss reads x in place, its gradients gather the rows that
    count, past the rows whose labels one block counts by itself."""
    x, c, y = make(0, N, K, D, dtype, seed=41, ids=torch.int64)
    g = torch.Generator(device="cuda").manual_seed(42)
    keep = torch.zeros(N, dtype=torch.bool, device="cuda")
    if live == "most":
        keep = torch.rand(N, device="cuda", generator=g) < 0.7
    elif live == "few":
        keep[torch.randint(0, N, (41,), device="cuda", generator=g)] = True
    elif live == "ends":
        keep[[0, -1]] = True
    else:
        keep[1024 * 3: 1024 * 4] = True
    y = torch.stack([torch.where(keep, y, -100), y], 1)[:, 0]       # (every other word)
    x[~keep] = float("nan")
    reduction = "sum" if dtype == HF else "mean"
    want = reference(x[keep], c, y[keep], 4.0, reduction)
    got = fk.cluster_cross_entropy_grad(x, c, y, scale=4.0, reduction=reduction)
    xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
    loss = fk.cluster_cross_entropy(xr, cr, y, scale=4.0, reduction=reduction)
    loss.backward()
    for l, gx, gc in (got, (loss, xr.grad, cr.grad)):
        assert gx[~keep].eq(0).all()
        for a, w, what in zip((l, gx[keep], gc), want, ("loss", "gx", "gc")):
            close(a, w, what)
    rows = fk.cluster_cross_entropy(x, c, y, scale=4.0, reduction="none")
    assert rows[~keep].eq(0).all()
    close(rows[keep], reference(x[keep], c, y[keep], 4.0, "none")[0], "rows")


def _row_gradients(x, c, y, scale, g):
    """Gradients of float16 row losses in float64, with bounds that follow each row's
    own weight.  P = w (softmax - one-hot) / 2^e with 1 <= |w| / 2^e < 2 is held in float16 times
    2^14: half a step, or half the smallest subnormal (2^-25, hence 2^-39 |w| of the
    gradient).  x in the centroids' gradient is held in float16 relative to the
    largest |w| |x| of all rows, which lies between 2^14 and 2^16 there: off by
    half the smallest subnormal, 2^-39 of that largest, times the softmax's 2."""
    xd, cd, w = x.double(), c.double(), g.double()[:, None]
    z = scale * xd @ cd.T
    p = torch.softmax(z, -1)
    own = torch.arange(len(y), device="cuda")
    # 1 - p at the label as the sum of the others: exact where it is small
    others = p.scatter(-1, y.long()[:, None], 0.0).sum(-1)
    p[own, y.long()] = -others
    ez = (scale * (xd.abs() @ cd.abs().T) * 2.0 ** -21).amax(-1, keepdim=True) + z.abs().amax(-1, keepdim=True) * 2.0 ** -22
    off = p.abs() * (2 * ez + 2.0 ** -18 + 2.0 ** -11) + 2.0 ** -39
    gx, gxt = scale * w * (p @ cd), scale * w.abs() * ((off + 2.0 ** -20 * p.abs()) @ cd.abs())
    top = (w.abs() * xd.abs().amax(-1, keepdim=True)).max()
    gc = scale * (p * w).T @ xd
    gct = scale * ((off + 2.0 ** -20 * p.abs()) * w.abs()).T @ xd.abs() + scale * 2.0 ** -38 * top * p.abs().sum(0)[:, None]
    step = lambda t: t.abs() * 2.0 ** -11 + 2.0 ** -25      # noqa: E731 (the outputs' own rounding)
    return (gx, gxt + step(gx)), (gc, gct + step(gc))


@pytest.mark.parametrize("N,K,D,ignored", [(64, 40000, 64, 0.0), (300, 131072, 24, 0.3), (1100, 60000, 1200, 0.2),
                                           (65, 3, 8, 0.0)])
@pytest.mark.parametrize("span", [20, 30])
def test_float16_rows_of_small_weight_keep_their_softmax(N, K, D, ignored, span):
    """One upstream gradient a row, over `span` powers of two; flat softmaxes of many
    centroids, whose entries are small against the label's."""
    gen = torch.Generator(device="cuda").manual_seed(43)
    c = (torch.randn(K, D, device="cuda", generator=gen) * 0.1 + 0.3).half()
    x = (torch.randn(N, D, device="cuda", generator=gen) * 0.02).half()
    y = torch.randint(0, K, (N,), device="cuda", generator=gen)
    g = torch.exp2(12.0 - span * torch.linspace(0, 1, N, device="cuda")) * (1 + torch.rand(N, device="cuda", generator=gen))
    g[1::3] *= -1
    keep = torch.rand(N, device="cuda", generator=gen) >= ignored
    keep[[0, -1]] = True
    y = y.masked_fill(~keep, -100)
    g[~keep] = 3e38                          # (an ignored row's counts for nothing)
    x[~keep] = float("nan")
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=0.5, reduction="none", grad_loss=g)
    wx, wc = _row_gradients(x[keep], c, y[keep], 0.5, g[keep])
    close(gx[keep], wx, "gx")
    assert gx[~keep].eq(0).all()
    close(gc, wc, "gc")
    xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
    fk.cluster_cross_entropy(xr, cr, y, scale=0.5, reduction="none").backward(g)
    close(xr.grad[keep], wx, "gx of autograd")
    close(cr.grad, wc, "gc of autograd")
    for t in (x, c):                         # one alone
        a = t.clone().requires_grad_()
        fk.cluster_cross_entropy(a if t is x else x, a if t is c else c, y, scale=0.5, reduction="none").backward(g)
        close(a.grad[keep] if t is x else a.grad, wx if t is x else wc, "alone")


def test_float16_row_weights_of_every_kind():
    """Zero, infinite and NaN upstream gradients, the largest and the smallest."""
    gen = torch.Generator(device="cuda").manual_seed(44)
    c = torch.randn(90, 40, device="cuda", generator=gen).half()
    x = torch.randn(2, 50, 40, device="cuda", generator=gen).half()
    y = torch.randint(0, 90, (2, 50), device="cuda", generator=gen)
    zero = torch.zeros(2, 50, device="cuda")
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c.expand(2, 90, 40), y, reduction="none", grad_loss=zero)
    assert gx.eq(0).all() and gc.eq(0).all()
    for big, tiny in ((1.0, 1e-45), (2.0 ** 127, 2.0 ** -126), (1e-30, 1e-40)):
        g = zero.clone()
        g[0, 3], g[1, 7] = big, tiny
        _, gx, gc = fk.cluster_cross_entropy_grad(x, c.expand(2, 90, 40), y, scale=1 / big, reduction="none",
                                                  grad_loss=g)
        _, ex, ec = fk.cluster_cross_entropy_grad(x, c.expand(2, 90, 40), y, scale=1 / big, reduction="none",
                                                  grad_loss=torch.where(g == tiny, 0.0, g))
        assert torch.isfinite(gx).all() and torch.isfinite(gc).all()
        assert gx[0, 3].abs().sum() > 0 and torch.equal(gx, ex)      # (the tiny one's underflows)
        assert torch.equal(gc, ec)
    for bad in (float("inf"), float("nan")):
        g = torch.ones(2, 50, device="cuda")
        g[1, 9] = bad
        _, gx, gc = fk.cluster_cross_entropy_grad(x, c.expand(2, 90, 40), y, reduction="none", grad_loss=g)
        _, ex, ec = fk.cluster_cross_entropy_grad(x, c.expand(2, 90, 40), y, reduction="none",
                                                  grad_loss=torch.ones_like(g))
        keep = torch.ones(2, 50, dtype=torch.bool, device="cuda")
        keep[1, 9] = False
        assert not torch.isfinite(gx[1, 9]).any() and torch.equal(gx[keep], ex[keep])
        assert not torch.isfinite(gc[1]).all() and torch.equal(gc[0], ec[0])


def test_float16_rows_of_no_weight_beside_small_ones():
    """Rows of weight 0 take no part in the scale of the others', however large they are."""
    gen = torch.Generator(device="cuda").manual_seed(45)
    c = torch.randn(500, 72, device="cuda", generator=gen).half()
    x = torch.randn(400, 72, device="cuda", generator=gen).half()
    y = torch.randint(0, 500, (400,), device="cuda", generator=gen, dtype=torch.int32)
    g = torch.full((400,), 2.0 ** -40, device="cuda")
    g[::2] = 0.0
    x[::2] *= 1000.0
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0 ** 20, reduction="none", grad_loss=g)
    one = torch.ones_like(g)
    _, ex, ec = fk.cluster_cross_entropy_grad(x[1::2], c, y[1::2], scale=2.0 ** 20, reduction="none",
                                              grad_loss=one[1::2] * 2.0 ** -40)
    assert gx[::2].eq(0).all() and torch.isfinite(gx).all() and torch.isfinite(gc).all()
    assert gx[1::2].abs().max() > 0 and gc.abs().max() > 0
    # the same sums of the same values; a scale this large makes softmaxes one-hot
    assert torch.equal(gx[1::2], ex) and torch.equal(gc, ec)


@pytest.mark.parametrize("low", [BF, HF], ids=["bf16", "fp16"])
def test_autocast_step(low):
    """A linear layer under autocast in front of a head kept in float32."""
    x, c, y = make(0, 200, 300, 64, FP, seed=46, ignored=0.1)
    lin = torch.nn.Linear(64, 64, device="cuda")
    head = c.clone().requires_grad_()
    with torch.autocast("cuda", dtype=low):
        h = lin(x)
        assert h.dtype == low
        h.retain_grad()
        loss = fk.cluster_cross_entropy(h, head, y, scale=3.0, reduction="sum")
    loss.backward()
    want = reference(h, head.to(low), y, 3.0, "sum")
    close(loss, want[0], "loss")
    close(h.grad, want[1], "h")
    assert head.grad.dtype == FP and lin.weight.grad is not None
    close(head.grad, want[2], "head")


def test_negated_views():
    x, c, y = make(0, 100, 200, 48, FP, seed=47)
    g = torch.rand(100, device="cuda")
    want = fk.cluster_cross_entropy_grad(x, c, y, reduction="none", grad_loss=g)
    neg = lambda t: torch._neg_view(t.neg())        # noqa: E731
    got = fk.cluster_cross_entropy_grad(neg(x), neg(c), y, reduction="none", grad_loss=neg(g))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xr = neg(x).requires_grad_()
    fk.cluster_cross_entropy(xr, c, y, reduction="none").backward(neg(g))
    assert torch.equal(xr.grad, want[1])
    # as one arises: the imaginary part of a conjugate
    z = torch.complex(x, x)
    assert torch.equal(fk.cluster_cross_entropy(z.conj().imag, c, y), fk.cluster_cross_entropy(-x, c, y))
    cq, cs = fk.quantize_rows(c)
    assert torch.equal(fk.int8_scores(neg(x), cq, neg(cs)), fk.int8_scores(x, cq, cs))
    assert all(torch.equal(a, b) for a, b in zip(fk.quantize_rows(neg(x)), fk.quantize_rows(x)))


def test_a_recorded_backward_pass():
    """Gradients with a graph are the same values; their derivative raises."""
    x, c, y = make(0, 300, 400, 64, BF, seed=48, ignored=0.1)
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0)
    xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
    loss = fk.cluster_cross_entropy(xr, cr, y, scale=2.0)
    got = torch.autograd.grad(loss, (xr, cr), create_graph=True)
    assert torch.equal(got[0], gx) and torch.equal(got[1], gc)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (loss + got[0].float().square().sum()).backward()


def _near_ties(N, K, D, seed, B=1, batched=False):
    """One direction for all centroids, scales and biases a few steps of float32 apart:
    most rows' best scores are equal or neighbours once they are rounded as documented."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    xq = torch.randint(-127, 128, (B, N, D), device="cuda", generator=g).to(torch.int8)
    c = torch.randint(-127, 128, (B, 1, D), device="cuda", generator=g).to(torch.int8).repeat(1, K, 1)
    xs = torch.rand(B, N, device="cuda", generator=g) * 0.02 + 1e-3
    cs = 0.01 * (1 + torch.randint(-4, 5, (B, K), device="cuda", generator=g) * 2.0 ** -23)
    size = (xq.double() @ c.double().transpose(-1, -2)).abs().mean() * xs.double().mean() * 0.01
    b = size.float() * (1 + torch.randint(-2, 3, (B, K), device="cuda", generator=g) * 2.0 ** -23)
    out = xq, c, xs, cs, b
    return out if batched else [t[0] for t in out]


def _first_of_the_largest(z):
    k = torch.arange(z.shape[-1], device="cuda", dtype=torch.int32)
    return torch.where(z == z.amax(-1, keepdim=True), k, z.shape[-1]).amin(-1).int()


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("N,K,D", [(20000, 60, 40), (3000, 700, 64), (70000, 256, 128), (1, 1000, 16), (200, 5000, 33)])
def test_labels_of_scores_that_nearly_tie(N, K, D, with_bias):
    """Labels are those of the scores as documented: the product rounded, then the
    sum.  One fused step of both ranks neighbours otherwise (a fifth of these rows)."""
    xq, c, xs, cs, b = _near_ties(N, K, D, seed=N + K)
    b = b if with_bias else None
    z = (xq.double() @ c.double().T).float() * xs[:, None] * cs
    z = z if b is None else z + b
    assert torch.equal(fk.int8_scores(xq, c, cs, x_scale=xs, bias=b), z)
    assert torch.equal(fk.int8_assign(xq, c, cs, x_scale=xs, bias=b), _first_of_the_largest(z))


def test_labels_of_scores_that_nearly_tie_in_batches():
    xq, c, xs, cs, b = _near_ties(9000, 700, 64, seed=50, B=3, batched=True)
    z = (xq.double() @ c.double().transpose(-1, -2)).float() * xs[..., None] * cs[:, None] + b[:, None]
    assert torch.equal(fk.int8_assign(xq, c, cs, x_scale=xs, bias=b), _first_of_the_largest(z))


@pytest.mark.parametrize("dtype", [BF, HF], ids=["bf16", "fp16"])
@pytest.mark.parametrize("B,N,K,D,shared,reduction", [
    (0, 300, 500, 64, False, "sum"), (3, 77, 131, 65, False, "sum"), (2, 130, 300, 100, True, "sum"),
    (0, 5, 9000, 40, False, "sum"),          # split along the centroids
    (0, 17001, 9001, 24, False, "sum"),      # pieces of centroids and chunks of rows
    (0, 20000, 9000, 392, False, "sum"),     # rows gathered
    (2, 600, 700, 200, False, "none"), (0, 1500, 2000, 257, False, "none")])
def test_the_label_takes_no_rounding_of_its_own_in_gx(B, N, K, D, shared, reduction, dtype):
    """softmax - 1 at the label, most of a row's P, is rounded to 16 bits with the
    rest; what that takes away is added again in float32.  So only the others'
    entries are off by half a step, which the label's would double at least."""
    x, c, y = make(B, N, K, D, dtype, seed=51, shared=shared, ignored=0.1, ids=torch.int64, spread=2.0)
    g = torch.rand(y.shape, device="cuda") + 0.5 if reduction == "none" else None
    scale = 2.0
    _, gx, _ = fk.cluster_cross_entropy_grad(x, c, y, scale=scale, reduction=reduction, grad_loss=g)
    xd, cd = x.double(), c.double()
    if c.dim() < x.dim():
        cd = cd.expand(x.shape[0], *c.shape)
    keep = (y != -100)[..., None]
    at = y.clamp(min=0)[..., None]
    z = scale * xd @ cd.transpose(-1, -2)
    ez = (scale * (xd.abs() @ cd.abs().transpose(-1, -2)) * 2.0 ** -21).amax(-1, keepdim=True) + z.abs().amax(
        -1, keepdim=True) * 2.0 ** -22
    p = torch.softmax(z, -1).scatter(-1, at, 0.0)
    others = p.sum(-1, keepdim=True)
    w = 1.0 if g is None else g.double()[..., None]
    u = torch.finfo(dtype).eps / 2
    own = torch.gather(cd, -2, at.expand(*at.shape[:-1], D))
    want = torch.where(keep, scale * w * (p @ cd - others * own), 0.0)
    # (the scores' own error and float32's sums, as elsewhere; no half step for the label)
    tails, label = u + 2 * ez + 2.0 ** -18, 2 * ez + 2.0 ** -18
    tol = scale * w * ((p * tails) @ cd.abs() + others * own.abs() * label)
    if dtype == HF:
        tol = tol + scale * w * 2.0 ** -39 * cd.abs().sum(-2, keepdim=True)
    tol = torch.where(keep, tol + want.abs() * u + 2.0 ** -25, 0.0)
    close(gx, (want, tol), "gx")
