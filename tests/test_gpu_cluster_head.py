"""Cluster head on the GPU: cross entropy over centroids, its gradients, 8-bit
scores and assignment, against plain float64 forms.

Tolerances are bounds on rounding, taken before the first run:
* a score is a float32 sum of D products: off by at most D_EPS = 2^-21 of
  sum |x||c| (the tensor core's sums keep 24 bits; 2^-21 leaves room for their
  truncation), times scale, plus half a step of the product with scale;
* exp2 and the sums over centroids add 2^-20 of the result;
* P = softmax - one-hot is rounded once to its 16-bit operand type (half a step,
  eps / 2), float32 inputs keep 24 bits of it in three parts;
* a gradient is a float32 sum of P times an operand and is rounded once.
"""
import math
import random

import pytest
import torch

import flash_kmeans as fk

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
D_EPS = 2.0 ** -21


def make(B, N, K, D, dtype, seed=0, shared=False, ignored=0.0, ids=torch.int32, spread=0.6):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Bx = max(B, 1)
    Bc = 1 if shared or B == 0 else Bx
    c = torch.randn(Bc, K, D, device="cuda", generator=g) / math.sqrt(D)
    y = torch.randint(0, K, (Bx, N), device="cuda", generator=g)
    batch = torch.arange(Bx, device="cuda").clamp(max=Bc - 1)[:, None]
    x = c[batch, y] + torch.randn(Bx, N, D, device="cuda", generator=g) * (spread / math.sqrt(D))
    if ignored:
        y = y.masked_fill(torch.rand(Bx, N, device="cuda", generator=g) < ignored, -100)
    x, c, y = x.to(dtype), c.to(dtype), y.to(ids)
    if B == 0:
        x, c, y = x[0], c[0], y[0]
    elif shared:
        c = c[0]
    return x, c, y


def reference(x, c, y, scale, reduction, ignore_index=-100, g=None):
    """(loss, gx, gc) in float64 with bounds on each: (value, tolerance) pairs."""
    dev = "cuda" if x.shape[-2] * c.shape[-2] > 1 << 24 else "cpu"
    xd, cd = x.detach().double().to(dev), c.detach().double().to(dev)
    y = y.to(dev).long()
    B, N, K, D = xd.shape[0] if x.dim() == 3 else 1, x.shape[-2], c.shape[-2], x.shape[-1]
    xb, yb = xd.reshape(B, N, D), y.reshape(B, N)
    cb = cd if c.dim() == 3 else cd.expand(B, K, D)
    u = torch.finfo(x.dtype).eps / 2
    up = 2.0 ** -24 if x.dtype == FP else u
    keep = yb != ignore_index
    xb = torch.where(keep[..., None], xb, torch.zeros((), dtype=torch.float64, device=dev))
    z = scale * torch.einsum("bnd,bkd->bnk", xb, cb)
    ez = scale * torch.einsum("bnd,bkd->bnk", xb.abs(), cb.abs()) * (D_EPS + 2.0 ** -23)
    ezm = ez.amax(-1) + z.abs().amax(-1) * 2.0 ** -23
    at = yb.clamp(min=0)[..., None]
    lp = torch.log_softmax(z, -1)
    # log-softmax itself would lose losses below 2^-53 beside the label's 1
    d = (z - z.gather(-1, at)).scatter(-1, at, -math.inf)
    top = d.amax(-1, keepdim=True).clamp(min=0.0)
    others, own = (d - top).exp().sum(-1), (-top).exp().squeeze(-1)
    rows = torch.where(top.squeeze(-1) > 0, top.squeeze(-1) + (others + own).log(), others.log1p())
    rows = torch.where(keep, rows, torch.zeros((), dtype=torch.float64, device=dev))
    rtol = rows * 2.0 ** -20 + 2 * ezm * rows.clamp(max=1.0) * 1.5 + 1e-30
    rtol = torch.where(keep, rtol, torch.zeros((), dtype=torch.float64, device=dev))
    count = keep.sum().double() if reduction == "mean" else torch.ones((), dtype=torch.float64, device=dev)
    if reduction == "none":
        loss, ltol = rows.reshape(y.shape), rtol.reshape(y.shape)
    else:
        loss = rows.sum() / count
        ltol = rtol.sum() / count + loss.abs() * 2.0 ** -23
    w = keep.double()
    if g is not None:
        w = w * (g.detach().double().to(dev).reshape(B, N) if reduction == "none" else g.double().to(dev))
    w = w / count.clamp(min=1)
    p = lp.exp()
    # 1 - p at the label from the loss, which keeps its small differences
    P = p.clone().scatter_(-1, at, torch.expm1(-rows)[..., None]) * w[..., None]
    rel = (2 * ezm[..., None] + 2.0 ** -19 + up)
    Pt = P.abs() * rel
    if x.dtype == HF:
        Pt = Pt + 2.0 ** -25 * 2.0 ** -14 * w.abs().amax()
    Pt = torch.where(keep[..., None], Pt, torch.zeros((), dtype=torch.float64, device=dev))
    sums = 2.0 ** -20
    gx = scale * torch.einsum("bnk,bkd->bnd", P, cb)
    gxt = scale * torch.einsum("bnk,bkd->bnd", Pt + sums * P.abs(), cb.abs())
    gc = scale * torch.einsum("bnk,bnd->bkd", P, xb)
    gct = scale * torch.einsum("bnk,bnd->bkd", Pt + sums * P.abs(), xb.abs())
    if c.dim() == 2:
        gc, gct = gc.sum(0), gct.sum(0)
    gx, gxt = gx.reshape(x.shape), gxt.reshape(x.shape)
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    gxt, gct = gxt + gx.abs() * u + tiny, gct + gc.abs() * u + tiny
    return (loss, ltol), (gx, gxt), (gc.reshape(c.shape), gct.reshape(c.shape))


def close(got, want, what):
    value, tol = want
    got = got.detach().double().to(value.device)
    assert got.shape == value.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - value).abs() - tol
    assert float(off.max()) <= 0, (
        f"{what}: off by {float((got - value).abs().max()):.3e}, worst over its bound by "
        f"{float(off.max()):.3e} at {int(off.argmax())} of {off.numel()}")


SIZES = [
    # B, N, K, D, shared
    (0, 1, 2, 8, False),
    (0, 1, 1, 1, False),
    (0, 5, 1000, 128, False),
    (0, 33, 257, 64, False),
    (0, 130, 300, 17, False),
    (2, 77, 1031, 100, False),
    (3, 40, 129, 65, True),
    (0, 700, 513, 320, False),
    (1, 300, 5000, 96, False),
    (0, 1500, 3000, 72, False),   # CTA pairs
    (5, 600, 512, 128, False),
    (0, 300, 40100, 512, False),  # columns past a window of tiles
    (1, 257, 256, 64, False), (0, 129, 65, 8, False),   # one row, one column more than a tile
]


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,N,K,D,shared", SIZES)
def test_loss_rows(B, N, K, D, shared, dtype):
    x, c, y = make(B, N, K, D, dtype, shared=shared, ignored=0.2)
    loss = fk.cluster_cross_entropy(x, c, y, scale=7.0, reduction="none")
    assert loss.dtype == FP and loss.shape == y.shape
    close(loss, reference(x, c, y, 7.0, "none")[0], "loss")


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,N,K,D,shared", SIZES)
def test_gradients(B, N, K, D, shared, dtype):
    reduction = "sum" if dtype == HF else "mean"
    x, c, y = make(B, N, K, D, dtype, seed=1, shared=shared, ignored=0.0 if N == 1 else 0.2,
                   ids=torch.int64)
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=5.0, reduction=reduction)
    assert gx.dtype == gc.dtype == dtype
    want = reference(x, c, y, 5.0, reduction)
    for got, w, what in zip((loss, gx, gc), want, ("loss", "gx", "gc")):
        close(got, w, what)
    # autograd runs the same kernels
    xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
    l2 = fk.cluster_cross_entropy(xr, cr, y, scale=5.0, reduction=reduction)
    l2.backward()
    assert torch.equal(l2.detach(), loss) and torch.equal(xr.grad, gx) and torch.equal(cr.grad, gc)


def quant_ref(x):
    """The documented quantisation in float32 on the CPU (tensor by tensor:
    torch divides a number by a tensor through its reciprocal)."""
    v = x.float().cpu()
    m = v.abs().amax(-1, keepdim=True)
    top = torch.full_like(m, 127.0)
    zero = torch.zeros(())
    inv = torch.where(m < 1e-36, zero, top / m)
    return (v * inv).round().clamp(-127, 127), torch.where(m < 1e-36, zero, m / top).squeeze(-1)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,N,D", [(0, 1, 1), (0, 3, 15), (2, 5, 16), (0, 4, 4097), (3, 1000, 100),
                                   (0, 3000, 64), (1, 2, 20000)])
def test_quantize_rows(B, N, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(max(B, 1), N, D, device="cuda", generator=g).mul(3.0).to(dtype)
    x = x if B else x[0]
    q, s = fk.quantize_rows(x)
    qr, sr = quant_ref(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(q.cpu().float(), qr) and torch.equal(s.cpu(), sr)


def int_case(B, N, K, D, seed=0, shared=False, bias=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Bc = 1 if shared else max(B, 1)
    xq = torch.randint(-127, 128, (max(B, 1), N, D), device="cuda", generator=g).to(torch.int8)
    cq = torch.randint(-127, 128, (Bc, K, D), device="cuda", generator=g).to(torch.int8)
    xs = torch.rand(max(B, 1), N, device="cuda", generator=g) * 0.02 + 1e-3
    cs = torch.rand(Bc, K, device="cuda", generator=g) * 0.02 + 1e-3
    b = torch.randn(Bc, K, device="cuda", generator=g) if bias else None
    pick = lambda t, s: None if t is None else t[0] if B == 0 or s else t  # noqa: E731
    return pick(xq, False), pick(cq, shared), pick(xs, False), pick(cs, shared), pick(b, shared)


def int_scores(xq, cq, xs, cs, b):
    """Exact sums in float64, then the documented float32 order on the CPU."""
    xq, cq, xs, cs = xq.cpu(), cq.cpu(), xs.cpu(), cs.cpu()
    acc = (xq.double() @ cq.double().transpose(-1, -2)).float()
    z = acc * xs[..., None] * cs[..., None, :]
    return z if b is None else z + b.cpu()[..., None, :]


INT_SIZES = [
    (0, 1, 1, 1, False), (0, 1, 1000, 128, False), (0, 7, 33, 100, False), (2, 65, 130, 97, False),
    (3, 50, 300, 256, True), (0, 400, 700, 255, False), (0, 1200, 2100, 160, False),
    (4, 300, 257, 1025, False), (0, 3, 4096, 4096, False),
    (3, 9000, 700, 64, False),    # several row blocks of CTA pairs in turn, one column chunk
    (0, 300, 9100, 4096, False),  # columns past a window of tiles
    (2, 2000, 900, 640, True),    # 256 columns wide and one chunk
    (1, 257, 128, 33, True), (2, 513, 129, 20, False),   # one row more than a block, or two blocks
]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("B,N,K,D,shared", INT_SIZES)
def test_int8_scores_and_assign(B, N, K, D, shared, bias):
    args = int_case(B, N, K, D, shared=shared, bias=bias)
    xq, cq, xs, cs, b = args
    z = int_scores(*args)
    got = fk.int8_scores(xq, cq, cs, x_scale=xs, bias=b)
    assert got.dtype == FP and torch.equal(got.cpu(), z)
    for t in (BF, HF):
        assert torch.equal(fk.int8_scores(xq, cq, cs, x_scale=xs, bias=b, out_dtype=t).cpu(), z.to(t))
    k = torch.arange(K)
    first = torch.where(z == z.amax(-1, keepdim=True), k, K).amin(-1).int()
    ids = fk.int8_assign(xq, cq, cs, x_scale=xs, bias=b)
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu(), first)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
def test_float_points_are_quantised_in_the_call(dtype):
    x, c, _ = make(2, 130, 300, 100, dtype, seed=4)
    cq, cs = fk.quantize_rows(c)
    xq, xs = fk.quantize_rows(x)
    assert torch.equal(fk.int8_scores(x, cq, cs, out_dtype=FP),
                       fk.int8_scores(xq, cq, cs, x_scale=xs))
    assert fk.int8_scores(x, cq, cs).dtype == dtype
    assert torch.equal(fk.int8_assign(x, cq, cs), fk.int8_assign(xq, cq, cs, x_scale=xs))


# ------------------------------------------------------------ cross entropy
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
def test_several_pieces_and_row_chunks(dtype):
    """N x K past a piece's 2^27 elements: the softmax goes in several pieces of
    centroids and of rows, whose sums are carried between products."""
    x, c, y = make(0, 17001, 9001, 24, dtype, seed=5, ignored=0.1)
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=4.0)
    for got, w, what in zip((loss, gx, gc), reference(x, c, y, 4.0, "mean"), ("loss", "gx", "gc")):
        close(got, w, what)


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("live", ["all", "most", "few", "first", "last", "one chunk", "none"])
def test_only_the_rows_that_count_are_multiplied(live, dtype):
    """Work large enough that the backward pass gathers the rows that are not
    ignored, in two chunks of rows, with float rows that ignored ones would spoil."""
    N, K, D = 20000, 9000, 392
    x, c, y = make(0, N, K, D, dtype, seed=26, ids=torch.int64)
    g = torch.Generator(device="cuda").manual_seed(27)
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    if live == "most":
        keep = torch.rand(N, device="cuda", generator=g) < 0.8
    elif live != "all":
        keep[:] = False
        if live == "few":
            keep[torch.randint(0, N, (37,), device="cuda", generator=g)] = True
        elif live == "first":
            keep[0] = True
        elif live == "last":
            keep[-1] = True
        elif live == "one chunk":
            keep[: 16384 // 2] = True      # as many as a chunk of rows holds, less than two
    y = torch.where(keep, y, torch.full_like(y, -100))
    dirty = x.clone()
    dirty[~keep] = float("nan")
    loss, gx, gc = fk.cluster_cross_entropy_grad(dirty, c, y, scale=4.0)
    if live == "none":
        assert torch.isnan(loss) and gx.eq(0).all() and gc.eq(0).all()
        return
    for got, w, what in zip((loss, gx, gc), reference(x, c, y, 4.0, "mean"), ("loss", "gx", "gc")):
        close(got, w, what)
    assert gx[~keep].eq(0).all()
    # the same through autograd, one gradient at a time, and a gradient per row
    xr, cr = dirty.clone().requires_grad_(), c.clone().requires_grad_()
    fk.cluster_cross_entropy(xr, cr, y, scale=4.0).backward()
    assert torch.equal(xr.grad, gx) and torch.equal(cr.grad, gc)
    cr = c.clone().requires_grad_()
    fk.cluster_cross_entropy(dirty, cr, y, scale=4.0).backward()
    close(cr.grad, reference(x, c, y, 4.0, "mean")[2], "gc alone")   # (split into other sums)
    up = torch.rand(N, device="cuda", generator=g)
    got = fk.cluster_cross_entropy_grad(dirty, c, y, scale=4.0, reduction="none", grad_loss=up)
    for a, w, what in zip(got, reference(x, c, y, 4.0, "none", g=up), ("rows", "gx", "gc")):
        close(a, w, what)


def test_few_rows_many_centroids_split_the_sums():
    """A short product over a long axis is split and joined."""
    for dtype in (BF, FP):
        x, c, y = make(0, 3, 20011, 40, dtype, seed=6)
        loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=3.0)
        for got, w, what in zip((loss, gx, gc), reference(x, c, y, 3.0, "mean"), ("loss", "gx", "gc")):
            close(got, w, what)
        x, c, y = make(0, 20011, 3, 40, dtype, seed=7)
        loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=3.0)
        for got, w, what in zip((loss, gx, gc), reference(x, c, y, 3.0, "mean"), ("loss", "gx", "gc")):
            close(got, w, what)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
def test_row_losses_take_one_gradient_each(dtype):
    x, c, y = make(2, 70, 150, 48, dtype, seed=8, ignored=0.2)
    g = torch.randn(2, 70, device="cuda") * torch.logspace(-3, 3, 70, device="cuda")
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0, reduction="none", grad_loss=g)
    for got, w, what in zip((loss, gx, gc), reference(x, c, y, 2.0, "none", g=g), ("loss", "gx", "gc")):
        close(got, w, what)
    xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
    fk.cluster_cross_entropy(xr, cr, y, scale=2.0, reduction="none").backward(g)
    assert torch.equal(xr.grad, gx) and torch.equal(cr.grad, gc)


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_upstream_factor(reduction):
    x, c, y = make(0, 50, 60, 32, BF, seed=9, ignored=0.3)
    g = torch.tensor(37.5, device="cuda")
    got = fk.cluster_cross_entropy_grad(x, c, y, reduction=reduction, grad_loss=g)
    for a, w, what in zip(got, reference(x, c, y, 1.0, reduction, g=g), ("loss", "gx", "gc")):
        close(a, w, what)


def test_saved_tensors_go_through_hooks():
    """What autograd keeps can be moved away or computed again."""
    from torch.utils.checkpoint import checkpoint
    x, c, y = make(0, 300, 500, 64, BF, seed=28, ignored=0.2)
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0)

    def step(wrap):
        xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
        wrap(lambda a, b: fk.cluster_cross_entropy(a, b, y, scale=2.0), xr, cr).backward()
        assert torch.equal(xr.grad, gx) and torch.equal(cr.grad, gc)

    def on_cpu(f, *args):
        with torch.autograd.graph.save_on_cpu():
            return f(*args)

    step(on_cpu)
    step(lambda f, *args: checkpoint(f, *args, use_reentrant=False))
    xr = x.clone().requires_grad_()
    loss = fk.cluster_cross_entropy(xr, c, y)
    with torch.no_grad():
        y[0] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_one_gradient_alone():
    x, c, y = make(0, 90, 120, 40, BF, seed=10)
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y)
    xr = x.clone().requires_grad_()
    fk.cluster_cross_entropy(xr, c, y).backward()
    assert torch.equal(xr.grad, gx)
    cr = c.clone().requires_grad_()
    fk.cluster_cross_entropy(x, cr, y).backward()
    assert torch.equal(cr.grad, gc)
    assert not fk.cluster_cross_entropy(x, c, y).requires_grad
    with pytest.raises(RuntimeError):
        xr = x.clone().requires_grad_()
        g, = torch.autograd.grad(fk.cluster_cross_entropy(xr, c, y), xr, create_graph=True)
        g.sum().backward()


def test_gradients_against_differences():
    """Central differences of the loss along random directions (float32)."""
    x, c, y = make(2, 21, 37, 19, FP, seed=11, ignored=0.1)
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=3.0, reduction="sum")
    for t, g, which in ((x, gx, 0), (c, gc, 1)):
        d = torch.randn_like(t)
        d = d / d.norm()
        h = 2.0 ** -6
        at = lambda s: fk.cluster_cross_entropy(*((t + s * d, c) if which == 0 else (x, t + s * d)),  # noqa: E731
                                                y, scale=3.0, reduction="sum").double()
        num = (at(h) - at(-h)) / (2 * h)
        exact = (g.double() * d.double()).sum()
        # truncation: h^2 / 6 times a third derivative of at most (scale |row|)^3 summed
        # over the rows that move; rounding: two sums of float32 losses over 2 h
        row = float(torch.maximum(x.norm(dim=-1).max(), c.norm(dim=-1).max()))
        bound = h * h / 6 * (3.0 * row) ** 3 * 2 + 2 * float(at(0.0)) * 2.0 ** -20 / (2 * h)
        assert abs(float(num - exact)) <= bound, (which, float(num), float(exact), bound)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
def test_whatever_an_ignored_row_holds(dtype):
    x, c, y = make(0, 200, 300, 40, dtype, seed=12)
    drop = torch.arange(0, 200, 3, device="cuda")
    y[drop] = -100
    clean = fk.cluster_cross_entropy_grad(x, c, y)
    rows = fk.cluster_cross_entropy(x, c, y, reduction="none")
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).max, torch.finfo(dtype).min):
        xb = x.clone()
        xb[drop] = bad
        for a, b in zip(fk.cluster_cross_entropy_grad(xb, c, y), clean):
            assert torch.equal(a, b)
        assert torch.equal(fk.cluster_cross_entropy(xb, c, y, reduction="none"), rows)
    assert rows[drop].eq(0).all() and clean[1][drop].eq(0).all()


@pytest.mark.parametrize("N,K,D", [(300, 400, 64), (20000, 9000, 392)])
def test_an_ignored_id_within_the_vocabulary(N, K, D):
    x, c, y = make(0, N, K, D, BF, seed=31, ids=torch.int64)
    y[: N // 2] = 5
    got = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0, ignore_index=5)
    for a, w, what in zip(got, reference(x, c, y, 2.0, "mean", ignore_index=5), ("loss", "gx", "gc")):
        close(a, w, what)
    want = fk.cluster_cross_entropy_grad(x, c, y.masked_fill(y == 5, -100), scale=2.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_points_that_are_their_own_centroids():
    """One tensor as both operands, expanded rows and centroids: each use has its gradient."""
    w = (torch.randn(40, 24, device="cuda") * 0.3).requires_grad_()
    y = torch.arange(40, device="cuda")
    fk.cluster_cross_entropy(w, w, y).backward()
    wd = w.detach().double().requires_grad_()
    torch.nn.functional.cross_entropy(wd @ wd.T, y).backward()
    assert torch.allclose(w.grad.double(), wd.grad, rtol=1e-5, atol=1e-6)
    w.grad = None
    fk.cluster_cross_entropy(w[:1].expand(3, 50, 24), w.expand(3, 40, 24), y[:1].expand(3, 50)).backward()
    wd.grad = None
    torch.nn.functional.cross_entropy(wd[:1] @ wd.T, y[:1]).backward()
    assert torch.allclose(w.grad.double(), wd.grad, rtol=1e-5, atol=1e-6)


def test_no_row_left():
    x, c, y = make(0, 40, 30, 16, BF, seed=13)
    y.fill_(7)
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, ignore_index=7)
    assert torch.isnan(loss) and gx.eq(0).all() and gc.eq(0).all()
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, ignore_index=7, reduction="sum")
    assert loss == 0 and gx.eq(0).all() and gc.eq(0).all()


@pytest.mark.parametrize("shape", [(0, 16), (2, 0, 16), (0, 5, 16)])
def test_empty(shape):
    x = torch.zeros(shape, dtype=BF, device="cuda")
    c = torch.ones(*shape[:-2], 9, 16, dtype=BF, device="cuda")
    y = torch.zeros(shape[:-1], dtype=torch.int32, device="cuda")
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y)
    assert torch.isnan(loss) and gx.shape == x.shape and gc.eq(0).all()
    assert fk.cluster_cross_entropy(x, c, y, reduction="sum") == 0
    assert fk.cluster_cross_entropy(x, c, y, reduction="none").shape == y.shape
    q, s = fk.quantize_rows(x)
    cq, cs = fk.quantize_rows(c)
    assert q.shape == x.shape and fk.int8_assign(x, cq, cs).shape == y.shape
    assert fk.int8_scores(q, cq, cs, x_scale=s).shape == (*y.shape, 9)


@pytest.mark.parametrize("bad", [300, 1 << 40, -1, -(1 << 40)])
def test_a_label_outside_is_loud_and_harmless(bad):
    from flash_kmeans import _ops
    x, c, y = make(0, 100, 300, 32, BF, seed=14, ids=torch.int64)
    good = fk.cluster_cross_entropy(x, c, y, reduction="none")
    y[17] = bad
    rows = fk.cluster_cross_entropy(x, c, y, reduction="none")
    keep = torch.arange(100, device="cuda") != 17
    assert torch.isnan(rows[17]) and torch.equal(rows[keep], good[keep])
    with pytest.raises(RuntimeError, match="outside"):
        _ops.DeviceStatus.raise_if_set("cuda:0")
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y)
    assert torch.isnan(loss) and torch.isnan(gx[17]).all() and torch.isnan(gc).all()
    assert torch.isfinite(gx[keep]).all()
    with pytest.raises(RuntimeError, match="outside"):
        _ops.DeviceStatus.raise_if_set("cuda:0")
    assert torch.equal(fk.cluster_cross_entropy(x, c, y, ignore_index=bad, reduction="none")[keep], good[keep])


def test_scores_that_are_not_finite():
    x, c, y = make(0, 64, 100, 32, BF, seed=15)
    x[3] = float("nan")
    x[5] = float("inf")
    rows = fk.cluster_cross_entropy(x, c, y, reduction="none")
    ok = torch.ones(64, dtype=torch.bool, device="cuda")
    ok[[3, 5]] = False
    assert torch.isnan(rows[[3, 5]]).all() and torch.isfinite(rows[ok]).all()
    # the largest finite scores: the sums are taken relative to the maximum
    big = torch.full((8, 32), 1e18, dtype=BF, device="cuda")
    cc = torch.zeros(5, 32, dtype=BF, device="cuda")
    cc[2] = 1e18
    yy = torch.tensor([2, 2, 0, 0, 1, 3, 4, 2], dtype=torch.int32, device="cuda")
    rows = fk.cluster_cross_entropy(big, cc, yy, reduction="none")
    want = float(32 * big[0, 0].double() * cc[2, 0].double())
    assert rows[yy == 2].eq(0).all()
    assert ((rows[yy != 2].double() / want - 1).abs() < 2.0 ** -20).all()
    # float32 past bf16's largest value
    xf = torch.full((4, 3), 3.4e38, device="cuda")
    cf = torch.zeros(2, 3, device="cuda")
    cf[0, 0] = 1e-37
    yf = torch.zeros(4, dtype=torch.int32, device="cuda")
    close(fk.cluster_cross_entropy(xf, cf, yf, reduction="none"), reference(xf, cf, yf, 1.0, "none")[0], "loss")


def test_strides_and_views():
    x, c, y = make(3, 90, 140, 64, BF, seed=16, ids=torch.int64)
    want = fk.cluster_cross_entropy_grad(x, c, y)
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)              # features far apart
    ct = torch.empty(140, 3, 64, dtype=BF, device="cuda").transpose(0, 1)  # batches interleaved
    ct.copy_(c)
    yt = torch.empty(90, 3, 2, dtype=torch.int64, device="cuda")[..., 1].t()
    yt.copy_(y)
    pad = torch.empty(3, 90, 67, dtype=BF, device="cuda")[..., 3:]   # rows off 16 bytes
    pad.copy_(x)
    rev = torch.empty(3, 200, 64, dtype=BF, device="cuda")[:, 5:185:2]
    rev.copy_(x)
    for xx in (xt, pad, rev):
        for cc in (c, ct):
            for a, b in zip(fk.cluster_cross_entropy_grad(xx, cc, yt), want):
                assert torch.equal(a, b)
    # one codebook, expanded or given once
    one = c[0]
    a = fk.cluster_cross_entropy_grad(x, one.expand(3, 140, 64), y)
    b = [fk.cluster_cross_entropy_grad(x, one.repeat(3, 1, 1), y)][0]
    s = fk.cluster_cross_entropy_grad(x, one, y)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # the tiles of a folded call fall elsewhere: sums in another order
    close(s[1], (b[1].double(), b[1].double().abs() * 2.0 ** -7 + 1e-6), "shared gx")
    assert s[2].shape == one.shape
    # x expanded over the batches, and one row broadcast
    xe = x[0].expand(3, 90, 64)
    a = fk.cluster_cross_entropy_grad(xe, c, y)
    b = fk.cluster_cross_entropy_grad(xe.contiguous(), c, y)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    xr = x[0, :1].clone().requires_grad_()
    fk.cluster_cross_entropy(xr.expand(90, 64), c[0], y[0], reduction="sum").backward()
    _, g, _ = fk.cluster_cross_entropy_grad(x[0, :1].expand(90, 64), c[0], y[0], reduction="sum")
    assert xr.grad.shape == (1, 64) and torch.allclose(xr.grad.float(), g.float().sum(0, keepdim=True), rtol=2.0 ** -6,
                                                       atol=90 * 2.0 ** -9 * float(g.abs().max()))


def test_same_bits_every_time():
    for dtype in (BF, FP):
        x, c, y = make(0, 3000, 2500, 72, dtype, seed=17, ignored=0.1)
        a = fk.cluster_cross_entropy_grad(x, c, y)
        for _ in range(3):
            b = fk.cluster_cross_entropy_grad(x, c, y)
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_streams_and_graphs():
    x, c, y = make(0, 500, 700, 96, BF, seed=18, ignored=0.1)
    x2, c2, y2 = make(0, 500, 700, 96, BF, seed=19, ignored=0.1)
    cq, cs = fk.quantize_rows(c)
    # (row losses of float16: a cleared word and two kernels of their own; the
    # long one: rows gathered, several pieces)
    xh, ch = x.half(), c.half()
    up = torch.rand(500, device="cuda")
    xl, cl, yl = make(0, 17000, 9000, 456, BF, seed=29, ignored=0.3)
    calls = [lambda: fk.cluster_cross_entropy_grad(x, c, y, scale=2.0), lambda: (fk.int8_assign(x, cq, cs),),
             lambda: (fk.int8_scores(x, cq, cs),), lambda: fk.quantize_rows(x),
             lambda: fk.cluster_cross_entropy_grad(xh, ch, y, reduction="none", grad_loss=up),
             lambda: fk.cluster_cross_entropy_grad(xl, cl, yl, scale=2.0)]
    want = [call() for call in calls]
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([call() for call in calls])
    torch.cuda.synchronize()
    for o in outs:
        for got, w in zip(o, want):
            assert all(torch.equal(p, q) for p, q in zip(got, w))
    # captured, replayed on new inputs, two graphs in turn
    graphs = []
    for call in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for g, out in graphs:
        g.replay()
    torch.cuda.synchronize()
    for (g, out), w in zip(graphs, want):
        assert all(torch.equal(p, q) for p, q in zip(out, w))
    # replayed on two streams at once, twice each
    for _, out in graphs:
        for t in out:
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(2):
        for i, (g, _) in enumerate(graphs):
            with torch.cuda.stream(streams[i % 2]):
                g.replay()
    torch.cuda.synchronize()
    for (g, out), w in zip(graphs, want):
        assert all(torch.equal(p, q) for p, q in zip(out, w))
    yl.fill_(-100)
    yl[1234] = 17
    xh.copy_(x2)
    x.copy_(x2)
    y.copy_(y2)
    c.copy_(c2)
    q2, s2 = fk.quantize_rows(c2)
    cq.copy_(q2)
    cs.copy_(s2)
    for g, _ in reversed(graphs):
        g.replay()
    torch.cuda.synchronize()
    for (g, out), call in zip(graphs, calls):
        assert all(torch.equal(p, q) for p, q in zip(out, call()))


def test_captured_autograd_step():
    """A training step captured whole, beside an eager graph of other leaves."""
    x, c, y = make(0, 300, 400, 64, BF, seed=20)
    _, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        xr, cr = x.clone().requires_grad_(), c.clone().requires_grad_()
        for _ in range(2):
            torch.autograd.grad(fk.cluster_cross_entropy(xr, cr, y, scale=2.0), (xr, cr))
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = torch.autograd.grad(fk.cluster_cross_entropy(xr, cr, y, scale=2.0), (xr, cr))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], gx) and torch.equal(got[1], gc)


# -------------------------------------------------------------- 8-bit scores
def test_int8_extremes_and_ties():
    # -128 is a legal operand; the sums reach 2^30
    D = 65536
    xq = torch.full((2, D), -128, dtype=torch.int8, device="cuda")
    cq = torch.full((5, D), -128, dtype=torch.int8, device="cuda")
    cq[1] = 127
    cq[4] = 0
    one = torch.ones(2, device="cuda")
    cs = torch.ones(5, device="cuda")
    z = fk.int8_scores(xq, cq, cs, x_scale=one)
    want = torch.tensor([2.0 ** 30, -128.0 * 127 * D, 2.0 ** 30, 2.0 ** 30, 0.0], device="cuda")
    assert torch.equal(z, want.expand(2, 5))
    assert fk.int8_assign(xq, cq, cs, x_scale=one).tolist() == [0, 0]      # lowest of equals
    # ties far apart, across tiles and column halves
    for K in (3, 200, 300, 1000, 9000):
        xq = torch.ones(300, 16, dtype=torch.int8, device="cuda")
        cq = torch.zeros(K, 16, dtype=torch.int8, device="cuda")
        first = K // 3
        cq[first] = 3
        cq[-1] = 3
        ids = fk.int8_assign(xq, cq, torch.ones(K, device="cuda"), x_scale=torch.ones(300, device="cuda"))
        assert ids.eq(first).all(), K


def test_int8_not_finite():
    """NaN scores come before all others, as argmax counts them; a point that
    holds NaN or infinity has a NaN scale and NaN scores."""
    x, c, _ = make(0, 300, 500, 64, FP, seed=21)
    x[7, 3] = float("nan")
    x[9, 0] = float("-inf")
    x[11] = 0
    x[12] = 1e-38
    cq, cs = fk.quantize_rows(c)
    q, s = fk.quantize_rows(x)
    assert torch.isnan(s[[7, 9]]).all() and q[[7, 9, 11, 12]].eq(0).all() and s[[11, 12]].eq(0).all()
    z = fk.int8_scores(x, cq, cs)
    assert torch.isnan(z[[7, 9]]).all() and z[[11, 12]].eq(0).all()
    ids = fk.int8_assign(x, cq, cs)
    assert ids[[7, 9, 11, 12]].eq(0).all()
    cs2 = cs.clone()
    cs2[[400, 333]] = float("nan")
    ids = fk.int8_assign(x, cq, cs2)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[7, 9]] = False
    assert ids[keep].eq(333).all() and ids[~keep].eq(0).all()
    # centroids taken out by their bias, and all of them
    bias = torch.zeros(500, device="cuda")
    bias[:490] = float("-inf")
    ids = fk.int8_assign(x, cq, cs, bias=bias)
    assert ids[keep].min() >= 490 and ids.max() < 500
    assert fk.int8_assign(x, cq, cs, bias=torch.full((500,), float("-inf"), device="cuda"))[keep].eq(0).all()
    low = torch.full((500,), torch.finfo(FP).min, device="cuda")
    assert fk.int8_assign(x, cq, cs, bias=low)[keep].max() < 500


def test_int8_strides_and_outputs():
    xq, cq, xs, cs, b = int_case(2, 100, 150, 48, seed=22, bias=True)
    want = fk.int8_scores(xq, cq, cs, x_scale=xs, bias=b)
    ids = fk.int8_assign(xq, cq, cs, x_scale=xs, bias=b)
    xv = xq.transpose(1, 2).contiguous().transpose(1, 2)
    cv = torch.empty(2, 150, 50, dtype=torch.int8, device="cuda")[..., 1:49]
    cv.copy_(cq)
    sv = torch.empty(100, 2, device="cuda").t()
    sv.copy_(xs)
    tv = torch.empty(2, 150, 3, device="cuda")[..., 2]
    tv.copy_(cs)
    bv = torch.empty(150, 2, device="cuda").t()
    bv.copy_(b)
    assert torch.equal(fk.int8_scores(xv, cv, tv, x_scale=sv, bias=bv), want)
    assert torch.equal(fk.int8_assign(xv, cv, tv, x_scale=sv, bias=bv), ids)
    # into a view: what lies around it stays
    frame = torch.full((2, 102, 157), 7.0, device="cuda")
    got = fk.int8_scores(xq, cq, cs, x_scale=xs, bias=b, out=frame[:, 1:101, 3:153])
    assert torch.equal(got, want)
    frame[:, 1:101, 3:153] = 7.0
    assert frame.eq(7.0).all()
    lab = torch.full((2, 102, 3), -5, dtype=torch.int32, device="cuda")
    fk.int8_assign(xq, cq, cs, x_scale=xs, bias=b, out=lab[:, 1:101, 1])
    assert torch.equal(lab[:, 1:101, 1], ids)
    lab[:, 1:101, 1] = -5
    assert lab.eq(-5).all()
    # one codebook: all rows in one call, into a view whose batches follow each other
    want1 = fk.int8_scores(xq, cq[0], cs[0], x_scale=xs)
    rows = torch.full((2, 100, 157), 7.0, device="cuda")
    assert torch.equal(fk.int8_scores(xq, cq[0], cs[0], x_scale=xs, out=rows[..., 4:154]), want1)
    rows[..., 4:154] = 7.0
    assert rows.eq(7.0).all()
    ids1 = torch.empty(2, 100, 2, dtype=torch.int32, device="cuda")[..., 0]
    assert torch.equal(fk.int8_assign(xq, cq[0], cs[0], x_scale=xs, out=ids1),
                       fk.int8_assign(xq, cq[0], cs[0], x_scale=xs))
    with pytest.raises(ValueError, match="follow each other"):
        fk.int8_scores(xq, cq[0], cs[0], x_scale=xs, out=frame[:, 1:101, 3:153])
    with pytest.raises(ValueError, match="follow each other"):
        fk.int8_assign(xq, cq[0], cs[0], x_scale=xs, out=lab[:, 1:101, 1])
    # a codebook expanded over the batches
    e = fk.int8_scores(xq, cq[0].expand(2, 150, 48), cs[0].expand(2, 150), x_scale=xs)
    assert torch.equal(e, fk.int8_scores(xq, cq[0], cs[0], x_scale=xs))


def test_scores_behind_32_bit_offsets():
    """Outputs and inputs whose element offsets pass 2^31."""
    N, K = 70000, 32768                     # 2.3e9 scores
    xq, cq, xs, cs, _ = int_case(0, N, K, 16, seed=23)
    z = fk.int8_scores(xq, cq, cs, x_scale=xs, out_dtype=BF)
    tail = fk.int8_scores(xq[-100:], cq, cs, x_scale=xs[-100:], out_dtype=BF)
    assert torch.equal(z[-100:], tail)
    del z
    wide = torch.empty(33000, 1 << 16, dtype=torch.int8, device="cuda")
    part = wide[:, :16]
    part.copy_(xq[:33000])
    assert torch.equal(fk.int8_assign(part, cq, cs, x_scale=xs[:33000]),
                       fk.int8_assign(xq[:33000], cq, cs, x_scale=xs[:33000]))
    del wide, part
    big = torch.empty(66000, 1 << 15, dtype=BF, device="cuda")
    x, c, y = make(0, 66000, 40, 24, BF, seed=24)
    v = big[:, :24]
    v.copy_(x)
    assert all(torch.equal(p, q) for p, q in zip(fk.cluster_cross_entropy_grad(v, c, y),
                                                 fk.cluster_cross_entropy_grad(x, c, y)))


# --------------------------------------------------------------- as it is used
@pytest.mark.parametrize("K", [16, 64])
def test_losses_behind_32_bit_offsets(K):
    """Rows past 2^31 elements, all multiplied (16 centroids) and gathered (64)."""
    N, D = (1 << 20) + 77, 2056
    x = torch.zeros(N, D, dtype=BF, device="cuda")
    ends = torch.cat([torch.arange(200), torch.arange(N - 300, N)]).cuda()
    xe, c, ye = make(0, 500, K, D, BF, seed=33, ids=torch.int64, ignored=0.1)
    x[ends] = xe
    y = torch.full((N,), -100, dtype=torch.int64, device="cuda")
    y[ends] = ye
    up = torch.zeros(N, device="cuda")
    up[ends] = torch.rand(500, device="cuda") + 0.5
    loss, gx, gc = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0, reduction="none", grad_loss=up)
    want = reference(xe, c, ye, 2.0, "none", g=up[ends])
    for a, w, what in zip((loss[ends], gx[ends], gc), want, ("rows", "gx", "gc")):
        close(a, w, what)
    assert loss[200:-300].eq(0).all() and gx[200:-300].eq(0).all()
    q, s = fk.quantize_rows(x)
    qe, se = fk.quantize_rows(xe)
    assert torch.equal(q[ends], qe) and torch.equal(s[ends], se) and q[200:-300].eq(0).all()


def _drawn(seed, most):
    """Sizes of any kind up to `most` products, short and long in every direction."""
    r = random.Random(seed)
    while True:
        B = r.choice([0, 0, 1, 3])
        N, K, D = (round(math.exp(r.uniform(0.0, math.log(n)))) for n in (12000, 12000, 4096))
        if max(B, 1) * N * K * D < most and max(B, 1) * N * K < 1 << 25:
            return r, B, N, K, D


@pytest.mark.parametrize("seed", range(24))
def test_drawn_sizes_of_8_bit_scores(seed):
    r, B, N, K, D = _drawn(seed, 1 << 36)
    args = int_case(B, N, K, D, seed=seed, shared=r.random() < 0.3, bias=r.random() < 0.5)
    xq, cq, xs, cs, b = args
    acc = (xq.double() @ cq.double().transpose(-1, -2)).float()     # (exact in 53 bits)
    z = acc * xs[..., None] * cs[..., None, :]
    z = z if b is None else z + b[..., None, :]
    k = torch.arange(K, device="cuda", dtype=torch.int32)
    first = torch.where(z == z.amax(-1, keepdim=True), k, K).amin(-1)
    assert torch.equal(fk.int8_assign(xq, cq, cs, x_scale=xs, bias=b), first), (B, N, K, D)
    assert torch.equal(fk.int8_scores(xq, cq, cs, x_scale=xs, bias=b), z), (B, N, K, D)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_sizes_of_losses(seed):
    r, B, N, K, D = _drawn(seed + 100, 1 << 34)
    dtype, reduction = r.choice([BF, HF, FP]), r.choice(["mean", "sum"])
    x, c, y = make(B, N, K, D, dtype, seed=seed, shared=r.random() < 0.3, ignored=0.2)
    y[..., 0] = 0                       # (a row that counts)
    got = fk.cluster_cross_entropy_grad(x, c, y, scale=2.0, reduction=reduction)
    for a, w, what in zip(got, reference(x, c, y, 2.0, reduction), ("loss", "gx", "gc")):
        close(a, w, f"{what} of {(B, N, K, D)}")


def test_from_clusters_to_an_8_bit_head():
    """k-means gives the ids, the head learns them, answers in 8 bits."""
    g = torch.Generator(device="cuda").manual_seed(25)
    centres = torch.randn(1, 50, 64, device="cuda", generator=g)
    pick = torch.randint(0, 50, (1, 4000), device="cuda", generator=g)
    x = (centres[0, pick] + 0.1 * torch.randn(1, 4000, 64, device="cuda", generator=g)).to(BF)
    ids, cent, _ = fk.batch_kmeans_Euclid(x, 50, max_iters=5, init_centroids=centres.to(BF))
    head = cent.clone().requires_grad_()
    loss = fk.cluster_cross_entropy(x, head, ids, scale=0.25)
    loss.backward()
    want = reference(x, cent, ids, 0.25, "mean")
    close(loss, want[0], "loss")
    close(head.grad, want[2], "centroids")
    with torch.no_grad():
        head -= 0.1 * head.grad
    cq, cs = fk.quantize_rows(head)
    assert not cq.requires_grad
    half = -0.5 * cent.float().square().sum(-1)
    z = fk.int8_scores(x, cq, cs, bias=half, out_dtype=FP)
    got = fk.int8_assign(x, cq, cs, bias=half)
    k = torch.arange(50, device="cuda", dtype=torch.int32)
    assert torch.equal(got, torch.where(z == z.amax(-1, keepdim=True), k, 50).amin(-1).int())
    assert (got == ids).float().mean() > 0.99
