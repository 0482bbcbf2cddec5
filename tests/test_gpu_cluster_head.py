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
    xd, cd = x.detach().double().cpu(), c.detach().double().cpu()
    y = y.cpu().long()
    B, N, K, D = xd.shape[0] if x.dim() == 3 else 1, x.shape[-2], c.shape[-2], x.shape[-1]
    xb, yb = xd.reshape(B, N, D), y.reshape(B, N)
    cb = cd if c.dim() == 3 else cd.expand(B, K, D)
    u = torch.finfo(x.dtype).eps / 2
    up = 2.0 ** -24 if x.dtype == FP else u
    keep = yb != ignore_index
    xb = torch.where(keep[..., None], xb, torch.zeros(()).double())
    z = scale * torch.einsum("bnd,bkd->bnk", xb, cb)
    ez = scale * torch.einsum("bnd,bkd->bnk", xb.abs(), cb.abs()) * (D_EPS + 2.0 ** -23)
    ezm = ez.amax(-1) + z.abs().amax(-1) * 2.0 ** -23
    at = yb.clamp(min=0)[..., None]
    lp = torch.log_softmax(z, -1)
    rows = torch.where(keep, -lp.gather(-1, at).squeeze(-1), torch.zeros(()).double())
    rtol = rows * 2.0 ** -20 + 2 * ezm * rows.clamp(max=1.0) * 1.5 + 1e-30
    rtol = torch.where(keep, rtol, torch.zeros(()).double())
    count = keep.sum().double() if reduction == "mean" else torch.ones(()).double()
    if reduction == "none":
        loss, ltol = rows.reshape(y.shape), rtol.reshape(y.shape)
    else:
        loss = rows.sum() / count
        ltol = rtol.sum() / count + loss.abs() * 2.0 ** -23
    w = keep.double()
    if g is not None:
        w = w * (g.detach().double().cpu().reshape(B, N) if reduction == "none" else g.double().cpu())
    w = w / count.clamp(min=1)
    p = lp.exp()
    # 1 - p at the label from the loss, which keeps its small differences
    P = p.clone().scatter_(-1, at, torch.expm1(-rows)[..., None]) * w[..., None]
    rel = (2 * ezm[..., None] + 2.0 ** -19 + up)
    Pt = P.abs() * rel
    if x.dtype == HF:
        Pt = Pt + 2.0 ** -25 * 2.0 ** -14 * w.abs().amax()
    Pt = torch.where(keep[..., None], Pt, torch.zeros(()).double())
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
    got = got.detach().double().cpu()
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
