"""A head on cluster ids: train it with a cross entropy, answer from it in 8 bits.

The assignments of this package (``cosine_assign_triton``, ``euclid_assign``)
keep the argmax or argmin of a point's scores against the centroids.  These
operators use the same scores, x (B, N, D) against centroids (B, K, D), further:

* ``cluster_cross_entropy``: softmax cross entropy of the scores against
  cluster ids (those of ``batch_kmeans_*``, or any vocabulary's), without
  keeping the (B, N, K) scores, differentiable by x and by the centroids;
  ``cluster_cross_entropy_grad``: loss and gradients in one call, without
  autograd.
* ``quantize_rows``: rows as 8-bit integers with one scale each.
* ``int8_scores``: the scores from 8-bit x and centroids; ``int8_assign``: their
  argmax, without keeping them.

Shapes: x (N, D) with centroids (K, D); x (B, N, D) with centroids (B, K, D); or
x (B, N, D) with centroids (K, D) shared by the batches.  Any strides are
accepted.  All calls run on the current stream of x's device, never synchronise
and can be captured into a CUDA graph.  The reference has no counterpart.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native as nat
from . import _ops

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _status_word(device):
    """The device's error word; None while capturing, if it is not there yet
    (it would belong to the graph's memory)."""
    key = torch.device(device).index
    if key not in _ops.DeviceStatus._words and torch.cuda.is_current_stream_capturing():
        return None
    return _ops.DeviceStatus.word(device)


def _batched(x, centroids, name):
    """(x, centroids) as (B, N, D) and (B, K, D), with how x was folded."""
    if not isinstance(x, torch.Tensor) or not isinstance(centroids, torch.Tensor):
        raise TypeError(f"{name}: x and centroids must be tensors")
    if x.dim() not in (2, 3) or centroids.dim() not in (2, 3) or centroids.dim() > x.dim():
        raise ValueError(f"{name}: x (N, D) or (B, N, D) with centroids (K, D) or (B, K, D), got "
                         f"{tuple(x.shape)} and {tuple(centroids.shape)}")
    if x.shape[-1] != centroids.shape[-1]:
        raise ValueError(f"{name}: x has {x.shape[-1]} features, centroids {centroids.shape[-1]}")
    if x.shape[-1] < 1 or centroids.shape[-2] < 1:
        raise ValueError(f"{name}: at least one feature and one centroid are needed")
    if centroids.dim() == 3 and centroids.shape[0] != x.shape[0]:
        raise ValueError(f"{name}: x has {x.shape[0]} batches, centroids {centroids.shape[0]}")
    _ops._require_cuda(x, centroids)
    if x.device != centroids.device:
        raise ValueError(f"{name}: x is on {x.device}, centroids on {centroids.device}")
    x, centroids = x.detach(), centroids.detach()
    if centroids.dim() == 2:
        # one codebook: all rows of x are one batch
        rows = x.reshape(1, -1, x.shape[-1]) if x.dim() == 3 else x.unsqueeze(0)
        return rows, centroids.unsqueeze(0)
    return x, centroids


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


# ------------------------------------------------------------- cross entropy
class _Xent:
    """Checked arguments of one cross entropy call."""

    def __init__(self, x, centroids, labels, scale, ignore_index, reduction, name):
        self.x, self.c = _batched(x, centroids, name)
        if x.dtype not in _FLOATS:
            raise TypeError(f"{name}: unsupported dtype {x.dtype}")
        if centroids.dtype != x.dtype:
            raise TypeError(f"{name}: centroids are {centroids.dtype}, x is {x.dtype}")
        if not isinstance(labels, torch.Tensor) or labels.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: labels must be an int32 or int64 tensor")
        if labels.shape != x.shape[:-1]:
            raise ValueError(f"{name}: labels have shape {tuple(labels.shape)}, "
                             f"x {tuple(x.shape)}")
        if labels.device != x.device:
            raise ValueError(f"{name}: x is on {x.device}, labels on {labels.device}")
        scale = float(scale)
        if not (scale > 0.0 and math.isfinite(scale)):
            raise ValueError(f"{name}: scale must be positive and finite, got {scale}")
        if reduction not in _REDUCTIONS:
            raise ValueError(f"{name}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
        self.labels = labels.reshape(self.x.shape[:2])
        self.scale = scale
        self.ignore = int(ignore_index)
        self.reduction = reduction
        self.rows_shape = x.shape[:-1]
        self.device = x.device

    def _sizes(self):
        B, N, D = self.x.shape
        return B, N, self.c.shape[1], D

    def _head(self):
        return (nat.ptr(self.x), nat.ptr(self.c), nat.ptr(self.labels),
                nat.dtype_code(self.x.dtype), nat.dtype_code(self.labels.dtype), *self._sizes(),
                nat.strides(self.x, 3), nat.strides(self.c, 3), nat.strides(self.labels, 2),
                self.scale, self.ignore, _REDUCTIONS[self.reduction])

    def _ws(self, lib, want_x, want_c):
        nbytes = lib.fk_xent_workspace_size(
            nat.ptr(self.x), nat.ptr(self.c), nat.dtype_code(self.x.dtype), *self._sizes(),
            nat.strides(self.x, 3), nat.strides(self.c, 3), _REDUCTIONS[self.reduction],
            int(want_x), int(want_c))
        return _workspace(nbytes, self.device), nbytes

    def forward(self, keep_stats: bool):
        """(loss, row statistics or None, count)"""
        lib = nat.load()
        B, N, _, _ = self._sizes()
        f32 = dict(dtype=torch.float32, device=self.device)
        loss = torch.empty(self.rows_shape if self.reduction == "none" else (), **f32)
        stats = torch.empty((B, N, 4), **f32) if keep_stats else None
        count = torch.empty((), dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            ws, nbytes = self._ws(lib, False, False)
            nat.check(lib.fk_xent_forward(*self._head(), nat.ptr(loss), nat.ptr(stats),
                                          nat.ptr(count), nat.ptr(ws), nbytes,
                                          nat.ptr(_status_word(self.device)),
                                          nat.stream_handle(self.device)), "fk_xent_forward")
        return loss, stats, count

    def backward(self, stats, count, grad_loss, want_x, want_c):
        """(gradient by the folded x or None, by the centroids or None)"""
        lib = nat.load()
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        gx = new(self.x) if want_x else None
        gc = new(self.c) if want_c else None
        with torch.cuda.device(self.device):
            ws, nbytes = self._ws(lib, want_x, want_c)
            nat.check(lib.fk_xent_backward(
                *self._head(), nat.ptr(stats), nat.ptr(count), nat.ptr(grad_loss), nat.ptr(gx),
                nat.ptr(gc), nat.strides(gx, 3) if want_x else None,
                nat.strides(gc, 3) if want_c else None, nat.ptr(ws), nbytes,
                nat.ptr(_status_word(self.device)), nat.stream_handle(self.device)),
                "fk_xent_backward")
        return gx, gc


class _ClusterCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, centroids, labels, scale, ignore_index, reduction):
        call = _Xent(x, centroids, labels, scale, ignore_index, reduction, "cluster_cross_entropy")
        loss, stats, count = call.forward(keep_stats=any(ctx.needs_input_grad[:2]))
        ctx.save_for_backward(x, centroids, labels, stats, count)
        ctx.args = (scale, ignore_index, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        x, centroids, labels, stats, count = ctx.saved_tensors
        call = _Xent(x, centroids, labels, *ctx.args, "cluster_cross_entropy")
        grad_loss = grad_loss.to(torch.float32).contiguous()
        gx, gc = call.backward(stats, count, grad_loss, *ctx.needs_input_grad[:2])
        return (gx.view(x.shape) if gx is not None else None,
                gc.view(centroids.shape) if gc is not None else None, None, None, None, None)


def cluster_cross_entropy(x: torch.Tensor, centroids: torch.Tensor, labels: torch.Tensor, *,
                          scale: float = 1.0, ignore_index: int = -100,
                          reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``scale * x @ centroids^T`` against cluster ids.

    Args:
        x: (N, D) or (B, N, D) float16 / bfloat16 / float32 CUDA tensor.
        centroids: (K, D) or (B, K, D), x's dtype.
        labels: (N,) or (B, N) int32 / int64 cluster ids, e.g. the ids that
            ``batch_kmeans_Euclid`` returns.
        scale: positive factor of the scores (an inverse temperature).
        ignore_index: rows with this label count for nothing, whatever x holds
            there: loss 0, no gradient, not in the mean's denominator.
        reduction: 'mean' over the rows that are not ignored (NaN if there are
            none), 'sum', or 'none' for one loss per row.
    Returns:
        float32 loss, differentiable (once) by x and centroids.

    The (N, K) scores are never stored, forward or backward; sums and softmax
    statistics are float32.  Gradients of 16-bit inputs round the softmax to 16
    bits once, piece by piece, as the tensor cores take it.  A label outside
    [0, K) other than ``ignore_index`` makes the loss NaN.
    """
    return _ClusterCrossEntropy.apply(x, centroids, labels, scale, ignore_index, reduction)


def cluster_cross_entropy_grad(x: torch.Tensor, centroids: torch.Tensor, labels: torch.Tensor, *,
                               scale: float = 1.0, ignore_index: int = -100,
                               reduction: str = "mean",
                               grad_loss: Optional[torch.Tensor] = None):
    """``cluster_cross_entropy`` and its gradients in one call: (loss, grad_x,
    grad_centroids), without autograd.

    Arguments as there.  ``grad_loss``, a float32 tensor of the loss's shape,
    is the gradient of what follows by the loss (ones if not given; for float16
    inputs a factor such as a loss scale goes in here).
    """
    name = "cluster_cross_entropy_grad"
    call = _Xent(x, centroids, labels, scale, ignore_index, reduction, name)
    shape = call.rows_shape if reduction == "none" else ()
    if grad_loss is not None:
        if not isinstance(grad_loss, torch.Tensor) or grad_loss.dtype != torch.float32:
            raise TypeError(f"{name}: grad_loss must be a float32 tensor")
        if grad_loss.shape != shape:
            raise ValueError(f"{name}: grad_loss has shape {tuple(grad_loss.shape)}, "
                             f"the loss {tuple(shape)}")
        if grad_loss.device != x.device:
            raise ValueError(f"{name}: x is on {x.device}, grad_loss on {grad_loss.device}")
        grad_loss = grad_loss.detach().contiguous()
    elif reduction == "none":
        grad_loss = torch.ones(shape, dtype=torch.float32, device=x.device)
    loss, stats, count = call.forward(keep_stats=True)
    gx, gc = call.backward(stats, count, grad_loss, True, True)
    return loss, gx.view(x.shape), gc.view(centroids.shape)


# ------------------------------------------------------------- 8-bit scores
def quantize_rows(x: torch.Tensor):
    """Rows of x as 8-bit integers: (q int8 of x's shape, scale float32 of its
    leading shape) with x close to ``q * scale[..., None]``.

    x: (N, D) or (B, N, D) float16 / bfloat16 / float32.  For a row's largest
    magnitude m: scale = m / 127 and q = round(x * (127 / m)) in float32, ties
    to even.  Rows with m < 1e-36 become zeros with scale 0; rows that hold a
    NaN or an infinity become zeros with scale NaN.  q's rows are padded to 16
    bytes in memory, so that the products below read them in place.
    """
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3):
        raise ValueError("quantize_rows: x must be (N, D) or (B, N, D)")
    if x.dtype not in _FLOATS:
        raise TypeError(f"quantize_rows: unsupported dtype {x.dtype}")
    if x.shape[-1] < 1:
        raise ValueError("quantize_rows: at least one feature is needed")
    _ops._require_cuda(x)
    x = x.detach()
    xb = x if x.dim() == 3 else x.unsqueeze(0)
    B, N, D = xb.shape
    Dp = -(-D // 16) * 16
    q = torch.empty((B, N, Dp), dtype=torch.int8, device=x.device)[..., :D]
    scale = torch.empty((B, N), dtype=torch.float32, device=x.device)
    lib = nat.load()
    with torch.cuda.device(x.device):
        nat.check(lib.fk_quantize_rows(nat.ptr(xb), nat.dtype_code(x.dtype), B, N, D,
                                       nat.strides(xb, 3), nat.ptr(q), nat.strides(q, 3),
                                       nat.ptr(scale), nat.strides(scale, 2),
                                       nat.stream_handle(x.device)), "fk_quantize_rows")
    return (q, scale) if x.dim() == 3 else (q[0], scale[0])


class _Scores:
    """Checked arguments of one 8-bit call."""

    def __init__(self, x, centroids, c_scale, x_scale, bias, name):
        self.x, self.c = _batched(x, centroids, name)
        self.lead = x.shape[:-1]
        self.device = x.device
        if centroids.dtype != torch.int8:
            raise TypeError(f"{name}: centroids must be int8 (see quantize_rows), got "
                            f"{centroids.dtype}")
        if x.dtype != torch.int8 and x.dtype not in _FLOATS:
            raise TypeError(f"{name}: unsupported dtype {x.dtype}")
        if (x_scale is None) == (x.dtype == torch.int8):
            raise ValueError(f"{name}: x_scale goes with int8 x, and only with it")
        self.c_scale = self._scale(c_scale, centroids.shape[:-1], "c_scale", name)
        self.bias = None if bias is None else self._scale(bias, centroids.shape[:-1], "bias", name)
        self.x_scale = None
        if x_scale is not None:
            self.x_scale = self._scale(x_scale, x.shape[:-1], "x_scale", name)
            if centroids.dim() == 2 and x.dim() == 3:
                self.x_scale = self.x_scale.reshape(1, -1)

    def _scale(self, t, shape, what, name):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
            raise TypeError(f"{name}: {what} must be a float32 tensor")
        if t.shape != shape:
            raise ValueError(f"{name}: {what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.device != self.device:
            raise ValueError(f"{name}: x is on {self.device}, {what} on {t.device}")
        t = t.detach()
        return t if t.dim() == 2 else t.unsqueeze(0)

    def sizes(self):
        B, N, D = self.x.shape
        return B, N, self.c.shape[1], D

    def operands(self):
        return (nat.ptr(self.x), nat.ptr(self.c), nat.ptr(self.x_scale), nat.ptr(self.c_scale),
                nat.ptr(self.bias))

    def strides(self):
        two = lambda t: None if t is None else nat.strides(t, 2)  # noqa: E731
        return (nat.strides(self.x, 3), nat.strides(self.c, 3), two(self.x_scale),
                two(self.c_scale), two(self.bias))

    def workspace(self, lib, argmax):
        nbytes = lib.fk_int8_workspace_size(
            nat.ptr(self.x), nat.ptr(self.c), nat.dtype_code(self.x.dtype), *self.sizes(),
            nat.strides(self.x, 3), nat.strides(self.c, 3), int(argmax))
        return _workspace(nbytes, self.device), nbytes


def _check_out(out, shape, dtype, device, name):
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.shape != shape:
        raise ValueError(f"{name}: out must be a {dtype} tensor of shape {tuple(shape)}")
    if out.device != device:
        raise ValueError(f"{name}: x is on {device}, out on {out.device}")


def int8_scores(x: torch.Tensor, centroids: torch.Tensor, c_scale: torch.Tensor, *,
                x_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None
                ) -> torch.Tensor:
    """Scores of points against 8-bit centroids: ``x @ centroids^T`` of the
    integers, times x_scale per point, times c_scale per centroid, plus bias.

    Args:
        x: (N, D) or (B, N, D); int8 with ``x_scale`` (see ``quantize_rows``), or
            float16 / bfloat16 / float32, whose rows are then quantised within
            the call.
        centroids, c_scale: int8 (K, D) or (B, K, D) with float32 scales (K,) or
            (B, K), as ``quantize_rows`` returns them.
        bias: optional float32 (K,) or (B, K), like ``c_scale``.
        out_dtype: float16, bfloat16 or float32 (default: x's dtype, float32 for
            int8 x).
        out: optional (N, K) or (B, N, K) output with rows of unit stride.
    Returns:
        The scores.  The integer sum is exact; scaling is float32 in the order
        above, rounded once to ``out_dtype``.
    """
    name = "int8_scores"
    q = _Scores(x, centroids, c_scale, x_scale, bias, name)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else x.dtype if x.dtype in _FLOATS else torch.float32
    if out_dtype not in _FLOATS:
        raise TypeError(f"{name}: unsupported out_dtype {out_dtype}")
    shape = (*q.lead, centroids.shape[-2])
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=q.device)
    else:
        _check_out(out, shape, out_dtype, q.device, name)
        if shape[-1] > 1 and out.stride(-1) != 1:
            raise ValueError(f"{name}: rows of out must have unit stride")
    B, N, K, _ = q.sizes()
    folded = out.view(B, N, K)
    lib = nat.load()
    with torch.cuda.device(q.device):
        ws, nbytes = q.workspace(lib, False)
        nat.check(lib.fk_int8_scores(
            *q.operands(), nat.ptr(folded), nat.dtype_code(q.x.dtype), nat.dtype_code(out_dtype),
            *q.sizes(), *q.strides(), nat.strides(folded, 3), nat.ptr(ws), nbytes,
            nat.ptr(_status_word(q.device)), nat.stream_handle(q.device)), "fk_int8_scores")
    return out


def int8_assign(x: torch.Tensor, centroids: torch.Tensor, c_scale: torch.Tensor, *,
                x_scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Centroid of the largest 8-bit score for every point; int32 (N,) or (B, N).

    ``int8_scores`` (float32) followed by an argmax, without storing the scores:
    the 8-bit counterpart of ``cosine_assign_triton``, and with
    ``bias = -0.5 * ||c||^2`` of ``euclid_assign``.  Arguments as there; ties go
    to the lowest index, a NaN score counts as the largest.
    """
    name = "int8_assign"
    q = _Scores(x, centroids, c_scale, x_scale, bias, name)
    if out is None:
        out = torch.empty(q.lead, dtype=torch.int32, device=q.device)
    else:
        _check_out(out, q.lead, torch.int32, q.device, name)
    B, N, _, _ = q.sizes()
    folded = out.view(B, N)
    lib = nat.load()
    with torch.cuda.device(q.device):
        ws, nbytes = q.workspace(lib, True)
        nat.check(lib.fk_int8_assign(
            *q.operands(), nat.ptr(folded), nat.dtype_code(q.x.dtype), *q.sizes(), *q.strides(),
            nat.strides(folded, 2), nat.ptr(ws), nbytes, nat.ptr(_status_word(q.device)),
            nat.stream_handle(q.device)), "fk_int8_assign")
    return out
