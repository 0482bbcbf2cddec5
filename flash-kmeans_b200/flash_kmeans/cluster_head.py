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

import contextlib
import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native as nat
from . import _ops

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class _Device:
    """What a call needs of a device: its index and its error word."""

    def __init__(self, device):
        self.index = device.index
        self.status = None

    def status_ptr(self):
        """The device's error word; None while capturing, if it is not there yet
        (it would belong to the graph's memory)."""
        if self.status is None:
            if self.index not in _ops.DeviceStatus._words and torch.cuda.is_current_stream_capturing():
                return None
            self.status = _ops.DeviceStatus.word(torch.device("cuda", self.index)).data_ptr()
        return self.status


_devices: dict = {}
# Checked arguments and sizes by everything that they depend on (shapes, strides,
# types, devices, alignment, options): a call with the same layout skips the
# checks.  Bounded, because lengths may differ from call to call.
_layouts: dict = {}
_MOST_LAYOUTS = 4096


def _device(device) -> _Device:
    d = _devices.get(device)
    if d is None:
        d = _devices[device] = _Device(device)
    return d


def _layout(key, make):
    found = _layouts.get(key)
    if found is None:
        found = make()
        if len(_layouts) >= _MOST_LAYOUTS:
            _layouts.clear()
        _layouts[key] = found
    return found


def _on(device):
    """Workspaces are sized for the current device."""
    return torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext()


# the current stream's handle; torch's public way makes an object of it first,
# a sixteenth of a small call's time
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, what, dev: _Device, *args):
    """fn(*args, status word, current stream) on device dev."""
    index = dev.index
    if torch.cuda.current_device() == index:
        st = fn(*args, dev.status or dev.status_ptr(), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, dev.status_ptr(), _raw_stream(index))
    if st:
        nat.check(st, what)


def _has_tangent(t):
    return isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None


def _refuse_tangents(name, *tensors):
    """A tangent would be dropped without a word: a dual tensor need not require grad."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(map(_has_tangent, tensors)):
        raise NotImplementedError(f"{name}: forward-mode derivatives are not implemented")


def _numbers(name, scale, ignore_index):
    """scale and ignore_index as Python's; what would be lost on the way is refused."""
    if type(scale) is float and type(ignore_index) is int:
        return scale, ignore_index
    if isinstance(scale, torch.Tensor):
        if scale.is_cuda:
            raise TypeError(f"{name}: scale must be a number; reading one from a GPU would wait for it "
                            "(multiply x by it instead)")
        if scale.requires_grad and torch.is_grad_enabled() or _has_tangent(scale):
            raise TypeError(f"{name}: scale must be a number; it gets no gradient (multiply a learnable "
                            "factor into x instead)")
    if isinstance(ignore_index, torch.Tensor) and ignore_index.is_cuda:
        raise TypeError(f"{name}: ignore_index must be a number; reading one from a GPU would wait for it")
    # (a fraction, NaN or an infinity is no id)
    if ignore_index != ignore_index or ignore_index in (math.inf, -math.inf) or (
            int(ignore_index) != ignore_index):
        raise TypeError(f"{name}: ignore_index must be a whole number, got {ignore_index}")
    return float(scale), int(ignore_index)


def _check_pair(x, centroids, name):
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


def _valued(t):
    """t in memory of its own where that holds t's negatives (such a view is
    what the imaginary part of a conjugate is): kernels read memory."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def _three(t):
    """Shape and strides of (M, D) or (B, M, D) as three."""
    sh, st = t.shape, t.stride()
    return (sh, st) if len(sh) == 3 else ((1, *sh), (sh[0] * st[0], *st))


def _two(t):
    sh, st = t.shape, t.stride()
    return st if len(sh) == 2 else (0, *st)


class _Strides:
    """Strides for the C side: an array and its address."""

    __slots__ = ("array", "at")

    def __init__(self, strides):
        self.array = (nat.ctypes.c_int64 * len(strides))(*strides)
        self.at = nat.ctypes.addressof(self.array)


# ------------------------------------------------------------- cross entropy
class _XentLayout:
    """Checked layout of a cross entropy call (x already folded)."""

    def __init__(self, x, centroids, labels, scale, ignore_index, reduction):
        (B, N, D), xs = _three(x)
        (_, K, _), cs = _three(centroids)
        self.lib = nat.load()
        code = _REDUCTIONS[reduction]
        dtype = nat.dtype_code(x.dtype)
        sizes = (B, N, K, D)
        self.rows = B * N
        self.kept = kept = [_Strides(s) for s in (xs, cs, _two(labels), (N * D, D, 1), (K * D, D, 1))]
        xs, cs, ls, gxs, gcs = (s.at for s in kept)
        self.middle = (dtype, nat.dtype_code(labels.dtype), *sizes, xs, cs, ls, scale, ignore_index,
                       code)
        self.grad_strides = gxs, gcs
        # by which gradients are wanted; (0, 0) is the forward pass
        self.bytes = {w: self.lib.fk_xent_workspace_size(x.data_ptr(), centroids.data_ptr(), dtype,
                                                         *sizes, xs, cs, code, *w)
                      for w in ((0, 0), (0, 1), (1, 0), (1, 1))}
        self.both = self.lib.fk_xent_loss_grad_workspace_size(
            x.data_ptr(), centroids.data_ptr(), dtype, *sizes, xs, cs, code, 1, 1)


def _check_xent(x, centroids, labels, scale, ignore_index, reduction, name):
    _check_pair(x, centroids, name)
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name}: unsupported dtype {x.dtype}")
    if centroids.dtype != x.dtype:
        raise TypeError(f"{name}: centroids are {centroids.dtype}, x is {x.dtype}")
    if not isinstance(labels, torch.Tensor) or labels.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: labels must be an int32 or int64 tensor")
    if labels.shape != x.shape[:-1]:
        raise ValueError(f"{name}: labels have shape {tuple(labels.shape)}, x {tuple(x.shape)}")
    if labels.device != x.device:
        raise ValueError(f"{name}: x is on {x.device}, labels on {labels.device}")
    # as the kernels hold it: in float32, and times log2(e)
    s32 = nat.ctypes.c_float(scale).value
    if not (s32 > 0.0 and s32 * 1.44269504 <= torch.finfo(torch.float32).max):
        raise ValueError(f"{name}: scale must be positive and finite in float32, got {scale}")
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"{name}: ignore_index does not fit 64 bits: {ignore_index}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{name}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")


class _Xent:
    """One cross entropy call: x and labels folded, its layout."""

    __slots__ = ("x", "c", "labels", "shapes", "none", "at", "dev")

    def __init__(self, x, centroids, labels, scale, ignore_index, reduction, name):
        tensors = isinstance(x, torch.Tensor) and isinstance(centroids, torch.Tensor) and isinstance(
            labels, torch.Tensor)
        if not tensors or not x.is_cuda:
            _check_xent(x, centroids, labels, scale, ignore_index, reduction, name)
        x, centroids = _valued(x), _valued(centroids)
        self.shapes = x.shape, centroids.shape
        self.none = reduction == "none"
        if x.dim() == 3 and centroids.dim() == 2:
            _check_xent(x, centroids, labels, scale, ignore_index, reduction, name)
            x, labels = x.reshape(-1, x.shape[-1]), labels.reshape(-1)
        self.x, self.c, self.labels = x, centroids, labels
        key = (x.shape, x.stride(), x.dtype, x.device, x.data_ptr() & 15, centroids.shape,
               centroids.stride(), centroids.dtype, centroids.device, centroids.data_ptr() & 15,
               labels.shape, labels.stride(), labels.dtype, labels.device, scale, ignore_index, reduction)

        def make():
            _check_xent(x, centroids, labels, scale, ignore_index, reduction, name)
            with _on(x.device):
                return _XentLayout(x, centroids, labels, scale, ignore_index, reduction)

        self.at = _layout(key, make)
        self.dev = _device(x.device)

    def forward(self, keep: bool):
        """(loss, row statistics and count for the backward pass, or None)"""
        at = self.at
        nbytes = at.bytes[0, 0]
        new = self.x.new_empty
        loss = new(self.shapes[0][:-1] if self.none else (), dtype=torch.float32)
        # the count of rows behind the statistics, or behind the workspace
        ws = new(nbytes + 16, dtype=torch.uint8)
        kept = new(4 * at.rows + 4, dtype=torch.float32) if keep else None
        stats = kept.data_ptr() if keep else None
        count = stats + 16 * at.rows if keep else ws.data_ptr() + nbytes
        _call(at.lib.fk_xent_forward, "fk_xent_forward", self.dev, self.x.data_ptr(), self.c.data_ptr(),
              self.labels.data_ptr(), *at.middle, loss.data_ptr(), stats, count, ws.data_ptr(), nbytes)
        return loss, kept

    def loss_grad(self, grad_loss):
        """(loss, gradient by x, by the centroids)"""
        at = self.at
        xshape, cshape = self.shapes
        new = self.x.new_empty
        loss = new(xshape[:-1] if self.none else (), dtype=torch.float32)
        gx, gc = new(xshape), new(cshape)
        ws = new(at.both, dtype=torch.uint8)
        _call(at.lib.fk_xent_loss_grad, "fk_xent_loss_grad", self.dev, self.x.data_ptr(),
              self.c.data_ptr(), self.labels.data_ptr(), *at.middle, loss.data_ptr(),
              None if grad_loss is None else grad_loss.data_ptr(), gx.data_ptr(), gc.data_ptr(),
              *at.grad_strides, ws.data_ptr(), at.both)
        return loss, gx, gc

    def backward(self, kept, grad_loss, want_x, want_c):
        """(gradient by x or None, by the centroids or None)"""
        at = self.at
        nbytes = at.bytes[int(want_x), int(want_c)]
        xshape, cshape = self.shapes
        new = self.x.new_empty
        gx = new(xshape) if want_x else None
        gc = new(cshape) if want_c else None
        ws = new(nbytes, dtype=torch.uint8)
        stats = kept.data_ptr()
        _call(at.lib.fk_xent_backward, "fk_xent_backward", self.dev, self.x.data_ptr(), self.c.data_ptr(),
              self.labels.data_ptr(), *at.middle, stats, stats + 16 * at.rows,
              None if grad_loss is None else grad_loss.data_ptr(), gx.data_ptr() if want_x else None,
              gc.data_ptr() if want_c else None, *at.grad_strides, ws.data_ptr(), nbytes)
        return gx, gc


def _gradients(ctx, grad_loss):
    call = _Xent(*ctx.saved_tensors, *ctx.args, "cluster_cross_entropy")
    return call.backward(ctx.kept, _valued(grad_loss).contiguous(), *ctx.needs_input_grad[:2])


class _OnceOnly(torch.autograd.Function):
    """Hands gradients on as functions of the tensors behind them, whose own
    derivative raises: without it a second derivative would be left out."""

    @staticmethod
    def forward(ctx, gx, gc, x, centroids, grad_loss):
        return gx, gc

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("cluster_cross_entropy is differentiable once; its gradients have no derivative")


class _ClusterCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, centroids, labels, scale, ignore_index, reduction):
        call = _Xent(x, centroids, labels, scale, ignore_index, reduction, "cluster_cross_entropy")
        loss, ctx.kept = call.forward(True)
        ctx.save_for_backward(x, centroids, labels)
        ctx.args = (scale, ignore_index, reduction)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        if not torch.is_grad_enabled():
            return *_gradients(ctx, grad_loss), None, None, None, None
        # a graph of the backward pass is recorded
        with torch.no_grad():
            gx, gc = _gradients(ctx, grad_loss)
        return *_OnceOnly.apply(gx, gc, *ctx.saved_tensors[:2], grad_loss), None, None, None, None


def _autocast(x, centroids):
    """Under autocast, operands of two float types meet in its type, as a matrix
    product's do; equal types stay."""
    dtypes = [getattr(t, "dtype", None) for t in (x, centroids)]
    if dtypes[0] != dtypes[1] and all(t in _FLOATS for t in dtypes):
        low = torch.get_autocast_dtype("cuda")
        x, centroids = x.to(low), centroids.to(low)
    return x, centroids


def cluster_cross_entropy(x: torch.Tensor, centroids: torch.Tensor, labels: torch.Tensor, *,
                          scale: float = 1.0, ignore_index: int = -100,
                          reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``scale * x @ centroids^T`` against cluster ids.

    Args:
        x: (N, D) or (B, N, D) float16 / bfloat16 / float32 CUDA tensor.
        centroids: (K, D) or (B, K, D), x's dtype; under autocast also another
            float type (both are then cast to autocast's).
        labels: (N,) or (B, N) int32 / int64 cluster ids, e.g. the ids that
            ``batch_kmeans_Euclid`` returns.
        scale: positive factor of the scores (an inverse temperature), a number:
            multiply a learnable one into x.
        ignore_index: rows with this label count for nothing, whatever x holds
            there: loss 0, no gradient, not in the mean's denominator.
        reduction: 'mean' over the rows that are not ignored (NaN if there are
            none), 'sum', or 'none' for one loss per row.
    Returns:
        float32 loss, differentiable (once, in reverse mode) by x and centroids;
        forward-mode tangents are refused.

    The (N, K) scores are never stored, forward or backward; sums and softmax
    statistics are float32.  Gradients of 16-bit inputs round the softmax to 16
    bits once, piece by piece, as the tensor cores take it (in the gradient by x,
    not the label's own entry).  A label outside
    [0, K) other than ``ignore_index`` makes the loss NaN.
    """
    _refuse_tangents("cluster_cross_entropy", x, centroids)
    scale, ignore_index = _numbers("cluster_cross_entropy", scale, ignore_index)
    if torch.is_autocast_enabled("cuda"):
        x, centroids = _autocast(x, centroids)
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False)
                                    or getattr(centroids, "requires_grad", False)):
        return _ClusterCrossEntropy.apply(x, centroids, labels, scale, ignore_index, reduction)
    return _Xent(x, centroids, labels, scale, ignore_index, reduction,
                 "cluster_cross_entropy").forward(False)[0]


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
    _refuse_tangents(name, x, centroids, grad_loss)
    scale, ignore_index = _numbers(name, scale, ignore_index)
    with torch.no_grad():
        call = _Xent(x, centroids, labels, scale, ignore_index, reduction, name)
        shape = x.shape[:-1] if call.none else ()
        if grad_loss is not None:
            if not isinstance(grad_loss, torch.Tensor) or grad_loss.dtype != torch.float32:
                raise TypeError(f"{name}: grad_loss must be a float32 tensor")
            if grad_loss.shape != shape:
                raise ValueError(f"{name}: grad_loss has shape {tuple(grad_loss.shape)}, "
                                 f"the loss {tuple(shape)}")
            if grad_loss.device != x.device:
                raise ValueError(f"{name}: x is on {x.device}, grad_loss on {grad_loss.device}")
            grad_loss = _valued(grad_loss).contiguous()
        elif call.none:
            grad_loss = torch.ones(shape, dtype=torch.float32, device=x.device)
        return call.loss_grad(grad_loss)


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
    x = _valued(x.detach())
    xb = x if x.dim() == 3 else x.unsqueeze(0)
    B, N, D = xb.shape
    Dp = -(-D // 16) * 16
    q = torch.empty((B, N, Dp), dtype=torch.int8, device=x.device)[..., :D]
    scale = torch.empty((B, N), dtype=torch.float32, device=x.device)
    lib = nat.load()
    with torch.cuda.device(x.device):
        xs, qs, ss = (_Strides(t.stride()) for t in (xb, q, scale))
        nat.check(lib.fk_quantize_rows(xb.data_ptr(), nat.dtype_code(x.dtype), B, N, D, xs.at,
                                       q.data_ptr(), qs.at, scale.data_ptr(), ss.at,
                                       nat.stream_handle(x.device)), "fk_quantize_rows")
    return (q, scale) if x.dim() == 3 else (q[0], scale[0])


def _check_scale(t, shape, device, what, name):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
        raise TypeError(f"{name}: {what} must be a float32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name}: x is on {device}, {what} on {t.device}")


def _check_int8(x, centroids, c_scale, x_scale, bias, name):
    _check_pair(x, centroids, name)
    if centroids.dtype != torch.int8:
        raise TypeError(f"{name}: centroids must be int8 (see quantize_rows), got {centroids.dtype}")
    if x.dtype != torch.int8 and x.dtype not in _FLOATS:
        raise TypeError(f"{name}: unsupported dtype {x.dtype}")
    if (x_scale is None) == (x.dtype == torch.int8):
        raise ValueError(f"{name}: x_scale goes with int8 x, and only with it")
    _check_scale(c_scale, centroids.shape[:-1], x.device, "c_scale", name)
    if bias is not None:
        _check_scale(bias, centroids.shape[:-1], x.device, "bias", name)
    if x_scale is not None:
        _check_scale(x_scale, x.shape[:-1], x.device, "x_scale", name)


class _ScoresLayout:
    """Checked layout of an 8-bit call (x already folded)."""

    def __init__(self, x, centroids, c_scale, x_scale, bias, argmax):
        (B, N, D), xs = _three(x)
        (_, K, _), cs = _three(centroids)
        self.lib = nat.load()
        self.x_code = nat.FK_I8 if x.dtype == torch.int8 else nat.dtype_code(x.dtype)
        self.sizes = (B, N, K, D)
        self.kept = [None if s is None else _Strides(s) for s in (
            xs, cs, *(None if t is None else _two(t) for t in (x_scale, c_scale, bias)))]
        self.strides = tuple(None if s is None else s.at for s in self.kept)
        xs, cs = self.strides[:2]
        self.bytes = self.lib.fk_int8_workspace_size(x.data_ptr(), centroids.data_ptr(), self.x_code,
                                                     *self.sizes, xs, cs, argmax)


class _Scores:
    """One 8-bit call: x folded, its layout."""

    __slots__ = ("lead", "device", "at", "dev", "operands")

    def __init__(self, x, centroids, c_scale, x_scale, bias, argmax, name):
        if not (isinstance(x, torch.Tensor) and x.is_cuda and isinstance(centroids, torch.Tensor)
                and isinstance(c_scale, torch.Tensor)
                and (x_scale is None or isinstance(x_scale, torch.Tensor))
                and (bias is None or isinstance(bias, torch.Tensor))):
            _check_int8(x, centroids, c_scale, x_scale, bias, name)
        x, c_scale, x_scale, bias = _valued(x), _valued(c_scale), _valued(x_scale), _valued(bias)
        self.lead, self.device = x.shape[:-1], x.device
        if x.dim() == 3 and centroids.dim() == 2:
            _check_int8(x, centroids, c_scale, x_scale, bias, name)
            x = x.reshape(-1, x.shape[-1])
            x_scale = None if x_scale is None else x_scale.reshape(-1)
        key = (x.shape, x.stride(), x.dtype, x.device, x.data_ptr() & 15, centroids.shape,
               centroids.stride(), centroids.dtype, centroids.device, centroids.data_ptr() & 15,
               c_scale.shape, c_scale.stride(), c_scale.dtype, c_scale.device,
               x_scale is not None and (x_scale.shape, x_scale.stride(), x_scale.dtype, x_scale.device),
               bias is not None and (bias.shape, bias.stride(), bias.dtype, bias.device), argmax)

        def make():
            _check_int8(x, centroids, c_scale, x_scale, bias, name)
            with _on(x.device):
                return _ScoresLayout(x, centroids, c_scale, x_scale, bias, argmax)

        self.at = _layout(key, make)
        self.dev = _device(self.device)
        # the folded tensors stay referenced until the call is queued
        self.operands = (x, centroids, x_scale, c_scale, bias)

    def pointers(self):
        return [None if t is None else t.data_ptr() for t in self.operands]

    def workspace(self):
        n = self.at.bytes
        if not n:
            return None, None, 0
        ws = self.operands[0].new_empty(n, dtype=torch.uint8)
        return ws, ws.data_ptr(), n


def _check_out(out, shape, dtype, device, name):
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.shape != shape:
        raise ValueError(f"{name}: out must be a {dtype} tensor of shape {tuple(shape)}")
    if out.device != device:
        raise ValueError(f"{name}: x is on {device}, out on {out.device}")
    if any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name}: out must not be expanded, its elements share memory")
    if out.is_neg():
        raise ValueError(f"{name}: out must not be a negated view")
    reach = 0      # of the dimensions with smaller strides
    for s, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        if s <= reach and 0 not in out.shape:
            raise ValueError(f"{name}: out must not overlap itself, got strides {out.stride()}")
        reach += s * (n - 1)
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: out must not require grad, the results have none")


def _written(out):
    """Kernels wrote it through its pointer: for autograd, it has changed in place."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def _fold_strides(out, name):
    """Strides of out with its first two dimensions as one batch of rows."""
    (B, N), st = out.shape[:2], out.stride()
    if B > 1 and N > 1 and st[0] != N * st[1]:
        raise ValueError(f"{name}: with shared centroids, out's batches must follow each other at the "
                         "distance of its rows")
    return (0, st[1] if N > 1 else st[0], *st[2:])


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
        out: optional (N, K) or (B, N, K) output with rows of unit stride, which
            shares no memory with itself or with the inputs.
    Returns:
        The scores.  The integer sum is exact; scaling is float32 in the order
        above, rounded once to ``out_dtype``.  They carry no gradient, whatever
        the inputs require.
    """
    name = "int8_scores"
    given = out is not None
    q = _Scores(x, centroids, c_scale, x_scale, bias, False, name)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else x.dtype if x.dtype in _FLOATS else torch.float32
    if out_dtype not in _FLOATS:
        raise TypeError(f"{name}: unsupported out_dtype {out_dtype}")
    shape = (*q.lead, centroids.shape[-2])
    if out is None:
        out = x.new_empty(shape, dtype=out_dtype)
    else:
        _check_out(out, shape, out_dtype, q.device, name)
        if shape[-1] > 1 and out.stride(-1) != 1:
            raise ValueError(f"{name}: rows of out must have unit stride")
    B, N, K, _ = q.at.sizes
    if out.dim() == 3:
        # (not .view(): a fold over batches needs rows at one distance)
        strides = out.stride() if B == out.shape[0] else _fold_strides(out, name)
    else:
        strides = (N * out.stride(0), *out.stride())
    strides = _Strides(strides)
    ws, ws_ptr, nbytes = q.workspace()
    _call(q.at.lib.fk_int8_scores, "fk_int8_scores", q.dev, *q.pointers(), out.data_ptr(), q.at.x_code,
          nat.dtype_code(out_dtype), *q.at.sizes, *q.at.strides, strides.at, ws_ptr, nbytes)
    return _written(out) if given else out


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
    given = out is not None
    q = _Scores(x, centroids, c_scale, x_scale, bias, True, name)
    if out is None:
        out = x.new_empty(q.lead, dtype=torch.int32)
    else:
        _check_out(out, q.lead, torch.int32, q.device, name)
    B = q.at.sizes[0]
    if out.dim() == 2:
        strides = out.stride() if B == out.shape[0] else _fold_strides(out, name)
    else:
        strides = (0, *out.stride())
    strides = _Strides(strides)
    ws, ws_ptr, nbytes = q.workspace()
    _call(q.at.lib.fk_int8_assign, "fk_int8_assign", q.dev, *q.pointers(), out.data_ptr(), q.at.x_code,
          *q.at.sizes, *q.at.strides, strides.at, ws_ptr, nbytes)
    return _written(out) if given else out
