"""Cluster head: what is refused, and the host-only entry points (CPU only)."""
import contextlib
import ctypes

import pytest
import torch

import flash_kmeans as fk

X = torch.randn(6, 8)
C = torch.randn(4, 8)
Y = torch.zeros(6, dtype=torch.int32)


@pytest.mark.parametrize("fn", [fk.cluster_cross_entropy, fk.cluster_cross_entropy_grad])
def test_cross_entropy_refusals(fn):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fn(X, C, Y)
    with pytest.raises(ValueError, match="features"):
        fn(X, torch.randn(4, 7), Y)
    with pytest.raises(ValueError, match="batches"):
        fn(torch.randn(2, 6, 8), torch.randn(3, 4, 8), torch.zeros(2, 6, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one"):
        fn(X, torch.randn(0, 8), Y)
    with pytest.raises(ValueError, match=r"x \(N, D\)"):
        fn(X[0], C, Y)
    with pytest.raises(ValueError, match=r"x \(N, D\)"):
        fn(X, torch.randn(1, 4, 8), Y)      # centroids of more dimensions than x
    with pytest.raises(TypeError, match="tensors"):
        fn([1.0], C, Y)


class _OnCuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks after the device's."""
    is_cuda = property(lambda self: True)


def _cuda(t):
    return t.as_subclass(_OnCuda)


@pytest.mark.parametrize("kw,err,match", [
    (dict(x=X.double()), TypeError, "dtype"),
    (dict(c=C.half()), TypeError, "centroids are"),
    (dict(y=Y.float()), TypeError, "int32 or int64"),
    (dict(y=Y[:5]), ValueError, "labels have shape"),
    (dict(scale=0.0), ValueError, "positive and finite"),
    (dict(scale=-1.0), ValueError, "positive and finite"),
    (dict(scale=float("nan")), ValueError, "positive and finite"),
    (dict(scale=float("inf")), ValueError, "positive and finite"),
    (dict(reduction="max"), ValueError, "reduction"),
    (dict(ignore_index=1 << 63), ValueError, "64 bits"),
])
def test_cross_entropy_argument_checks(kw, err, match):
    a = dict(x=X, c=C, y=Y, scale=1.0, reduction="mean", ignore_index=-100) | kw
    with pytest.raises(err, match=match):
        fk.cluster_cross_entropy_grad(_cuda(a["x"]), _cuda(a["c"]), a["y"], scale=a["scale"],
                                      reduction=a["reduction"], ignore_index=a["ignore_index"])


@pytest.mark.parametrize("g,err", [(torch.ones(6), ValueError), (torch.ones((), dtype=torch.float16), TypeError),
                                   (2.0, TypeError)])
def test_grad_loss_checks(g, err):
    with pytest.raises(err, match="grad_loss"):
        fk.cluster_cross_entropy_grad(_cuda(X), _cuda(C), Y, grad_loss=g)


def test_the_layouts_kept_are_bounded(monkeypatch):
    from flash_kmeans import cluster_head as ch
    monkeypatch.setattr(ch, "_layouts", {})
    monkeypatch.setattr(ch, "_MOST_LAYOUTS", 5)
    for i in range(23):
        assert ch._layout(("size", i), lambda: i) == i
        assert ch._layout(("size", i), lambda: -1) == i
        assert len(ch._layouts) <= 5


XQ, CQ = torch.zeros(6, 8, dtype=torch.int8), torch.zeros(4, 8, dtype=torch.int8)
XS, CS = torch.ones(6), torch.ones(4)


@pytest.mark.parametrize("fn", [fk.int8_scores, fk.int8_assign])
@pytest.mark.parametrize("kw,err,match", [
    (dict(x=XQ), ValueError, "x_scale goes with int8"),
    (dict(x_scale=XS), ValueError, "x_scale goes with int8"),
    (dict(c=C), TypeError, "must be int8"),
    (dict(x=X.double()), TypeError, "dtype"),
    (dict(c_scale=CS.double()), TypeError, "c_scale"),
    (dict(c_scale=torch.ones(5)), ValueError, "c_scale has shape"),
    (dict(bias=torch.ones(6)), ValueError, "bias has shape"),
    (dict(x=XQ, x_scale=torch.ones(4)), ValueError, "x_scale has shape"),
    (dict(out=torch.zeros(3)), ValueError, "out must be"),
])
def test_int8_argument_checks(fn, kw, err, match):
    a = dict(x=X, c=CQ, c_scale=CS) | kw
    x, c, cs = _cuda(a.pop("x")), _cuda(a.pop("c")), a.pop("c_scale")
    with pytest.raises(err, match=match):
        fn(x, c, cs, **a)


def test_int8_output_checks():
    with pytest.raises(TypeError, match="out_dtype"):
        fk.int8_scores(_cuda(X), _cuda(CQ), CS, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="unit stride"):
        fk.int8_scores(_cuda(X), _cuda(CQ), CS, out=torch.zeros(4, 6).t())
    with pytest.raises(ValueError, match="expanded"):
        fk.int8_scores(_cuda(X), _cuda(CQ), CS, out=torch.zeros(4).expand(6, 4))
    with pytest.raises(ValueError, match="expanded"):
        fk.int8_assign(_cuda(X), _cuda(CQ), CS, out=torch.zeros(1, dtype=torch.int32).expand(6))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fk.int8_scores(X, CQ, CS)


def test_quantize_rows_refusals():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fk.quantize_rows(X)
    with pytest.raises(TypeError, match="dtype"):
        fk.quantize_rows(XQ)
    with pytest.raises(ValueError, match=r"\(N, D\)"):
        fk.quantize_rows(X[0])
    with pytest.raises(ValueError, match="at least one"):
        fk.quantize_rows(torch.zeros(3, 0))


@pytest.fixture(scope="module")
def lib():
    from flash_kmeans import _native
    return _native.load()


P = ctypes.c_void_p(1 << 20)
L3 = ctypes.c_int64 * 3
L2 = ctypes.c_int64 * 2


def _fwd(lib, x=P, c=P, y=P, dtype=1, ydtype=3, B=1, N=4, K=3, D=8, scale=1.0, reduction=1, loss=P,
         stats=None, count=P, ws=None, nbytes=0):
    return lib.fk_xent_forward(x, c, y, dtype, ydtype, B, N, K, D, L3(32, 8, 1), L3(24, 8, 1),
                               L2(4, 1), scale, -100, reduction, loss, stats, count, ws, nbytes,
                               None, None)


@pytest.mark.parametrize("kw,code", [
    (dict(K=0), 1), (dict(D=0), 1), (dict(N=-1), 1), (dict(dtype=3), 1), (dict(dtype=6), 1),
    (dict(ydtype=2), 1), (dict(scale=0.0), 1), (dict(scale=float("inf")), 1), (dict(scale=3e38), 1),
    (dict(reduction=3), 1), (dict(x=None), 1), (dict(loss=None), 1), (dict(count=None), 1),
    (dict(stats=ctypes.c_void_p(8)), 1), (dict(N=1 << 30), 2), (dict(B=2, N=(1 << 30) - 1, K=1 << 30), 2),
    (dict(), 3),                                     # no workspace
    (dict(ws=ctypes.c_void_p((1 << 20) + 16), nbytes=1 << 30), 3),
])
def test_xent_entry_point_checks(lib, kw, code):
    assert _fwd(lib, **kw) == code
    assert lib.fk_last_error()


def _bwd(lib, x=P, c=P, y=P, dtype=1, B=1, N=4, K=3, D=8, reduction=1, stats=P, count=P, g=P, gx=P, gc=P,
         gxs=(32, 8, 1), gcs=(24, 8, 1), ws=None, nbytes=0):
    return lib.fk_xent_backward(x, c, y, dtype, 3, B, N, K, D, L3(32, 8, 1), L3(24, 8, 1), L2(4, 1), 1.0,
                                -100, reduction, stats, count, g, gx, gc, gxs and L3(*gxs),
                                gcs and L3(*gcs), ws, nbytes, None, None)


def _both(lib, x=P, c=P, y=P, dtype=1, B=1, N=4, K=3, D=8, reduction=1, loss=P, g=P, gx=P, gc=P,
          gxs=(32, 8, 1), gcs=(24, 8, 1), ws=None, nbytes=0):
    return lib.fk_xent_loss_grad(x, c, y, dtype, 3, B, N, K, D, L3(32, 8, 1), L3(24, 8, 1), L2(4, 1), 1.0,
                                 -100, reduction, loss, g, gx, gc, gxs and L3(*gxs),
                                 gcs and L3(*gcs), ws, nbytes, None, None)


@pytest.mark.parametrize("fn,kw,code", [
    *((fn, kw, code) for fn in (_bwd, _both) for kw, code in [
        (dict(K=0), 1), (dict(dtype=6), 1), (dict(x=None), 1), (dict(y=None), 1),
        (dict(reduction=0, g=None), 1), (dict(gxs=None), 1), (dict(gcs=None), 1),
        (dict(gxs=(32, 1, 4)), 2), (dict(gcs=(24, 1, 3)), 2), (dict(N=1 << 30), 2),
        (dict(B=1 << 20, N=1, K=1 << 20, D=1 << 20), 2),
        (dict(), 3), (dict(ws=ctypes.c_void_p((1 << 20) + 16), nbytes=1 << 30), 3),
    ]),
    (_bwd, dict(stats=None), 1), (_bwd, dict(count=None), 1), (_bwd, dict(stats=ctypes.c_void_p(8)), 1),
    (_bwd, dict(gx=None, gc=None), 0),               # nothing wanted
    (_both, dict(gx=None, gc=None), 1), (_both, dict(loss=None), 1),
])
def test_xent_gradient_entry_point_checks(lib, fn, kw, code):
    assert fn(lib, **kw) == code


def test_xent_workspace_covers_copies_and_the_piece(lib):
    def size(dtype, D, bx, bc, N=1000, K=5000, p=P):
        return lib.fk_xent_workspace_size(p, p, dtype, 1, N, K, D, L3(N * D, D, 1), L3(K * D, D, 1),
                                          1, bx, bc)
    plain = size(1, 128, 0, 0)
    assert 0 < plain < 8 << 20
    # rows of 200 bytes are copied, padded
    assert size(1, 100, 0, 0) >= plain + 6000 * 104 * 2
    # float32: three bf16 parts of x and c
    assert size(2, 128, 0, 0) >= plain + 3 * 6000 * 128 * 2
    # backward: a copy of x and a piece of the softmax
    assert size(1, 128, 1, 1) >= 1000 * 128 * 2 + 1000 * 5000 * 2
    # and never more than a piece of a long vocabulary
    assert size(1, 128, 1, 1, N=1 << 16, K=1 << 20) < (1 << 28) + (1 << 16) * 128 * 8 + (1 << 27)
    assert lib.fk_xent_workspace_size(P, P, 1, 0, 4, 3, 8, L3(0, 8, 1), L3(24, 8, 1), 1, 0, 0) == 0


def test_int8_entry_point_checks(lib):
    def scores(x=P, c=P, sx=P, sc=P, out=P, xdt=6, odt=2, B=1, N=4, K=3, D=16, ostr=(12, 3, 1), n=0):
        return lib.fk_int8_scores(x, c, sx, sc, None, out, xdt, odt, B, N, K, D, L3(64, 16, 1),
                                  L3(48, 16, 1), L2(4, 1), L2(3, 1), None, L3(*ostr), None, n, None,
                                  None)
    assert scores(K=0) == 1 and scores(D=0) == 1 and scores(xdt=3) == 1 and scores(odt=6) == 1
    assert scores(sx=None) == 1 and scores(xdt=1) == 1 and scores(sc=None) == 1 and scores(out=None) == 1
    assert scores(D=65537) == 2 and b"overflow" in lib.fk_last_error()
    assert scores(N=1 << 30) == 2
    assert scores(B=1 << 22, N=1, K=1 << 22, D=1 << 15) == 2
    assert scores(ostr=(12, 1, 4)) == 2
    assert scores(xdt=1, sx=None) == 3              # float x needs room for its integers
    assert scores(N=0) == 0
    assert lib.fk_quantize_rows(P, 6, 1, 4, 8, L3(32, 8, 1), P, L3(32, 8, 1), P, L2(4, 1), None) == 1
    assert lib.fk_quantize_rows(P, 1, 1, 4, 8, L3(32, 8, 1), P, L3(32, 1, 4), P, L2(4, 1), None) == 2
    assert lib.fk_quantize_rows(P, 1, 1, 0, 8, L3(32, 8, 1), P, L3(32, 8, 1), P, L2(4, 1), None) == 0
    # 8-bit rows in place need no workspace, others a padded copy
    ok = lib.fk_int8_workspace_size(P, P, 6, 1, 300, 300, 128, L3(0, 128, 1), L3(0, 128, 1), 0)
    odd = lib.fk_int8_workspace_size(P, P, 6, 1, 300, 300, 100, L3(0, 100, 1), L3(0, 100, 1), 0)
    assert ok == 0 and odd >= 600 * 112


class _Unread(torch.Tensor):
    """A scalar whose value may not be fetched, as a GPU's cannot without waiting for it."""
    is_cuda = property(lambda self: True)

    def __float__(self):
        raise AssertionError("fetched")

    __int__ = __index__ = item = __float__


@pytest.mark.parametrize("fn", [fk.cluster_cross_entropy, fk.cluster_cross_entropy_grad])
@pytest.mark.parametrize("kw", [dict(scale=torch.tensor(2.0).as_subclass(_Unread)),
                                dict(ignore_index=torch.tensor(3).as_subclass(_Unread))])
def test_a_scalar_on_a_gpu_is_not_fetched(fn, kw):
    with pytest.raises(TypeError, match=next(iter(kw))):
        fn(_cuda(X), _cuda(C), Y, **kw)


@pytest.mark.parametrize("fn", [fk.cluster_cross_entropy, fk.cluster_cross_entropy_grad])
@pytest.mark.parametrize("kw,err,match", [
    (dict(scale=3.0e38), ValueError, "positive and finite"),     # times log2(e): past float32
    (dict(scale=1e39), ValueError, "positive and finite"),
    (dict(scale=1e-46), ValueError, "positive and finite"),      # 0 in float32
    (dict(ignore_index=0.5), TypeError, "ignore_index"),
    (dict(ignore_index=float("nan")), TypeError, "ignore_index"),
])
def test_values_that_the_kernels_cannot_hold(fn, kw, err, match):
    with pytest.raises(err, match=match):
        fn(_cuda(X), _cuda(C), Y, **kw)


def test_int8_points_are_still_a_type_error_in_k_means(monkeypatch):
    """8-bit integers are the cluster head's alone."""
    from flash_kmeans import _native, _ops
    from flash_kmeans.assign_euclid_triton import euclid_assign
    with pytest.raises(TypeError, match="unsupported dtype"):
        _native.dtype_code(torch.int8)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    xq, cq = _cuda(XQ[None]), _cuda(CQ[None])
    with pytest.raises(TypeError, match="unsupported dtype"):
        euclid_assign(xq, cq, _cuda(torch.ones(1, 6)))
    with pytest.raises(TypeError, match="unsupported dtype"):
        _ops.row_sqnorm(xq)


@pytest.fixture
def _no_launch(monkeypatch):
    from flash_kmeans import cluster_head as ch
    monkeypatch.setattr(ch, "_call", lambda *args: None)


@pytest.mark.parametrize("fn,out", [(fk.int8_scores, torch.zeros(6, 4)),
                                    (fk.int8_assign, torch.zeros(6, dtype=torch.int32))])
def test_a_written_out_counts_as_changed(_no_launch, fn, out):
    """What autograd saved of it is not what it holds any more."""
    w = torch.ones(out.shape, requires_grad=True)
    later = (w * out).sum()
    before = out._version
    assert fn(_cuda(X), _cuda(CQ), CS, out=out) is out
    assert out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        later.backward()


@pytest.mark.parametrize("fn,bad,good", [
    (fk.int8_scores,
     [torch.zeros(9).as_strided((6, 4), (1, 1)), torch.zeros(24).as_strided((6, 4), (3, 1)),
      torch.zeros(6, 4, requires_grad=True)],
     [torch.zeros(6, 4), torch.zeros(12, 9)[::2, 3:7], torch.zeros(1, 4).expand(1, 4),
      torch.zeros(3, 6, 4)[1]]),
    (fk.int8_assign,
     [torch.zeros(1, dtype=torch.int32).expand(6)],
     [torch.zeros(6, dtype=torch.int32), torch.zeros(12, 3, dtype=torch.int32)[::2, 1],
      torch.zeros(6, 6, dtype=torch.int32).diagonal()]),
])
def test_out_has_elements_of_its_own(_no_launch, fn, bad, good):
    for out in bad:
        with pytest.raises(ValueError, match="out must not"):
            fn(_cuda(X), _cuda(CQ), CS, out=out)
    for out in good:
        x = X[: out.shape[0]]
        assert fn(_cuda(x), _cuda(CQ), CS, out=out) is out


def test_batched_outputs_have_elements_of_their_own(_no_launch):
    xb, cb, sb = torch.randn(3, 6, 8), torch.zeros(3, 4, 8, dtype=torch.int8), torch.ones(3, 4)
    for out in (torch.zeros(3, 6, 4), torch.zeros(6, 3, 4).transpose(0, 1), torch.zeros(3, 8, 9)[:, 1:7, 2:6]):
        assert fk.int8_scores(_cuda(xb), _cuda(cb), sb, out=out) is out
    for out in (torch.zeros(60).as_strided((3, 6, 4), (8, 4, 1)), torch.zeros(90).as_strided((3, 6, 4), (4, 4, 1))):
        with pytest.raises(ValueError, match="out must not"):
            fk.int8_scores(_cuda(xb), _cuda(cb), sb, out=out)
    ids = torch.zeros(40, dtype=torch.int32).as_strided((3, 6), (5, 1))
    with pytest.raises(ValueError, match="out must not"):
        fk.int8_assign(_cuda(xb), _cuda(cb), sb, out=ids)
    with torch.no_grad():       # no graph that the writing could spoil
        out = torch.zeros(6, 4, requires_grad=True)
        assert fk.int8_scores(_cuda(X), _cuda(CQ), CS, out=out) is out


def test_a_loss_over_few_centroids_copies_no_points(lib):
    """Gathering the rows that count costs a copy of x, which few centroids do not
    give back; the backward pass copies x in any case."""
    def size(N, K, D, dtype=1, bx=0, bc=0):
        return lib.fk_xent_workspace_size(P, P, dtype, 1, N, K, D, L3(N * D, D, 1), L3(K * D, D, 1), 1, bx, bc)
    for N, K, D in ((65536, 256, 4096), (1 << 20, 64, 1024), (65536, 4096, 1024)):
        assert size(N, K, D) < N * D             # (half a copy)
        assert size(N, K, D, bx=1, bc=1) >= N * D * 2
    assert size(16384, 32768, 1024) >= 16384 * 1024 * 2
    # float32 is copied as its three parts, with or without
    assert size(65536, 256, 4096, dtype=2) >= 65536 * 4096 * 6


def test_the_error_word_is_public_and_names_every_kernel(monkeypatch, lib):
    word = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(fk.DeviceStatus, "_words", {0: word})
    fk.DeviceStatus.raise_if_set("cuda:0")
    for code, text in ((101, "outside"), (102, "pipeline wait")):
        word[0] = code
        with pytest.raises(RuntimeError, match=text) as e:
            fk.DeviceStatus.raise_if_set("cuda:0")
        assert "assignment" not in str(e.value)      # (other kernels wait too)
        assert word[0] == 0
        fk.DeviceStatus.raise_if_set("cuda:0")


def test_a_wait_that_ran_out_is_not_hidden_by_a_bad_label():
    """The word keeps the largest code: waits raise it, labels only set it while it is 0."""
    import pathlib
    csrc = pathlib.Path(fk.__file__).parent.parent / "csrc"
    assert fk._native.FK_DEV_WAIT_TIMEOUT > fk._native.FK_DEV_BAD_LABEL
    waits = (csrc / "fk_ptx.cuh").read_text()
    assert "atomicCAS(dev_status" not in waits and waits.count("atomicMax(dev_status, code)") == 2


def _negated(t):
    """The same values through memory that holds their negatives (as the imaginary
    part of a conjugate, and gradients that pass one, do)."""
    v = torch._neg_view(t.neg())
    assert v.is_neg() and torch.equal(v, t)
    return v


def _floats(p, n):
    return [ctypes.cast(p, ctypes.POINTER(ctypes.c_float))[k] for k in range(n)]


def test_negated_views_are_read_by_their_values(monkeypatch):
    """By the pointers that a call hands to the library."""
    from flash_kmeans import cluster_head as ch
    sizes, got = {}, []
    monkeypatch.setattr(ch, "_call", lambda fn, what, dev, *args: got.append(
        [_floats(args[i], n) for i, n in sizes.items()]))
    x, c, g = X.abs(), C.abs(), torch.ones(6)
    sizes |= {0: 48, 1: 32}
    fk.cluster_cross_entropy(_cuda(_negated(x)), _cuda(_negated(c)), Y)
    assert got.pop() == [x.flatten().tolist(), c.flatten().tolist()]
    sizes.clear()
    sizes[16] = 6
    fk.cluster_cross_entropy_grad(_cuda(x), _cuda(c), Y, reduction="none", grad_loss=_negated(g))
    assert got.pop() == [g.tolist()]
    sizes.clear()
    xr = _cuda(x).requires_grad_()
    loss = fk.cluster_cross_entropy(xr, _cuda(c), Y, reduction="none")
    sizes[17] = 6
    loss.backward(_negated(g))
    assert got.pop() == [g.tolist()]
    sizes.clear()
    s, b = torch.ones(4), torch.ones(4) * 2
    sizes |= {2: 6, 3: 4, 4: 4}
    fk.int8_scores(_cuda(XQ), _cuda(CQ), _negated(s), x_scale=_negated(XS), bias=_negated(b))
    assert got.pop() == [XS.tolist(), s.tolist(), b.tolist()]
    sizes.clear()
    sizes[0] = 48
    fk.int8_scores(_cuda(_negated(x)), _cuda(CQ), s)
    assert got.pop() == [x.flatten().tolist()]
    sizes.clear()
    with pytest.raises(ValueError, match="out must not"):
        fk.int8_scores(_cuda(XQ), _cuda(CQ), s, x_scale=XS, out=_negated(torch.zeros(6, 4)))


def test_negated_views_are_quantised_by_their_values(monkeypatch):
    from flash_kmeans import _native
    seen = []

    class Lib:
        def fk_quantize_rows(self, x, *args):
            seen.extend(_floats(x, 48))
            return 0

    monkeypatch.setattr(_native, "load", Lib)
    monkeypatch.setattr(_native, "stream_handle", lambda device: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    fk.quantize_rows(_cuda(_negated(X)))
    assert seen == X.flatten().tolist()
