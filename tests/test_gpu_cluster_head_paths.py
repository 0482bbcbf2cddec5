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
