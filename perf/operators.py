"""The operators of a cluster head: a codebook's cross entropy and its 8-bit scores.

A cluster head scores points x (N, D) against a codebook of K centroids (K, D),
z[n, k] = x[n] . c[k], as the cosine and dot-product assignments of this
package do.  Four operators are listed here:

loss       the softmax cross entropy of scale * z against cluster ids, without
           keeping z
loss_grad  the same with its gradients by x and by the centroids
scores     z itself from 8-bit integers, one scale per point and per centroid
assign     argmax_k of those scores, without keeping them

Every case is a dict of plain values; sizes are B batches (0: unbatched), N
points, K centroids, D features.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}
IGNORE = -100


def _case(name, op, **kw):
    base = {"op": op, "B": 0, "shared": False, "dtype": "bf16"}
    if op in ("loss", "loss_grad"):
        base |= {"scale": 10.0, "ignored": 0.0, "reduction": "mean", "ids": "int32",
                 "autograd": False}
    else:
        base |= {"x": "bf16", "bias": False}
    return ({"name": name} if name else {}) | base | kw


def listed():
    return [
        # a few frames of a stream scored against a codebook: latency
        _case("loss_few", "loss", N=5, K=1000, D=128),
        # evaluation over a large vocabulary, one loss per token, part of them padding
        _case("loss_eval", "loss", N=4096, K=32768, D=1024, dtype="fp16", ignored=0.15,
              reduction="none", ids="int64"),
        # several small heads trained side by side, no size a multiple of anything
        _case("grad_heads", "loss_grad", B=3, N=77, K=1031, D=100, dtype="fp32", ignored=0.1),
        # a head on k-means labels of a float32 embedding
        _case("grad_fp32", "loss_grad", N=8192, K=1024, D=512, dtype="fp32"),
        # a training step of a language model's head, padding ignored
        _case("grad_step", "loss_grad", N=16384, K=32768, D=1024, ignored=0.15, ids="int64",
              autograd=True),
        # sequences that share one codebook, small features: the softmax outweighs the products
        _case("grad_narrow", "loss_grad", B=4, N=8111, K=8192, D=128, shared=True, dtype="fp16",
              reduction="sum"),
        # the largest vocabulary
        _case("grad_vocab", "loss_grad", N=8192, K=131072, D=2048, ids="int64", autograd=True),
        # one token answered from an 8-bit head: the codebook is read once
        _case("scores_token", "scores", N=1, K=32768, D=4096),
        # odd sizes, points quantised before
        _case("scores_odd", "scores", B=2, N=333, K=1031, D=97, x="int8", bias=True, dtype="fp32"),
        # a prompt's tokens against a codebook
        _case("scores_prompt", "scores", N=4096, K=8192, D=4096, x="fp16", dtype="fp16"),
        # nearest centroids of quantised points, a codebook for each batch
        _case("assign_batch", "assign", B=8, N=75600, K=1000, D=128, x="int8", bias=True),
        # long feature rows quantised and assigned in one call
        _case("assign_wide", "assign", N=65537, K=500, D=1024, x="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "loss_grad", "loss_grad", "scores", "assign"])
    B = rng.choice([0, 0, 1, 2, 5])
    shared = B > 0 and rng.random() < 0.5
    while True:
        N, K, D = _log(rng, 1, 65536), _log(rng, 2, 131072), _log(rng, 8, 4096)
        if rng.random() < 0.5:
            D = max(16, D // 16 * 16)
        rows = max(B, 1) * N
        if rows * K * D <= 8192 * 131072 * 2048 // 16 and rows * K <= 1 << 30:
            break
    if op in ("loss", "loss_grad"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _case(None, op, B=B, N=N, K=K, D=D, shared=shared, dtype=dtype,
                     scale=rng.choice([1.0, 4.0, 8.0]),
                     ignored=rng.choice([0.0, 0.1, 0.5]),
                     reduction=rng.choice(["mean", "sum", "none"]) if op == "loss"
                     # a mean's float16 gradients underflow: such a step scales its loss
                     else "sum" if dtype == "fp16" else rng.choice(["mean", "sum"]),
                     ids=rng.choice(["int32", "int64"]),
                     autograd=op == "loss_grad" and rng.random() < 0.5)
    return _case(None, op, B=B, N=N, K=K, D=D, shared=shared,
                 x=rng.choice(["int8", "bf16", "fp16", "fp32"]), bias=rng.random() < 0.4,
                 dtype=rng.choice(["bf16", "fp16", "fp32"]) if op == "scores" else "fp32")


def _quantised(v):
    """Rows of float32 as 8-bit integers in [-127, 127] and one scale each."""
    most = v.abs().amax(-1, keepdim=True)
    # a quotient of two tensors is rounded once; one with a number is not
    top = torch.full_like(most, 127.0)
    inv = torch.where(most > 0, top / most, 0.0)
    return (v * inv).round(), (most / top).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    B, N, K, D = max(case["B"], 1), case["N"], case["K"], case["D"]
    Bc = 1 if case["shared"] or case["B"] == 0 else B

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)

    # unit-length codebook rows on average; points scatter about their cluster's row
    c = randn(Bc, K, D) / math.sqrt(D)
    ids = torch.randint(0, K, (B, N), device="cuda", generator=g)
    batch = torch.arange(B, device="cuda").clamp(max=Bc - 1)[:, None]
    x = randn(B, N, D).mul_(0.6 / math.sqrt(D)).add_(c[batch, ids])
    s = {"case": case}
    if case["op"] in ("loss", "loss_grad"):
        t = DTYPES[case["dtype"]]
        if case["ignored"]:
            drop = torch.rand(B, N, device="cuda", generator=g) < case["ignored"]
            ids = ids.masked_fill(drop, IGNORE)
        s |= {"x": x.to(t), "c": c.to(t), "ids": ids.to(getattr(torch, case["ids"]))}
    else:
        # the codebook is quantised once, when it is trained
        cq, cs = _quantised(c)
        s |= {"c": cq.to(torch.int8), "c_scale": cs}
        if case["bias"]:  # -|c|^2 / 2 turns the largest score into the nearest centroid
            s["bias"] = c.square().sum(-1) * -0.5
        if case["x"] == "int8":
            xq, xs = _quantised(x)
            s |= {"x": xq.to(torch.int8), "x_scale": xs}
        else:
            s["x"] = x.to(DTYPES[case["x"]])
    if case["B"] == 0:
        s |= {k: v[0] for k, v in s.items() if k != "case"}
    elif case["shared"]:
        s |= {k: s[k][0] for k in ("c", "c_scale", "bias") if k in s}
    if case["op"] == "loss_grad" and case["autograd"]:
        s["x"].requires_grad_()
        s["c"].requires_grad_()
    return s


def _transposed(c):
    return c.transpose(-1, -2)


def _plain_loss(s, grads):
    case = s["case"]
    x, c, ids = s["x"].detach().float(), s["c"].detach().float(), s["ids"].long()
    logits = (x @ _transposed(c)).mul_(case["scale"])
    keep = ids != IGNORE
    at = ids.clamp(min=0)[..., None]
    most = logits.amax(-1, keepdim=True)
    # the label's own term stays out of the sum: a well-fitted row's loss is
    # log1p of what the others add, and would be lost beside a 1
    d = logits.sub_(logits.gather(-1, at)).scatter_(-1, at, -math.inf)
    most = d.amax(-1, keepdim=True).clamp(min=0.0)
    e = d.sub_(most).exp_()
    others = e.sum(-1, keepdim=True)
    total = others + (-most).exp()
    rows = torch.where(most > 0, most + total.log(), others.log1p()).squeeze(-1)
    rows = torch.where(keep, rows, 0.0)
    count = keep.sum() if case["reduction"] == "mean" else 1
    loss = rows if case["reduction"] == "none" else rows.sum() / count
    if not grads:
        return loss
    p = e.scatter_(-1, at, -others).div_(total)
    p.mul_(torch.where(keep, case["scale"] / count, 0.0)[..., None])
    gx = p @ c
    if c.dim() < x.dim():  # one codebook for all batches
        p, x = p.flatten(0, 1), x.flatten(0, 1)
    gc = _transposed(p) @ x
    return {"loss": loss, "x": gx.to(s["x"].dtype), "centroids": gc.to(s["c"].dtype)}


def _plain_scores(s):
    x, xs = (s["x"], s["x_scale"]) if "x_scale" in s else _quantised(s["x"].float())
    # the integer sums pass 24 bits from 1040 features on
    t = torch.float32 if x.shape[-1] <= 1040 else torch.float64
    z = (x.to(t) @ _transposed(s["c"]).to(t)).float()
    z = z.mul_(xs[..., None]).mul_(s["c_scale"][..., None, :])
    return z.add_(s["bias"][..., None, :]) if "bias" in s else z


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        path = os.path.abspath("flash-kmeans_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import flash_kmeans as fk

        if op in ("loss", "loss_grad"):
            kw = {"scale": case["scale"], "ignore_index": IGNORE, "reduction": case["reduction"]}
            args = (state["x"], state["c"], state["ids"])
            if op == "loss":
                return fk.cluster_cross_entropy(*args, **kw)
            if case["autograd"]:
                loss = fk.cluster_cross_entropy(*args, **kw)
                gx, gc = torch.autograd.grad(loss, args[:2])
                loss = loss.detach()
            else:
                loss, gx, gc = fk.cluster_cross_entropy_grad(*args, **kw)
            return {"loss": loss, "x": gx, "centroids": gc}
        kw = {"x_scale": state.get("x_scale"), "bias": state.get("bias")}
        if op == "scores":
            kw["out_dtype"] = DTYPES[case["dtype"]]
            return fk.int8_scores(state["x"], state["c"], state["c_scale"], **kw)
        return fk.int8_assign(state["x"], state["c"], state["c_scale"], **kw)
    if op in ("loss", "loss_grad"):
        return _plain_loss(state, op == "loss_grad")
    z = _plain_scores(state)
    if op == "scores":
        return z.to(DTYPES[case["dtype"]])
    # the lowest index among equal scores
    k = torch.arange(z.shape[-1], device=z.device, dtype=torch.int32)
    return torch.where(z == z.amax(-1, keepdim=True), k, z.shape[-1]).amin(-1).int()


def work(case):
    B, N, K, D = max(case["B"], 1), case["N"], case["K"], case["D"]
    rows, cents = B * N, K * (1 if case["shared"] else B)
    if case["op"] in ("loss", "loss_grad"):
        e = BYTES[case["dtype"]]
        used = rows * (1.0 - case["ignored"])  # an ignored row needs no score
        read = (used + cents) * D * e + rows * (4 if case["ids"] == "int32" else 8)
        if case["op"] == "loss":
            return {"bytes": read + (rows * 4 if case["reduction"] == "none" else 4),
                    "flops": 2.0 * used * K * D}
        return {"bytes": read + (rows + cents) * D * e + 4, "flops": 6.0 * used * K * D}
    read = rows * D * BYTES[case["x"]] + cents * (D + 4)
    read += rows * 4 if case["x"] == "int8" else 0
    read += cents * 4 if case["bias"] else 0
    out = rows * K * BYTES[case["dtype"]] if case["op"] == "scores" else rows * 4
    return {"bytes": float(read + out), "flops": 2.0 * rows * K * D}


def exact(case, seed):
    """The definitions in float64, a slab of rows at a time."""
    if case["op"] == "assign":
        return None
    s = prepare(case, seed)
    B = max(case["B"], 1)
    wide = {k: v.detach().double() for k, v in s.items() if k in ("x", "c", "c_scale", "x_scale",
                                                                  "bias")}
    if case["B"] == 0:
        wide = {k: v[None] for k, v in wide.items()}
    elif case["shared"]:
        wide |= {k: wide[k][None] for k in ("c", "c_scale", "bias") if k in wide}
    slab = max(1, (1 << 28) // case["K"])
    x, c = wide["x"], wide["c"]
    if case["op"] == "scores":
        out = torch.empty(B, case["N"], case["K"], dtype=torch.float64, device="cuda")
        for b in range(B):
            bc = min(b, c.shape[0] - 1)
            xb = x[b]
            if "x_scale" in wide:
                xs = wide["x_scale"][b]
            else:  # what 8 bits hold goes by the 32-bit quotient that places it
                v = xb.float()
                top = v.abs().max(-1).values.double()
                xs = (top / 127.0).float().double()
                by = torch.nan_to_num(127.0 / top, posinf=0.0).float()
                xb = torch.round(v * by[:, None]).double()
            out[b] = torch.einsum("nd,kd->nk", xb, c[bc]) * xs[:, None] * wide["c_scale"][bc]
            if "bias" in wide:
                out[b] += wide["bias"][bc]
        return out[0] if case["B"] == 0 else out
    ids = s["ids"].long().view(B, -1)
    losses = torch.zeros(B, case["N"], dtype=torch.float64, device="cuda")
    gx, gc = torch.zeros_like(x), torch.zeros_like(c)
    for b in range(B):
        bc = min(b, c.shape[0] - 1)
        for lo in range(0, case["N"], slab):
            rows = torch.nonzero(ids[b, lo:lo + slab] != IGNORE).squeeze(1) + lo
            y = ids[b, rows]
            logp = torch.log_softmax(case["scale"] * torch.einsum("nd,kd->nk", x[b, rows], c[bc]), 1)
            here = torch.arange(len(rows), device="cuda")
            losses[b, rows] = -logp[here, y]
            if case["op"] == "loss_grad":
                d = logp.exp_()
                d[here, y] -= 1.0
                gx[b, rows] = case["scale"] * torch.einsum("nk,kd->nd", d, c[bc])
                gc[bc] += case["scale"] * torch.einsum("nk,nd->kd", d, x[b, rows])
    count = int((ids != IGNORE).sum()) if case["reduction"] == "mean" else 1
    # a mean over no row is 0 / 0; ignored rows have no gradient all the same
    loss = losses if case["reduction"] == "none" else losses.sum() / torch.tensor(
        float(count), dtype=torch.float64, device="cuda")
    if case["op"] == "loss":
        return loss[0] if loss.dim() and case["B"] == 0 else loss
    gx, gc = gx / max(count, 1), gc / max(count, 1)
    if case["B"] == 0:
        gx, gc = gx[0], gc[0]
    elif case["shared"]:
        gc = gc[0]
    return {"loss": loss, "x": gx, "centroids": gc}
