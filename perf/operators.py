"""The measured cases of the device operators for leaf-wise linear models.

Three operators, each beside a plain form made of elementary torch operations:
the softmax cross entropy of a linear head over many classes (evaluation, and
training with both gradients), the products grouped by leaf (forward, and both
gradients), and the global norm of many gradients with clipping.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ops():
    """The framework's operators (its package lies one folder below the root)."""
    where = os.path.join(ROOT, "bsscl-gbm_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    from bsscl_gbm_b200 import linear
    return linear


def listed():
    return [
        # one row scored against a large class set: the reply to one request, bound by reading the weights once
        {"name": "xent_eval_one_row", "op": "xent", "n": 1, "d": 1024, "v": 32768, "type": "bf16", "ignored": 0.0},
        # validation loss of a batch on a large class set
        {"name": "xent_eval_batch", "op": "xent", "n": 8192, "d": 1024, "v": 32768, "type": "f16", "ignored": 0.1},
        # a training step on a small table: 100 features, an odd number of classes and rows
        {"name": "xent_train_small_odd", "op": "xent_train", "n": 999, "d": 100, "v": 1501, "type": "bf16", "ignored": 0.05},
        # an ordinary training step, a third of the rows without a label
        {"name": "xent_train_ordinary", "op": "xent_train", "n": 4096, "d": 512, "v": 16384, "type": "f16", "ignored": 0.33},
        # the largest training step: long batch, wide features, odd class count
        {"name": "xent_train_large", "op": "xent_train", "n": 16384, "d": 1024, "v": 50001, "type": "bf16", "ignored": 0.0},
        # a few rows answered by the linear models of 63 leaves: bound by reading the weights that are hit
        {"name": "leaf_serve", "op": "leaf", "t": 64, "e": 63, "din": 1024, "dout": 1024, "type": "bf16", "spread": 0.5},
        # a whole table through its leaves' linear models
        {"name": "leaf_forward_large", "op": "leaf", "t": 262144, "e": 63, "din": 1024, "dout": 1024, "type": "bf16", "spread": 0.5},
        # gradients on a small table: 10,000 rows, 31 leaves, 100 features, odd output width
        {"name": "leaf_train_small_odd", "op": "leaf_train", "t": 10000, "e": 31, "din": 100, "dout": 61, "type": "f16", "spread": 1.0},
        # gradients of an ordinary step
        {"name": "leaf_train_large", "op": "leaf_train", "t": 131072, "e": 63, "din": 1024, "dout": 1024, "type": "bf16", "spread": 0.5},
        # the gradients of one small model
        {"name": "clip_small", "op": "clip", "tensors": 5, "total": 20000, "type": "f32", "limit": 1.0},
        # many ragged bf16 gradients
        {"name": "clip_many_ragged", "op": "clip", "tensors": 300, "total": 30000001, "type": "bf16", "limit": 1.0},
        # the gradients of a large model, more than the caches hold
        {"name": "clip_large", "op": "clip", "tensors": 64, "total": 400000000, "type": "f32", "limit": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "xent_train", "xent_train", "leaf", "leaf_train", "clip"])
    kind = rng.choice(["bf16", "f16"])
    if op in ("xent", "xent_train"):
        while True:
            n, d, v = _log(rng, 1, 16384), _log(rng, 16, 2048), _log(rng, 2, 65536)
            if rng.random() < 0.5:
                d = max(16, d // 64 * 64)
            if n * d * v <= 16384 * 1024 * 50001:
                return {"op": op, "n": n, "d": d, "v": v, "type": kind, "ignored": rng.choice([0.0, 0.1, 0.5])}
    if op in ("leaf", "leaf_train"):
        while True:
            t, e, din, dout = _log(rng, 1, 262144), _log(rng, 1, 256), _log(rng, 8, 2048), _log(rng, 8, 2048)
            if rng.random() < 0.5:
                din, dout = max(8, din // 64 * 64), max(8, dout // 64 * 64)
            # the plain form pads every leaf to the largest
            if t * din * dout <= 131072 * 1024 * 1024 and e * din * dout <= 1 << 28:
                return {"op": op, "t": t, "e": e, "din": din, "dout": dout, "type": kind, "spread": rng.choice([0.0, 0.5, 1.0])}
    return {"op": "clip", "tensors": _log(rng, 1, 400), "total": _log(rng, 1000, 400000000), "type": rng.choice(["f32", "bf16", "f16"]),
            "limit": rng.choice([0.5, 1.0, 1e9])}


def _counts(seed, t, e, spread):
    """Rows of each leaf: uneven shares (some leaves may be empty), t rows in all."""
    r = random.Random(seed)
    share = [math.exp(r.gauss(0.0, spread)) for _ in range(e)]
    edge, at, total = [0], 0.0, sum(share)
    for s in share:
        at += s
        edge.append(min(t, int(round(t * at / total))))
    edge[-1] = t
    return [edge[i + 1] - edge[i] for i in range(e)]


def _sizes(count, total):
    """Element counts of a model's gradients: uneven, each at least 1, the same for every batch."""
    r = random.Random(count)
    share = [math.exp(r.gauss(0.0, 1.5)) for _ in range(count)]
    whole = sum(share)
    return [max(1, int(total * s / whole)) for s in share]


def _flat(sizes, dtype):
    """A zeroed buffer, and its views of these sizes, each on a 64-element boundary."""
    start = [0]
    for n in sizes:
        start.append(start[-1] + -(-n // 64) * 64)
    flat = torch.zeros(start[-1], dtype=dtype, device="cuda")
    return flat, [flat[a:a + n] for a, n in zip(start, sizes)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = TYPES[case["type"]], case["op"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    state = {"op": op}
    if op in ("xent", "xent_train"):
        n, d, v = case["n"], case["d"], case["v"]
        state["x"] = normal(n, d)
        # logits of standard deviation 2: a model some way into its training
        state["w"] = normal(v, d, scale=2.0 / math.sqrt(d))
        target = torch.randint(0, v, (n,), generator=g, device="cuda")
        gone = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        gone[0] = False
        state["target"] = torch.where(gone, -1, target)
        # the weights of the rows (class weights differ from row to row)
        state["grad_loss"] = 0.5 + torch.rand(n, generator=g, device="cuda")
    elif op in ("leaf", "leaf_train"):
        t, e, din, dout = case["t"], case["e"], case["din"], case["dout"]
        counts = _counts(seed, t, e, case["spread"])
        c = torch.tensor(counts, dtype=torch.int64)
        state["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), c.cumsum(0)]).to(torch.int32).cuda()
        state["most"] = max(counts)
        state["x"] = normal(t, din)
        state["w"] = normal(e, dout, din, scale=1.0 / math.sqrt(din))
        if op == "leaf_train":
            state["dy"] = normal(t, dout)
    else:
        sizes = _sizes(case["tensors"], case["total"])
        state["grads"] = [normal(s, scale=0.02) for s in sizes]
        # the clipped gradients go to places of one buffer, as an exchange between ranks takes them
        state["flat"], state["outs"] = _flat(sizes, dt)
        state["limit"] = case["limit"]
        if own:  # the handle that a training loop makes once for its gradients
            state["clip"] = _ops().GradClip(state["grads"], out=state["outs"])
    return state


def _xent_plain(s):
    logits = s["x"].float() @ s["w"].float().T
    has = s["target"] >= 0
    at = s["target"].clamp(min=0)[:, None]
    top = logits.max(1, keepdim=True).values
    e = (logits - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    loss = torch.where(has, (lse - logits.gather(1, at))[:, 0], 0.0)
    return loss, lse[:, 0], e, total, has, at


def _xent_train_plain(s):
    loss, _, e, total, has, at = _xent_plain(s)
    p = e / total
    p.scatter_add_(1, at, torch.full_like(p[:, :1], -1.0))
    p *= torch.where(has, s["grad_loss"], 0.0)[:, None]
    dx = p @ s["w"].float()
    dw = p.T @ s["x"].float()
    return loss, dx.to(s["x"].dtype), dw.to(s["w"].dtype)


def _places(s):
    """Leaf of each row, and its place among the leaf's rows."""
    o = s["offsets"].long()
    row = torch.arange(s["x"].shape[0], device="cuda")
    leaf = torch.searchsorted(o, row, right=True) - 1
    return leaf, row - o[leaf]


def _padded(v, leaf, at, e, most):
    out = torch.zeros(e, most, v.shape[1], device="cuda")
    out[leaf, at] = v.float()
    return out


def _leaf_plain(s):
    leaf, at = _places(s)
    x = _padded(s["x"], leaf, at, s["w"].shape[0], s["most"])
    return torch.bmm(x, s["w"].float().transpose(1, 2))[leaf, at].to(s["x"].dtype)


def _leaf_train_plain(s):
    leaf, at = _places(s)
    x = _padded(s["x"], leaf, at, s["w"].shape[0], s["most"])
    dy = _padded(s["dy"], leaf, at, s["w"].shape[0], s["most"])
    dx = torch.bmm(dy, s["w"].float())[leaf, at]
    dw = torch.bmm(dy.transpose(1, 2), x)
    return dx.to(s["x"].dtype), dw.to(s["w"].dtype)


def _clip_plain(s):
    # 64-bit sums: the squares of a long gradient
    parts = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    norm = parts.sum().sqrt()
    scale = (s["limit"] / (norm + 1e-6)).clamp(max=1.0).float()
    [o.copy_(g.float() * scale) for g, o in zip(s["grads"], s["outs"])]
    return norm.float(), s["flat"]


def run(s):
    op = s["op"]
    if not own:
        if op == "xent":
            return _xent_plain(s)[:2]
        if op == "xent_train":
            return _xent_train_plain(s)
        if op == "leaf":
            return _leaf_plain(s)
        if op == "leaf_train":
            return _leaf_train_plain(s)
        return _clip_plain(s)
    ops = _ops()
    if op == "xent":
        return ops.softmax_xent(s["x"], s["w"], s["target"])
    if op == "xent_train":
        loss, lse = ops.softmax_xent(s["x"], s["w"], s["target"])
        return (loss,) + ops.softmax_xent_grad(s["x"], s["w"], s["target"], lse, s["grad_loss"])
    if op == "leaf":
        return ops.leaf_linear(s["x"], s["w"], s["offsets"])
    if op == "leaf_train":
        return ops.leaf_linear_grad(s["x"], s["w"], s["offsets"], s["dy"])
    return s["clip"].clip(s["limit"]), s["flat"]


def work(case):
    op = case["op"]
    if op in ("xent", "xent_train"):
        n, d, v = case["n"], case["d"], case["v"]
        if op == "xent":
            return {"bytes": 2 * d * (n + v) + 16 * n, "flops": 2 * n * d * v}
        return {"bytes": 4 * d * (n + v) + 20 * n, "flops": 6 * n * d * v}
    if op in ("leaf", "leaf_train"):
        t, din, dout = case["t"], case["din"], case["dout"]
        hit = min(case["e"], t)  # a leaf without rows needs no weights
        if op == "leaf":
            return {"bytes": 2 * (t * (din + dout) + hit * din * dout), "flops": 2 * t * din * dout}
        return {"bytes": 2 * (t * (2 * din + dout) + (hit + case["e"]) * din * dout), "flops": 4 * t * din * dout}
    size = 4 if case["type"] == "f32" else 2
    return {"bytes": 2 * size * case["total"], "flops": 3 * case["total"]}


def exact(case, seed):
    """The operators from their definitions in 64 bits, a block of rows, a leaf or a gradient at a time."""
    s = prepare(case, seed)
    op = case["op"]
    if op in ("xent", "xent_train"):
        x, w = s["x"].double(), s["w"].double()
        n, v = x.shape[0], w.shape[0]
        loss, norm = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(2))
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        step = max(1, (1 << 27) // v)
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            y = s["target"][lo:hi]
            z = x[lo:hi] @ w.T
            norm[lo:hi] = torch.logsumexp(z, 1)
            rows = (y >= 0).nonzero()[:, 0]
            if not len(rows):
                continue
            z, lse = z[rows], norm[lo:hi][rows]
            loss[lo + rows] = lse - z[torch.arange(len(rows), device="cuda"), y[rows]]
            if op == "xent":
                continue
            z = torch.exp(z - lse[:, None])
            z[torch.arange(len(rows), device="cuda"), y[rows]] -= 1.0
            z = z * s["grad_loss"][lo:hi][rows].double()[:, None]
            dx[lo + rows] = z @ w
            dw += z.T @ x[lo:hi][rows]
        return (loss, norm) if op == "xent" else (loss, dx, dw)
    if op in ("leaf", "leaf_train"):
        edge = s["offsets"].tolist()
        y = torch.zeros(case["t"], case["dout"] if op == "leaf" else case["din"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(case["e"], case["dout"], case["din"], dtype=torch.float64, device="cuda") if op == "leaf_train" else None
        for k in range(case["e"]):
            lo, hi = edge[k], edge[k + 1]
            if op == "leaf":
                y[lo:hi] = s["x"][lo:hi].double() @ s["w"][k].double().T
            else:
                y[lo:hi] = s["dy"][lo:hi].double() @ s["w"][k].double()
                dw[k] = s["dy"][lo:hi].double().T @ s["x"][lo:hi].double()
        return y if op == "leaf" else (y, dw)
    norm = torch.stack([(g.double() * g.double()).sum() for g in s["grads"]]).sum().sqrt()
    scale = torch.clamp(case["limit"] / (norm + 1e-6), max=1.0)
    flat, outs = _flat([len(g) for g in s["grads"]], torch.float64)
    for g, o in zip(s["grads"], outs):
        o.copy_(g.double() * scale)
    return norm, flat
