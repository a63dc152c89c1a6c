"""Class losses over voxel features and scores: the cases they are measured at.

Two operators, each with its gradient:

* "linear": ``losses.linear_cross_entropy`` - softmax cross entropy of
  ``features @ weight.T`` against labels, without the [rows, classes] scores
  in memory;
* "scores": ``losses.softmax_cross_entropy`` - the same loss of scores that
  are in memory (the channels of a volume, or the output of a caller's head).

``run`` computes them in plain torch operations in float32, or through the
package where ``own`` is true. ``exact`` evaluates the definition in float64.
"""
from __future__ import annotations

import math

import torch

own = False

IGNORE = -100
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16,
          "float16": torch.float16}

# A case: op, rows (leading shape as "ZxYxX" or a plain count), V classes,
# D channels (linear), dtype, train (gradients too), ignored (share of rows
# without a label), smoothing, softcap, z_loss, reduction, scale (the upstream
# gradient: a loss scale, or the size of per-row weights with "none").
_BASE = dict(train=True, ignored=0.0, smoothing=0.0, softcap=0.0, z_loss=0.0,
             reduction="mean", scale=1.0)


def _case(name, op, rows, V, D, dtype, **kw):
    return {"name": name, "op": op, "rows": rows, "V": V, "D": D,
            "dtype": dtype, **_BASE, **kw}


def listed():
    return [
        # serving: the log-probability of one token over a vocabulary; the
        # table is read once, latency counts
        _case("token_score", "linear", "1", 32768, 2048, "bfloat16",
              train=False, reduction="none"),
        # the framework's 256^3 volume with 4 channels decoded into 20 voxel
        # classes by a learned table, a tenth of the voxels unlabelled
        _case("voxel_classes", "linear", "256x256x256", 20, 4, "float32",
              ignored=0.1),
        # a smaller feature volume of odd size with more channels, float32
        _case("feature_volume", "linear", "40x48x37", 203, 32, "float32",
              ignored=0.25),
        # a small ragged batch with per-row weights and every option, odd
        # sizes that no alignment suits
        _case("train_odd", "linear", "1001", 5003, 257, "bfloat16",
              ignored=0.2, smoothing=0.1, softcap=30.0, reduction="none"),
        # half precision under a loss scale
        _case("train_half", "linear", "2048", 32000, 1024, "float16",
              z_loss=1e-4, scale=4096.0),
        # scoring a padded batch of rows without gradients
        _case("score_rows", "linear", "512", 131072, 1024, "bfloat16",
              train=False, ignored=0.3, reduction="none"),
        # the largest training step: a long batch over a large vocabulary
        _case("train_large", "linear", "8192", 131072, 4096, "bfloat16"),
        # the voxelizer's own output as class scores, four classes
        _case("volume_scores", "scores", "256x256x256", 4, 0, "float32",
              ignored=0.1),
        # a class head's output for a volume, class count of no alignment
        _case("class_volume", "scores", "64x128x96", 37, 0, "bfloat16",
              ignored=0.1, smoothing=0.05),
        # a handful of rows: latency
        _case("few_rows", "scores", "7", 1003, 0, "float32"),
        # a language model head's output, odd vocabulary, capped
        _case("vocab_odd", "scores", "1021", 50021, 0, "float16",
              smoothing=0.1, softcap=30.0, scale=4096.0),
        # the same at the size of a long batch
        _case("vocab_large", "scores", "4096", 131072, 0, "bfloat16",
              ignored=0.1, z_loss=1e-4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "scores"])
    dtype = rng.choice(list(DTYPES))
    V = _log_int(rng, 2, 131072)
    if op == "linear":
        D = _log_int(rng, 1, 4096)
        # at most a quarter of the largest listed case's products, and at
        # most 2^31 scores for the plain form to hold
        top = min(2 ** 31 // V, 2 ** 40 // (V * D), 2 ** 29 // D, 2 ** 23)
    else:
        D = 0
        top = min(2 ** 29 // V, 2 ** 23)
    rows = _log_int(rng, 1, max(1, top))
    train = rng.random() < 0.75
    reduction = rng.choice(["mean", "mean", "sum", "none"])
    return {
        "op": op, "rows": str(rows), "V": V, "D": D, "dtype": dtype,
        "train": train, "ignored": rng.choice([0.0, 0.1, 0.5]),
        "smoothing": rng.choice([0.0, 0.0, 0.1]),
        "softcap": rng.choice([0.0, 0.0, 30.0]),
        "z_loss": rng.choice([0.0, 0.0, 1e-4]), "reduction": reduction,
        "scale": 4096.0 if dtype == "float16" else 1.0,
    }


def _shape(case):
    return tuple(int(v) for v in case["rows"].split("x"))


def _inputs(case, seed):
    """Features with scores of standard deviation about 2 in which the
    label's class stands out, as in the middle of a training run."""
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    shape, V, D = _shape(case), case["V"], case["D"]
    n = math.prod(shape)
    dtype = DTYPES[case["dtype"]]
    labels = torch.randint(0, V, (n,), generator=g, device=dev)
    if case["op"] == "linear":
        std = 2.0 / math.sqrt(D)
        weight = (std * torch.randn((V, D), generator=g, device=dev)).to(dtype)
        features = torch.randn((n, D), generator=g, device=dev)
        features += weight[labels].float()
        inputs = (features.to(dtype).view(*shape, D), weight)
    else:
        scores = 2.0 * torch.randn((n, V), generator=g, device=dev)
        scores[torch.arange(n, device=dev), labels] += 4.0
        inputs = (scores.to(dtype).view(*shape, V),)
    if case["ignored"] > 0:
        drop = torch.rand((n,), generator=g, device=dev) < case["ignored"]
        labels = labels.masked_fill(drop, IGNORE)
    upstream = None
    if case["train"]:
        if case["reduction"] == "none":
            upstream = case["scale"] / n * (
                0.5 + torch.rand((n,), generator=g, device=dev))
            upstream = upstream.view(shape)
        else:
            upstream = torch.full((), case["scale"], device=dev)
    return inputs, labels.view(shape), upstream


def prepare(case, seed):
    inputs, labels, upstream = _inputs(case, seed)
    if case["train"] and own:
        inputs = tuple(t.requires_grad_(True) for t in inputs)
    return {"case": case, "inputs": inputs, "labels": labels,
            "upstream": upstream}


def _run_own(state):
    from gs_voxelizer_b200 import losses
    case = state["case"]
    fn = (losses.linear_cross_entropy if case["op"] == "linear"
          else losses.softmax_cross_entropy)
    loss = fn(*state["inputs"], state["labels"], ignore_index=IGNORE,
              label_smoothing=case["smoothing"], softcap=case["softcap"],
              z_loss=case["z_loss"], reduction=case["reduction"])
    if not case["train"]:
        return (loss,)
    grads = torch.autograd.grad(loss, state["inputs"], state["upstream"])
    return (loss.detach(), *grads)


def _run_plain(state):
    case, inputs = state["case"], state["inputs"]
    V, eps, cap, zeta = case["V"], case["smoothing"], case["softcap"], case["z_loss"]
    shape = state["labels"].shape
    y = state["labels"].reshape(-1)
    keep = y != IGNORE
    at = y.clamp_min(0).unsqueeze(1)
    if case["op"] == "linear":
        x = inputs[0].reshape(-1, case["D"]).float()
        w = inputs[1].float()
        z = x @ w.t()
    else:
        z = inputs[0].reshape(-1, V).float()
    if cap > 0:
        z = cap * torch.tanh(z / cap)
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    lse = (torch.log(total) + top).squeeze(1)
    rows = lse - (1.0 - eps) * z.gather(1, at).squeeze(1)
    if eps > 0:
        rows = rows - eps * z.mean(dim=1)
    if zeta > 0:
        rows = rows + zeta * lse * lse
    rows = torch.where(keep, rows, torch.zeros_like(rows))
    count = keep.sum().clamp_min(1).float()
    if case["reduction"] == "none":
        loss = rows.view(shape)
    elif case["reduction"] == "sum":
        loss = rows.sum()
    else:
        loss = rows.sum() / count
    if not case["train"]:
        return (loss,)
    g = state["upstream"].reshape(-1).float()
    if case["reduction"] == "mean":
        g = g / count
    g = torch.where(keep, g.expand(y.shape), torch.zeros_like(lse)).unsqueeze(1)
    p /= total
    if zeta > 0:
        p *= (1.0 + 2.0 * zeta * lse).unsqueeze(1)
    if eps > 0:
        p -= eps / V
    p.scatter_add_(1, at, torch.full_like(lse, eps - 1.0).unsqueeze(1))
    p *= g
    if cap > 0:
        p *= 1.0 - (z / cap) ** 2
    if case["op"] == "linear":
        return (loss, (p @ w).to(inputs[0].dtype).view_as(inputs[0]),
                (p.t() @ x).to(inputs[1].dtype))
    return (loss, p.to(inputs[0].dtype).view_as(inputs[0]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    n, V, D = math.prod(_shape(case)), case["V"], case["D"]
    b = 4 if case["dtype"] == "float32" else 2
    kept = n * (1.0 - case["ignored"])
    out = 4 * n if case["reduction"] == "none" else 4
    passes = 2 if case["train"] else 1  # inputs in, gradients out
    if case["op"] == "linear":
        return {"bytes": 8 * n + out + passes * b * (n * D + V * D),
                "flops": (6 if case["train"] else 2) * kept * V * D}
    return {"bytes": 8 * n + out + passes * b * n * V,
            "flops": (6 if case["train"] else 4) * kept * V}


def exact(case, seed):
    inputs, labels, upstream = _inputs(case, seed)
    V, D = case["V"], case["D"]
    y = labels.reshape(-1)
    n = y.numel()
    valid = int((y != IGNORE).sum())
    weight64 = inputs[1].double() if case["op"] == "linear" else None
    flat = inputs[0].reshape(n, -1)
    up = None
    if case["train"]:
        up = upstream.double().reshape(-1).expand(n)
        if case["reduction"] == "mean":
            up = up / max(valid, 1)
    losses, grads = [], []
    dw = torch.zeros_like(weight64) if weight64 is not None and case["train"] else None
    step = max(1, min(n, 2 ** 28 // V))
    for lo in range(0, n, step):
        yy = y[lo:lo + step]
        has = (yy != IGNORE)
        rows64 = flat[lo:lo + step].double()
        s = torch.mm(rows64, weight64.T) if weight64 is not None else rows64
        slope = None
        if case["softcap"] > 0:
            t = torch.tanh(s / case["softcap"])
            slope = 1.0 - t.square()
            s = t * case["softcap"]
        logp = torch.log_softmax(s, dim=1)
        norm = torch.logsumexp(s, dim=1)
        # the smoothed target distribution q; cross entropy = -sum q log p
        q = torch.full_like(s, case["smoothing"] / V)
        q[torch.arange(yy.numel(), device=y.device)[has], yy[has]] += 1.0 - case["smoothing"]
        row = -(q * logp).sum(dim=1) + case["z_loss"] * norm.square()
        losses.append(row.masked_fill(~has, 0.0))
        if case["train"]:
            ds = logp.exp() * (1.0 + 2.0 * case["z_loss"] * norm[:, None]) - q
            if slope is not None:
                ds = ds * slope
            ds = ds * up[lo:lo + step, None]
            ds = ds.masked_fill(~has[:, None], 0.0)
            if weight64 is not None:
                grads.append(torch.mm(ds, weight64))
                dw += torch.mm(ds.T, rows64)
            else:
                grads.append(ds)
    loss = torch.cat(losses)
    if case["reduction"] == "none":
        loss = loss.view(labels.shape)
    else:
        loss = loss.sum() / (max(valid, 1) if case["reduction"] == "mean" else 1)
    if not case["train"]:
        return (loss,)
    grad = torch.cat(grads).view(inputs[0].shape)
    return (loss, grad, dw) if dw is not None else (loss, grad)
