"""Class losses in float64 from their definition, and the error bounds their
float32 evaluation may have."""
import math

import torch

HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8,
            torch.float16: 2.0 ** -11}


def reference(scores, labels, ignore=-100, smoothing=0.0, softcap=0.0,
              z_loss=0.0, reduction="mean", upstream=None):
    """scores [n, V] float64, labels [n], upstream None, 0-d or [n]. Returns a
    dict: loss, rows (per-row losses), ds (d loss / d scores, all of
    upstream and reduction in it), dabs (the same sum of magnitudes before
    cancellation), lse."""
    n, V = scores.shape
    keep = labels != ignore
    bad = keep & ((labels < 0) | (labels >= V))
    y = labels.clamp(0, V - 1)
    # what an ignored row holds plays no part
    s = torch.where(keep[:, None], scores, torch.zeros_like(scores))
    z = softcap * torch.tanh(s / softcap) if softcap > 0 else s
    lse = torch.logsumexp(z, 1)
    rows = lse - (1 - smoothing) * z.gather(1, y[:, None])[:, 0]
    if smoothing > 0:
        rows = rows - smoothing * z.mean(1)
    if z_loss > 0:
        rows = rows + z_loss * lse ** 2
    nan = torch.full_like(rows, math.nan)
    rows = torch.where(bad, nan, torch.where(keep, rows, torch.zeros_like(rows)))
    count = max(int(keep.sum()), 1)
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / count}[reduction]
    out = {"loss": loss, "rows": rows, "lse": lse, "count": count}
    if upstream is not None:
        g = upstream.double().reshape(-1).expand(n)
        if reduction == "mean":
            g = g / count
        g = torch.where(keep, g, torch.zeros_like(g))[:, None]
        soft = (1 + 2 * z_loss * lse)[:, None] * torch.exp(z - lse[:, None])
        hit = torch.zeros_like(z).scatter_(1, y[:, None], 1 - smoothing)
        slope = 1 - (z / softcap) ** 2 if softcap > 0 else torch.ones_like(z)
        ds = (soft - hit - smoothing / V) * slope * g
        dabs = (soft.abs() + hit + smoothing / V) * g.abs()
        zero = torch.zeros_like(ds)
        out["ds"] = torch.where(bad[:, None], zero + math.nan,
                                torch.where(keep[:, None], ds, zero))
        out["dabs"] = torch.where(keep[:, None], dabs, zero)
        out["g"] = g[:, 0]
    return out


def score_error(magnitude, D, softcap):
    """Largest error of a float32 score: D products summed (each addition off
    by at most an ulp of the running magnitude, 2^-23, matrix units truncate),
    and the cap's tanh (2^-21 of the cap)."""
    return (D + 8) * 2.0 ** -23 * magnitude + softcap * 2.0 ** -21


def loss_error(ref, es, z_loss):
    """Of one row: twice the scores' error (lse and the label's score), the
    exponentials and their sum (ex2 2^-22 relative; at most 2^11 additions in
    sequence before a pairwise merge: 2^11 2^-24), the exponent's rounding
    (|lse| 2^-22), final additions."""
    big = float(ref["lse"].abs().max()) + 1.0
    return (1 + 2 * z_loss * big) * (2 * es + 2.0 ** -13 + 2.0 ** -21 * big)


def grad_error(ref, es):
    """Relative error of d loss / d scores against dabs: the probability's
    own (exponent off by es and lse's error), products."""
    big = float(ref["lse"].abs().max()) + 1.0
    return 4 * es + 2.0 ** -13 + 2.0 ** -20 * big
