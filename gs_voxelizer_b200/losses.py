"""L1 loss against a target volume, standalone or fused into voxelization.

The reference leaves losses to its callers (FaCT-GS trains with L1 / SSIM in
PyTorch). These helpers compute the same L1 loss with this package's CUDA
kernels:

* ``l1_loss(vol, target)`` - drop-in for ``torch.nn.functional.l1_loss``
  (mean reduction by default): one reduction pass forward, one pass backward.
* ``voxelize_gaussians_l1(...)`` - voxelization with the loss fused in: the
  forward kernel reduces |vol - target| per tile while it stores the volume,
  and the backward kernel forms sign(vol - target) while it stages each tile,
  so dL/dvol is never materialised. Returns ``(loss, volume)``; gradients
  flow from the loss to the Gaussians (the volume output is not
  differentiable). With a ``SlabPlan`` it voxelizes one z-slab and, in the
  backward, all-reduces the per-Gaussian gradients over the process group.

Further losses of a volume: ``fused_ssim3d`` and ``tv3d``, and the class
losses ``softmax_cross_entropy`` (the channels are class scores) and
``linear_cross_entropy`` (the channels are features, scored against a table of
class embeddings without keeping the scores).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import Function, forward_ad

from . import cuda as _C
from ._lib import CeOptions, check, i3, lib
from .slab import SlabPlan, allreduce_gaussian_grads, tile_layers


def _dev_check(t: torch.Tensor, name: str) -> None:
    _C._check_input(t, name)
    _C._check_f32(t, name)


class _L1Loss(Function):
    @staticmethod
    def forward(ctx, vol, target, denom):
        vol, target = vol.contiguous(), target.contiguous()
        _dev_check(vol, "vol")
        _dev_check(target, "target")
        if vol.shape != target.shape:
            raise ValueError(f"shape mismatch: {vol.shape} vs {target.shape}")
        n = vol.numel()
        loss = torch.empty((), dtype=torch.float32, device=vol.device)
        ws = _C._workspace(lib.gsv_l1_loss_workspace_bytes(n), vol.device)
        check(lib.gsv_l1_loss_forward(n, _C._ptr(vol), _C._ptr(target),
                                      float(denom), loss.data_ptr(),
                                      ws.data_ptr(), ws.numel(),
                                      _C._stream(vol.device)))
        ctx.denom = float(denom)
        ctx.save_for_backward(vol, target)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        vol, target = ctx.saved_tensors
        grad_loss = grad_loss.contiguous().to(torch.float32)
        g = torch.empty_like(vol)
        check(lib.gsv_l1_loss_backward(vol.numel(), _C._ptr(vol),
                                       _C._ptr(target), grad_loss.data_ptr(),
                                       ctx.denom, _C._ptr(g),
                                       _C._stream(vol.device)))
        return g, None, None


def l1_loss(vol: torch.Tensor, target: torch.Tensor,
            reduction: str = "mean") -> torch.Tensor:
    """sum |vol - target| / numel ("mean") or the plain sum ("sum")."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"unsupported reduction {reduction!r}")
    denom = vol.numel() if reduction == "mean" else 1.0
    return _L1Loss.apply(vol, target, max(denom, 1))


class _VoxelizeL1(Function):
    @staticmethod
    def forward(ctx, pos3d_radii, conics, intensities, target, plan,
                tile_min, tile_max, denom, group, reduce):
        one_d = intensities.dim() == 1
        if one_d:
            intensities = intensities.unsqueeze(-1)
        C = _C._channels(intensities)
        for t, name in ((pos3d_radii, "pos3d_radii"), (conics, "conics"),
                        (intensities, "intensities"), (target, "target")):
            _dev_check(t, name)
        dev = pos3d_radii.device
        if tuple(target.shape) != (*plan.shape, C):
            raise ValueError(f"target shape {tuple(target.shape)} != "
                             f"{(*plan.shape, C)}")
        tile_min, tile_max = tile_min.contiguous(), tile_max.contiguous()
        n = int(pos3d_radii.shape[0])
        n_isect = plan.count(tile_min, tile_max)
        i32 = dict(dtype=torch.int32, device=dev)
        ids = torch.empty((n_isect,), **i32)
        bins = torch.empty((plan.num_tiles, 2), **i32)
        out = torch.empty(target.shape, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        ws = _C._workspace(lib.gsv_voxelize_l1_workspace_bytes(
            n, C, n_isect, i3(plan.vol), plan.tz0, plan.tz1), dev)
        # one call: binning, voxelization + loss, backward work plan in ws
        check(lib.gsv_voxelize_forward_l1(
            i3(plan.vol), plan.tz0, plan.tz1, C, n, n_isect,
            tile_min.data_ptr(), tile_max.data_ptr(), _C._ptr(pos3d_radii),
            _C._ptr(conics), _C._ptr(intensities), _C._ptr(target),
            float(denom), _C._ptr(ids), _C._ptr(bins), _C._ptr(out),
            loss.data_ptr(), None, None, ws.data_ptr(), ws.numel(),
            _C._stream(dev)))
        ctx.ws = ws
        ctx.plan, ctx.denom, ctx.group, ctx.one_d = plan, float(denom), group, one_d
        ctx.reduce = reduce
        ctx.save_for_backward(pos3d_radii, conics, intensities, ids, bins, out,
                              target)
        ctx.mark_non_differentiable(out)
        return loss, out

    @staticmethod
    def backward(ctx, grad_loss, _grad_out):
        pr, cq, inten, ids, bins, out, target = ctx.saved_tensors
        plan = ctx.plan
        C = inten.shape[1]
        n, n_isect, dev = int(pr.shape[0]), int(ids.numel()), pr.device
        f = dict(device=dev, dtype=torch.float32)
        gp = torch.empty((n, 4), **f)
        gc = torch.empty((n, 6), **f)
        gi = torch.empty((n, C), **f)
        if grad_loss is None:
            grad_loss = torch.zeros((), **f)
        grad_loss = grad_loss.contiguous().to(torch.float32)
        ws = ctx.ws  # records and work plan left by the forward
        check(lib.gsv_voxelize_backward_per_gaussian_l1(
            i3(plan.vol), plan.tz0, plan.tz1, C, n, n_isect, _C._ptr(ids),
            _C._ptr(bins), _C._ptr(pr), _C._ptr(cq), _C._ptr(inten),
            _C._ptr(out), _C._ptr(target), grad_loss.data_ptr(), ctx.denom,
            _C._ptr(gp), _C._ptr(gc), _C._ptr(gi), ws.data_ptr(), ws.numel(),
            _C._stream(dev)))
        if ctx.reduce:
            gp, gc, gi = allreduce_gaussian_grads([gp, gc, gi], ctx.group)
        if ctx.one_d:
            gi = gi.reshape(-1)
        return gp, gc, gi, None, None, None, None, None, None, None


def voxelize_gaussians_l1(
    pos3d_radii: torch.Tensor,
    conics: torch.Tensor,
    intensities: torch.Tensor,
    vol_size_voxel: Tuple[int, int, int],
    tile_min: torch.Tensor,
    tile_max: torch.Tensor,
    target: torch.Tensor,
    denom: Optional[float] = None,
    plan: Optional[SlabPlan] = None,
    group=None,
):
    """Voxelize and compute L = sum |vol - target| / denom in one pass.

    Args: as ``voxelize.voxelize_gaussians`` plus
        target: [Z,Y,X,C] float32 target (the slab's part with a plan).
        denom: normaliser; default the full volume's element count (mean).
        plan: SlabPlan for z-slab sharding; default the whole volume (then no
            collective, even inside a distributed job).
        group: process group for the gradient all-reduce (slab mode; default
            the default group when torch.distributed is initialised).
    Returns:
        (loss, volume): loss is a 0-d tensor (this slab's share with a plan),
        volume the forward volume (no gradient).
    """
    reduce = plan is not None
    if plan is None:
        plan = SlabPlan(vol_size_voxel, 0, tile_layers(vol_size_voxel))
    if denom is None:
        z, y, x = (int(v) for v in vol_size_voxel)
        C = 1 if intensities.dim() == 1 else int(intensities.shape[1])
        denom = float(z * y * x * C)
    return _VoxelizeL1.apply(pos3d_radii.contiguous(), conics.contiguous(),
                             intensities.contiguous(), target.contiguous(),
                             plan, tile_min.contiguous(),
                             tile_max.contiguous(), denom, group, reduce)


# ------------------------------------------------------------- 3D SSIM / TV

def _planar(t: torch.Tensor, name: str) -> Tuple[int, Tuple[int, int, int]]:
    """(channels, (D, H, W)) of a [..., D, H, W] volume: every leading
    dimension counts as a channel (the [B, C, D, H, W] layout of
    fused_ssim3d's callers, or [D, H, W])."""
    if t.dim() < 3:
        raise ValueError(f"{name} must have at least 3 dimensions (D, H, W)")
    d, h, w = (int(v) for v in t.shape[-3:])
    nch = 1
    for v in t.shape[:-3]:
        nch *= int(v)
    return nch, (d, h, w)


class _Ssim3d(Function):
    @staticmethod
    def forward(ctx, img1, img2, c1, c2):
        img1, img2 = img1.contiguous(), img2.contiguous()
        _dev_check(img1, "img1")
        _dev_check(img2, "img2")
        if img1.shape != img2.shape:
            raise ValueError(f"shape mismatch: {img1.shape} vs {img2.shape}")
        nch, dhw = _planar(img1, "img1")
        dims = i3(dhw)
        ws = _C._workspace(lib.gsv_ssim3d_workspace_bytes(nch, dims), img1.device)
        out = torch.empty((), dtype=torch.float32, device=img1.device)
        check(lib.gsv_ssim3d_forward(nch, dims, img1.data_ptr(), img2.data_ptr(),
                                     float(c1), float(c2), out.data_ptr(),
                                     ws.data_ptr(), ws.numel(),
                                     _C._stream(img1.device)))
        ctx.save_for_backward(img1, img2, ws)
        ctx.nch, ctx.dims = nch, dhw
        return out

    @staticmethod
    def backward(ctx, grad_out):
        img1, img2, ws = ctx.saved_tensors
        g = torch.empty_like(img1)
        grad_out = grad_out.contiguous().to(torch.float32)
        check(lib.gsv_ssim3d_backward(ctx.nch, i3(ctx.dims), img1.data_ptr(),
                                      img2.data_ptr(), grad_out.data_ptr(),
                                      ws.data_ptr(), ws.numel(), g.data_ptr(),
                                      _C._stream(img1.device)))
        return g, None, None, None


def fused_ssim3d(img1: torch.Tensor, img2: torch.Tensor,
                 c1: float = 0.01 ** 2, c2: float = 0.03 ** 2) -> torch.Tensor:
    """Mean 3D SSIM of img1 against img2 (Wang et al. 2004; 11^3 separable
    Gaussian window with sigma 1.5, zero padding), differentiable in img1.

    Volumes are [..., D, H, W] float32 CUDA tensors, every leading dimension
    a channel: the [B, C, D, H, W] call of the external fused_ssim3d in the
    reference's tests (test/test_gs_voxelizer.py:62) works unchanged, e.g.
    ``fused_ssim3d(vol.squeeze().unsqueeze(0).unsqueeze(0), target[None, None])``
    for a one-channel voxelizer output. Returns a 0-d tensor (higher is more
    similar; train with ``1 - fused_ssim3d(...)``)."""
    return _Ssim3d.apply(img1, img2, c1, c2)


class _Tv3d(Function):
    @staticmethod
    def forward(ctx, vol, isotropic, eps):
        vol = vol.contiguous()
        _dev_check(vol, "vol")
        nch, dhw = _planar(vol, "vol")
        dims = i3(dhw)
        ws = _C._workspace(lib.gsv_tv3d_workspace_bytes(nch, dims), vol.device)
        out = torch.empty((), dtype=torch.float32, device=vol.device)
        check(lib.gsv_tv3d(nch, dims, vol.data_ptr(), int(bool(isotropic)),
                           float(eps), out.data_ptr(), None, None, ws.data_ptr(),
                           ws.numel(), _C._stream(vol.device)))
        ctx.save_for_backward(vol, ws)
        ctx.nch, ctx.dims, ctx.iso, ctx.eps = nch, dhw, bool(isotropic), float(eps)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        vol, ws = ctx.saved_tensors
        g = torch.empty_like(vol)
        grad_out = grad_out.contiguous().to(torch.float32)
        check(lib.gsv_tv3d(ctx.nch, i3(ctx.dims), vol.data_ptr(), int(ctx.iso),
                           ctx.eps, None, grad_out.data_ptr(), g.data_ptr(),
                           ws.data_ptr(), ws.numel(), _C._stream(vol.device)))
        return g, None, None


def tv3d(vol: torch.Tensor, isotropic: bool = True, eps: float = 1e-8) -> torch.Tensor:
    """3D total variation of a [..., D, H, W] volume (leading dimensions are
    channels), mean over voxels and channels, with forward differences that
    are 0 across the far boundary: isotropic sqrt(dx^2 + dy^2 + dz^2 + eps)
    or anisotropic |dx| + |dy| + |dz|. Differentiable; a 0-d tensor."""
    if isotropic and not eps > 0:
        raise ValueError("isotropic TV needs eps > 0")
    return _Tv3d.apply(vol, isotropic, eps)


# ---------------------------------------------------------- class losses

_CE_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CE_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _ce_args(named, labels, ignore_index, label_smoothing, softcap, z_loss,
             reduction):
    """Checks what both class losses take; returns (labels as contiguous
    int64, options)."""
    first_name, first = named[0]
    for name, t in named:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.dtype not in _CE_DTYPES:
            raise RuntimeError(f"{name} must be float32, bfloat16 or float16, "
                               f"got {t.dtype}")
        if t.dtype != first.dtype or t.device != first.device:
            raise RuntimeError(f"{name} must share dtype and device with "
                               f"{first_name}")
    if first.dim() < 1:
        raise ValueError(f"{first_name} must have at least one dimension")
    if labels.device != first.device:
        raise RuntimeError(f"labels must be on the device of {first_name}")
    if labels.dtype.is_floating_point or labels.dtype.is_complex \
            or labels.dtype == torch.bool:
        raise RuntimeError(f"labels must be integers, got {labels.dtype}")
    if labels.shape != first.shape[:-1]:
        raise ValueError(f"labels shape {tuple(labels.shape)} != "
                         f"{tuple(first.shape[:-1])}")
    if reduction not in _CE_REDUCTIONS:
        raise ValueError(f"unsupported reduction {reduction!r}")
    # (the largest float32 below 1: what rounds to 1 is refused too)
    if not 0.0 <= label_smoothing <= 1.0 - 2.0 ** -24:
        raise ValueError("label_smoothing must be in [0, 1)")
    # (a softcap below float32's least number would be none)
    if not ((softcap == 0.0 or 1e-30 <= softcap <= 1e30) and 0.0 <= z_loss <= 1e30):
        raise ValueError("softcap and z_loss must be finite and >= 0, and a "
                         "softcap at least 1e-30")
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must be a 64-bit integer")
    opt = CeOptions(int(ignore_index), label_smoothing, softcap, z_loss,
                    _CE_REDUCTIONS[reduction])
    return labels.to(torch.int64).contiguous(), opt


def _ce_loss_out(labels, opt, dev):
    return torch.empty(labels.shape if opt.reduction == 0 else (),
                       dtype=torch.float32, device=dev)


def _ce_call(fn, dev, *args):
    """fn(*args, stream) on the current stream of dev. These losses may be of
    a few rows, where a call's own microseconds count: the stream is asked for
    by number and the device is set only where it is not the current one."""
    i = dev.index
    stream = torch._C._cuda_getCurrentRawStream(i)
    if torch.cuda.current_device() == i:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(i):
            status = fn(*args, stream)
    if status:
        check(status)


class _Once(Function):
    """The identity on a gradient, whose own backward is refused: the class
    losses are differentiable once. Only entered under create_graph (a
    decorator that marks every backward costs each call a tenth)."""

    @staticmethod
    def forward(ctx, grad, *inputs):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the class losses are differentiable once")


def _recorded(a, b):
    """Whether autograd has to see the call: an input needs a gradient, or may
    carry a tangent, which the function refuses (a dual tensor needs no gradient
    and would lose its tangent in silence)."""
    return forward_ad._current_level >= 0 or (
        (a.requires_grad or b.requires_grad) and torch.is_grad_enabled())


def _as_kept(saved):
    """Saved tensors that a hook brought back with other strides, or the last
    one (raw bytes) off the alignment of what it holds, as the kernels take
    them."""
    *rest, raw = (t.contiguous() for t in saved)
    return (*rest, raw.clone() if raw.data_ptr() & 15 else raw)


def _softmax_ce(scores, labels, opt):
    """(loss, stats, where in stats the count is): per row of more than 1024
    classes (maximum, log2 of the sum), then the number of labelled rows, then
    the call's workspace."""
    dev, V, rows = scores.device, scores.size(-1), labels.numel()
    loss = _ce_loss_out(labels, opt, dev)
    if rows == 0:
        return loss.zero_(), None, 0
    lse = lib.gsv_softmax_ce_lse_bytes(rows, V)
    nbytes = lib.gsv_softmax_ce_workspace_bytes(rows, V)
    stats = torch.empty((lse + 8 + nbytes,), dtype=torch.uint8, device=dev)
    p = stats.data_ptr()
    _ce_call(lib.gsv_softmax_ce_forward, dev, rows, V, _CE_DTYPES[scores.dtype],
             scores.data_ptr(), labels.data_ptr(), opt, loss.data_ptr(), p,
             p + lse, p + lse + 8, nbytes)
    return loss, stats, lse


class _SoftmaxCe(Function):
    @staticmethod
    def forward(ctx, scores, labels, opt):
        ctx.opt = opt
        loss, stats, ctx.lse = _softmax_ce(scores, labels, opt)
        if stats is None:
            ctx.save_for_backward(scores)
        else:
            ctx.save_for_backward(scores, labels, stats)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        saved = ctx.saved_tensors
        if len(saved) == 1:
            return torch.zeros_like(saved[0]), None, None
        scores, labels, stats = saved
        if stats.data_ptr() & 15 or not (
                scores.is_contiguous() and labels.is_contiguous()
                and stats.is_contiguous()):
            scores, labels, stats = _as_kept(saved)
        dev, rows, V = scores.device, labels.numel(), scores.size(-1)
        grad_loss = grad_loss.contiguous()  # float32, as the loss is
        g = torch.empty_like(scores)
        p = stats.data_ptr()
        _ce_call(lib.gsv_softmax_ce_backward, dev, rows, V,
                 _CE_DTYPES[scores.dtype], scores.data_ptr(), labels.data_ptr(),
                 ctx.opt, p, p + ctx.lse, grad_loss.data_ptr(), g.data_ptr())
        if torch.is_grad_enabled():
            g = _Once.apply(g, scores, grad_loss)
        return g, None, None


def softmax_cross_entropy(
    scores: torch.Tensor,
    labels: torch.Tensor,
    ignore_index: int = -100,
    label_smoothing: float = 0.0,
    softcap: float = 0.0,
    z_loss: float = 0.0,
    reduction: str = "mean",
) -> torch.Tensor:
    """Softmax cross entropy of class scores against labels, e.g. of a
    [Z, Y, X, C] volume whose channels are class scores.

    With z = scores (or softcap * tanh(scores / softcap)) over the V classes
    of the last dimension and lse = log sum exp z, a row's loss is
    ``lse - (1 - s) z[label] - s mean(z) + z_loss lse^2`` with s =
    label_smoothing.

    Args:
        scores: [..., V] float32, bfloat16 or float16.
        labels: [...] integers. Rows labelled ``ignore_index`` have loss 0 and
            a zero gradient whatever they hold; any other label outside
            [0, V) makes the row's loss and gradient NaN.
        ignore_index, label_smoothing, softcap, z_loss: see above.
        reduction: "mean" over the labelled rows of this call (0 if there is
            none), "sum" or "none" (the losses in the shape of labels). Ranks
            that each hold a slab of a volume take "sum" over the all-reduced
            number of labelled voxels: a slab's mean is over its own.
    Returns:
        float32 loss, differentiable once in scores, in reverse mode (gradient
        in their type).
    """
    labels, opt = _ce_args([("scores", scores)], labels, ignore_index,
                           label_smoothing, softcap, z_loss, reduction)
    if scores.shape[-1] < 1:
        raise ValueError("scores must have at least one class")
    scores = scores.contiguous()
    if not _recorded(scores, scores):
        return _softmax_ce(scores, labels, opt)[0]
    return _SoftmaxCe.apply(scores, labels, opt)


def _linear_ce(features, weight, labels, opt, with_state):
    """(loss, state for the backward or None)."""
    dev, rows, (V, D) = features.device, labels.numel(), weight.shape
    loss = _ce_loss_out(labels, opt, dev)
    if rows == 0:
        return loss.zero_(), None
    dtype = _CE_DTYPES[features.dtype]
    state = None
    if with_state:
        state = _C._workspace(
            lib.gsv_linear_ce_state_bytes(rows, V, D, dtype), dev)
    x, w = features.data_ptr(), weight.data_ptr()
    call = (2 if with_state else 8) | (0 if (x | w) & 15 else 4)  # gsv_ce_call
    ws = _C._workspace(lib.gsv_linear_ce_workspace_bytes(
        rows, V, D, dtype, opt, call), dev)
    _ce_call(lib.gsv_linear_ce_forward, dev, rows, V, D, dtype, x, w,
             labels.data_ptr(), opt, loss.data_ptr(), _C._ptr(state),
             ws.data_ptr(), ws.numel())
    return loss, state


class _LinearCe(Function):
    @staticmethod
    def forward(ctx, features, weight, labels, opt):
        ctx.opt = opt
        loss, state = _linear_ce(features, weight, labels, opt, True)
        if state is None:
            ctx.save_for_backward(features, weight)
        else:
            ctx.save_for_backward(features, weight, labels, state)
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        need_x, need_w = ctx.needs_input_grad[:2]
        saved = ctx.saved_tensors
        if len(saved) == 2:
            return (*(torch.zeros_like(t) if need else None for t, need in
                      zip(saved, (need_x, need_w))), None, None)
        features, weight, labels, state = saved
        if state.data_ptr() & 15 or not (
                features.is_contiguous() and weight.is_contiguous()
                and labels.is_contiguous() and state.is_contiguous()):
            features, weight, labels, state = _as_kept(saved)
        dev = features.device
        rows, (V, D) = labels.numel(), weight.shape
        dtype = _CE_DTYPES[features.dtype]
        grad_loss = grad_loss.contiguous()  # float32, as the loss is
        gx = torch.empty_like(features) if need_x else None
        gw = torch.empty_like(weight) if need_w else None
        x, w = features.data_ptr(), weight.data_ptr()
        call = 1 if (x | w) & 15 else 1 | 4  # gsv_ce_call
        ws = _C._workspace(lib.gsv_linear_ce_workspace_bytes(
            rows, V, D, dtype, ctx.opt, call), dev)
        _ce_call(lib.gsv_linear_ce_backward, dev, rows, V, D, dtype, x, w,
                 labels.data_ptr(), ctx.opt, state.data_ptr(),
                 grad_loss.data_ptr(), _C._ptr(gx), _C._ptr(gw), ws.data_ptr(),
                 ws.numel())
        if torch.is_grad_enabled():
            gx, gw = (g if g is None else _Once.apply(g, features, weight, grad_loss)
                      for g in (gx, gw))
        return gx, gw, None, None


def linear_cross_entropy(
    features: torch.Tensor,
    weight: torch.Tensor,
    labels: torch.Tensor,
    ignore_index: int = -100,
    label_smoothing: float = 0.0,
    softcap: float = 0.0,
    z_loss: float = 0.0,
    reduction: str = "mean",
) -> torch.Tensor:
    """``softmax_cross_entropy(features @ weight.T, labels, ...)`` without the
    scores in memory: e.g. a [Z, Y, X, C] volume decoded by a table of V class
    embeddings, or the hidden states of a model against a vocabulary.

    The scores are products of the inputs summed in float32 and are not
    rounded to the inputs' type. The forward keeps 8 or 16 bytes a row and, up
    to 16 MB each, its packed operands; the backward computes the scores again
    in pieces, with a workspace of a few hundred MB beside packed copies of the
    features (and of a table that cannot be read in place) and float32 copies
    of what it accumulates over several pieces. (Scores of at most 16 classes
    over more than 32 float32 channels, less than half of the features' size,
    are kept instead, from 16384 rows on.) The derivatives in the scores are
    rounded to a 16-bit type before its gradients are formed of them; in
    float16 with ``reduction="none"`` relative to the largest row's upstream
    gradient, below 2^-10 of which a row loses digits. With
    ``reduction="none"`` and no gradient it is minus the log-probability of
    each row's label.

    Args:
        features: [..., D] float32, bfloat16 or float16.
        weight: [V, D] of the same type.
        labels, ignore_index, label_smoothing, softcap, z_loss, reduction: as
            for ``softmax_cross_entropy``.
    Returns:
        float32 loss, differentiable once in features and weight, in reverse
        mode (gradients in their type).
    """
    labels, opt = _ce_args([("features", features), ("weight", weight)], labels,
                           ignore_index, label_smoothing, softcap, z_loss,
                           reduction)
    if weight.dim() != 2 or weight.shape[1] != features.shape[-1]:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match "
                         f"features {tuple(features.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("weight must have at least one class and one channel")
    features, weight = features.contiguous(), weight.contiguous()
    if not _recorded(features, weight):
        return _linear_ce(features, weight, labels, opt, False)[0]
    return _LinearCe.apply(features, weight, labels, opt)
