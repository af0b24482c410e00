"""The plane-sweep volume as a distribution over depth planes (csrc/cv_plane_stats.hip).

A volume [b, D, h, w] scores D depth planes per pixel.  The reference takes one thing from it outside the networks, the plane of
the highest score (argmax + gather, modules/cost_volume.py:355-361: ``lowest_cost``).  Read as logits the same scores also say how
probable any other depth is and how sure the matching is:

    plane_log_probs  log probability of a given plane, entropy, normaliser and the most probable planes of every pixel; differentiable
    nearest_planes   the plane index a metric depth falls on -- what a predicted, rendered or measured depth map is scored by

``CostVolumeManager.plane_statistics`` puts the two together; ``model.enable_plane_statistics()`` adds the result to the model's
outputs.  No CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad as _forward_ad

from .. import _abi

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
#: most alternatives per pixel (DT_PLANE_MAX_TOP)
MAX_TOP = 8
#: factors on the scores; the gradient's intermediate values (scale * gradient * log probability) stay finite for gradients up to 1e4
MIN_SCALE, MAX_SCALE = 1e-30, 1e30
#: planes per volume (DT_PLANE_MAX_PLANES: what float32 sums bear); depth planes nearest_planes searches (DT_PLANE_MAX_NEAREST)
MAX_PLANES, MAX_NEAREST = 1 << 16, 1 << 30


class PlaneLogProbs(NamedTuple):
    """What ``plane_log_probs`` returns; entries that were not asked for are None.  Real-valued entries are float32."""
    log_prob_bhw: Optional[torch.Tensor]        # of the given plane; ``outside`` (0) where it is not in 0..D-1
    entropy_bhw: torch.Tensor                   # nats
    log_sum_bhw: torch.Tensor                   # log of the sum of exp(scale * score)
    top_log_prob_bkhw: Optional[torch.Tensor]   # descending
    top_plane_bkhw: Optional[torch.Tensor]      # int64, as indices_to_disparity takes them; -1 where there is none
    top_depth_bkhw: Optional[torch.Tensor]


def check_scale(scale):
    if not MIN_SCALE <= scale <= MAX_SCALE:
        raise ValueError(f"scale={scale} must be a positive number between {MIN_SCALE} and {MAX_SCALE}")


def _require_gpu(t, name):
    if not t.is_cuda:
        raise _abi.DoubletakeHipError(f"{name} is on {t.device}; doubletake_amd plane statistics only run on a ROCm GPU (no CPU fallback)")


def _refuse_tangent(t, name):
    if _forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} carries a forward-mode tangent: plane_ops has reverse-mode gradients only")


def _broadcast(t, shape, device, name):
    """``t`` as a view of ``shape`` = (b, D, h, w) with stride 0 along the axes it is broadcast over."""
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.shape == shape:
        return t
    if t.dim() != 4 or any(n != m and n != 1 for n, m in zip(t.shape, shape)):
        raise ValueError(f"{name} {tuple(t.shape)} does not broadcast to {tuple(shape)}")
    return t.expand(shape)


def _desc(vol, top, scale, mask, planes, outside=0.0):
    d = _abi.PlaneDesc()
    d.b, d.d, d.h, d.w = vol.shape
    d.dtype, d.top, d.scale = _DTYPES[vol.dtype], top, scale
    if outside:
        d.outside = outside
    d.vol_stride[:] = vol.stride()
    if mask is not None:
        d.mask_stride[:] = mask.stride()
    if planes is not None:
        d.planes_stride[:] = planes.stride()
    return d


def _forward(vol, plane, top, scale, mask, planes, outside, for_grad):
    """(outputs, row statistics [2, b, h, w] or None, descriptor, stream)"""
    b, _, h, w = vol.shape
    ent = torch.empty((b, h, w), device=vol.device, dtype=torch.float32)
    lsum = torch.empty_like(ent)
    lp = torch.empty_like(ent) if plane is not None else None
    tlp = tpl = tdep = rows = None
    if top:
        tlp = torch.empty((b, top, h, w), device=vol.device, dtype=torch.float32)
        tpl = torch.empty_like(tlp, dtype=torch.int64)
        if planes is not None:
            tdep = torch.empty_like(tlp)
    rmax = rlog = None
    if for_grad:
        rows = torch.empty((2, b, h, w), device=vol.device, dtype=torch.float32)
        rmax = rows.data_ptr()
        rlog = rmax + 4 * b * h * w
    stream = _abi.current_stream(vol.device)
    desc = _desc(vol, top, scale, mask, planes, outside)
    if b * h * w:
        p = _abi.ptr
        _abi.check(_abi.lib().dt_cv_plane_log_probs(
            desc, vol.data_ptr(), p(mask), p(plane), p(planes), p(lp), ent.data_ptr(), lsum.data_ptr(), p(tlp), p(tpl), p(tdep), rmax, rlog,
            stream), "dt_cv_plane_log_probs")
    return PlaneLogProbs(lp, ent, lsum, tlp, tpl, tdep), rows, desc, stream


def _dense_f32(g):
    if g is None or (g.dtype is torch.float32 and g.is_contiguous() and not g.is_neg()):
        return g
    return g.to(torch.float32).resolve_neg().contiguous()


def _refuse_saved(ctx, *saved):
    back = [f"{t.dtype} {tuple(t.shape)} on {t.device}" for t in saved if t is not None]
    raise RuntimeError(f"a hook on saved tensors brought one back on another device, of another type or size than it was saved with "
                       f"({ctx.dtype} {tuple(ctx.shape)} on {ctx.rows.device}): {'; '.join(back)}")


def _backward(ctx, g_lp, g_ent, g_lsum, g_top, _g_plane, _g_depth):
    vol, plane, mask, ent, tpl = ctx.saved_tensors
    rows, shape = ctx.rows, ctx.shape
    dev, n = rows.device, rows.numel() // 2
    # Hooks on saved tensors may bring a tensor back in another layout than it was saved in, which is fine, but also on another device or
    # of another type or size, and the kernel is given addresses: refused.  (Written out: as a loop it cost 2.3 us of every call.)
    if (vol.device != dev or vol.dtype is not ctx.dtype or vol.shape != shape
            or ent.device != dev or ent.dtype is not torch.float32 or ent.numel() != n
            or (plane is not None and (plane.device != dev or plane.dtype is not torch.int64 or plane.numel() != n))
            or (mask is not None and (mask.device != dev or mask.dtype is not torch.bool or mask.shape != shape))
            or (tpl is not None and (tpl.device != dev or tpl.dtype is not torch.int64 or tpl.numel() != n * ctx.top))):
        _refuse_saved(ctx, vol, plane, mask, ent, tpl)
    if g_lp is not None:
        g_lp = _dense_f32(g_lp)
    if g_ent is not None:
        g_ent = _dense_f32(g_ent)
    if g_lsum is not None:
        g_lsum = _dense_f32(g_lsum)
    if g_top is not None:
        g_top = _dense_f32(g_top)
    grad = torch.empty_like(vol)   # (dense, in the order of the volume's own strides)
    if n:
        p, desc = _abi.ptr, ctx.desc
        if vol.stride() != ctx.vol_stride or (mask is not None and mask.stride() != ctx.mask_stride):
            desc = _desc(vol, ctx.top, ctx.scale, mask, None)
        desc.grad_stride[:] = grad.stride()
        if not ent.is_contiguous():
            ent = ent.contiguous()
        if plane is not None and not plane.is_contiguous():
            plane = plane.contiguous()
        if tpl is not None and not tpl.is_contiguous():
            tpl = tpl.contiguous()
        rmax = rows.data_ptr()
        _abi.check(_abi.lib().dt_cv_plane_log_probs_grad(
            desc, vol.data_ptr(), p(mask), p(plane), ent.data_ptr(), p(tpl), rmax, rmax + 4 * n, p(g_lp), p(g_ent), p(g_lsum), p(g_top),
            grad.data_ptr(), ctx.stream), "dt_cv_plane_log_probs_grad")
    return grad, None, None, None, None, None, None


class _PlaneLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, vol, plane, top, scale, mask, planes, outside):
        out, rows, ctx.desc, ctx.stream = _forward(vol, plane, top, scale, mask, planes, outside, True)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(*[t for t in out[4:] if t is not None])
        ctx.save_for_backward(vol, plane, mask, out[1], out[4])
        # made here, neither inputs nor outputs.  The engine runs a backward on the stream its forward ran on: the handle is kept, asking
        # for it in the engine's thread costs 6 us
        ctx.rows, ctx.top, ctx.scale, ctx.dtype, ctx.shape = rows, top, scale, vol.dtype, vol.shape
        # (the descriptor serves the backward too, unless a hook on saved tensors brings one back in another layout)
        ctx.vol_stride, ctx.mask_stride = vol.stride(), None if mask is None else mask.stride()
        return tuple(out)

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():  # create_graph=True: a second derivative raises where it is asked for (the wrapper costs 9 us)
            return _backward_once(ctx, *grads)
        return _backward(ctx, *grads)


_backward_once = torch.autograd.function.once_differentiable(_backward)


def plane_log_probs(volume_bdhw, plane_bhw=None, top=0, scale=1.0, mask_bdhw=None, depth_planes_bdhw=None, outside=0.0) -> PlaneLogProbs:
    """Log probabilities over the depth planes of a volume [b, D, h, w], in one pass over it.

    volume_bdhw: float32, float16 or bfloat16 scores in any layout (NCHW, channels_last, slices), 1..65536 planes; statistics are
        float32, the log probabilities within 2^-24 (D / 4 + 6 ln D + 40) nats plus 2^-22 of their value.
    plane_bhw: plane indices [b, h, w] (int64 or int32) whose log probability is wanted; one outside 0..D-1 (-1: no depth there)
        scores ``outside`` and takes no part in the gradient.
    top: how many of the most probable planes to return, 0..min(D, 8); equal scores in the order of their planes.
    scale: factor on the scores in front of the softmax (inverse temperature), a positive number, 1e-30..1e30.
    mask_bdhw: bool, broadcastable to the volume; False leaves a plane out, whatever the volume holds there.  A pixel without a
        visible plane of a score above -inf has entropy 0, log_sum and log_prob -inf, no alternatives (plane -1, log probability -inf,
        depth 0) and gradient 0.
    depth_planes_bdhw: float32 depths of the planes, broadcastable to the volume (what the managers return): the alternatives' depths
        are returned too.
    outside: log probability of a plane index outside 0..D-1: 0 drops such pixels out of a loss, -inf says that no plane is certain there.

    Differentiable in the volume (gradients of log_prob, entropy, log_sum and top_log_prob; not twice, not in forward mode): the
    gradient has the volume's type and layout.  It is for a caller's own differentiable volume: the managers' volumes carry no graph.
    A visible NaN or +inf makes the pixel's statistics NaN.  The call allocates its outputs, launches one kernel on the current stream
    (planes innermost: one per 2^29 pixels) and can be captured into a graph; capture a backward pass only together with its forward
    pass."""
    vol = volume_bdhw
    if vol.dim() != 4:
        raise ValueError(f"volume_bdhw must be [b, D, h, w], got {tuple(vol.shape)}")
    if vol.dtype not in _DTYPES:
        raise ValueError(f"volume_bdhw is {vol.dtype}; float32, float16 and bfloat16 are supported")
    b, D, h, w = vol.shape
    if not 1 <= D <= MAX_PLANES:
        raise ValueError(f"volume_bdhw has {D} planes; 1..{MAX_PLANES} are supported")
    if b * h * w >= 2**31 - 1:
        raise ValueError(f"volume_bdhw has {b * h * w} pixels; fewer than 2^31 - 1 are supported")
    top = int(top)
    if not 0 <= top <= min(D, MAX_TOP):
        raise ValueError(f"top={top} not in 0..{min(D, MAX_TOP)}")
    scale, outside = float(scale), float(outside)
    check_scale(scale)
    plane = plane_bhw
    if plane is not None:
        if plane.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"plane_bhw is {plane.dtype}; int64 or int32 plane indices expected")
        if plane.shape != (b, h, w):
            raise ValueError(f"plane_bhw {tuple(plane.shape)} does not match the volume's pixels {(b, h, w)}")
        if plane.device != vol.device:
            raise ValueError(f"plane_bhw is on {plane.device}, expected {vol.device}")
        if plane.dtype != torch.int64:
            plane = plane.to(torch.int64)
        if not plane.is_contiguous():
            plane = plane.contiguous()
    mask = mask_bdhw
    if mask is not None:
        if mask.dtype != torch.bool:
            raise ValueError(f"mask_bdhw is {mask.dtype}; bool expected")
        mask = _broadcast(mask, vol.shape, vol.device, "mask_bdhw")
    planes = depth_planes_bdhw
    if planes is not None:
        if not top:
            raise ValueError("depth_planes_bdhw gives the alternatives their depths: it goes with top > 0")
        if planes.dtype != torch.float32:
            raise ValueError(f"depth_planes_bdhw is {planes.dtype}; float32 expected")
        planes = _broadcast(planes, vol.shape, vol.device, "depth_planes_bdhw")
    if _forward_ad._current_level >= 0:   # (one comparison outside forward mode: unpack_dual costs 3 us)
        _refuse_tangent(vol, "volume_bdhw")
    _require_gpu(vol, "volume_bdhw")
    # (the imaginary part of a conjugate is a view that torch negates when it is read; the kernels read memory)
    if vol.is_neg():
        vol = vol.resolve_neg()
    if planes is not None and planes.is_neg():
        planes = planes.resolve_neg()
    if vol.requires_grad and torch.is_grad_enabled():
        return PlaneLogProbs(*_PlaneLogProbsFn.apply(vol, plane, top, scale, mask, planes, outside))
    return _forward(vol, plane, top, scale, mask, planes, outside, False)[0]


@torch.no_grad()
def nearest_planes(depth_bhw, depth_planes_bdhw):
    """int64 [b, h, w]: index of the depth plane nearest to each depth (absolute difference, the lowest index of equally near ones), the
    depths taken in float32 and the differences in float64: exact within a factor of 2^29, beyond it planes whose distances round to the
    same number are equally near (all planes of a few metres to a depth of 1e20: plane 0).  -1 where the depth is not finite or not
    positive (holes of a sensor's map, a renderer's background).  depth_planes_bdhw is float32 and broadcastable to [b, D, h, w] (what
    the cost-volume managers return)."""
    depth, planes = depth_bhw, depth_planes_bdhw
    if depth.dim() != 3:
        raise ValueError(f"depth_bhw must be [b, h, w], got {tuple(depth.shape)}")
    if not depth.is_floating_point():
        raise ValueError(f"depth_bhw is {depth.dtype}; metric depths are floating point")
    if planes.dim() != 4 or not 1 <= planes.shape[1] <= MAX_NEAREST:
        raise ValueError(f"depth_planes_bdhw must be [b, D, h, w] with 1..{MAX_NEAREST} planes, got {tuple(planes.shape)}")
    if planes.dtype != torch.float32:
        raise ValueError(f"depth_planes_bdhw is {planes.dtype}; float32 expected")
    b, h, w = depth.shape
    D = planes.shape[1]
    if b * h * w >= 2**31 - 1:
        raise ValueError(f"depth_bhw has {b * h * w} pixels; fewer than 2^31 - 1 are supported")
    planes = _broadcast(planes, (b, D, h, w), depth.device, "depth_planes_bdhw")
    if planes.is_neg():
        planes = planes.resolve_neg()
    _require_gpu(depth, "depth_bhw")
    depth = _dense_f32(depth)
    out = torch.empty((b, h, w), device=depth.device, dtype=torch.int64)
    if out.numel():
        _abi.check(_abi.lib().dt_cv_nearest_planes_f32(_abi.ptr(depth), _abi.ptr(planes), (C.c_int64 * 4)(*planes.stride()), b, D, h, w,
                                                       _abi.ptr(out), _abi.current_stream(depth.device)), "dt_cv_nearest_planes_f32")
    return out
