"""Group normalisation with the activation behind it, forward and backward (csrc/group_norm.hip).

The reference's networks normalise over the batch (networks/networks.py:147-190); per-GPU batches of one to eight volumes, and
statistics that stay per rank, are what that serves worst (the refiner's innermost stage is 1^3: BatchNorm refuses to train on
one image).  Group statistics belong to one image: the result does not depend on the batch or on the ranks.

GPU tensors only, like the other native ops."""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .._ext import group_norm_lib as _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_LAST = {4: torch.channels_last, 5: torch.channels_last_3d}


def _map(t):
    """the strides (image, channel, position) with which the kernels walk t [N, C, space...], and whether it is channels last (a row
    of channels per position; gaps between rows are fine) or first (a plane of positions per channel) -- or None: neither"""
    n, c = t.shape[:2]
    s = t.numel() // (n * c)
    if s > 1 and c > 1:
        if t.is_contiguous():
            return (c * s, s, 1), False
        if t.dim() in _LAST and t.is_contiguous(memory_format=_LAST[t.dim()]):
            return (c * s, 1, c), True
    step = expect = None                                # distance of two positions, if they all lie at one
    for size, stride in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != expect:
            return None
        expect = stride * size
    image, channel = t.stride(0), t.stride(1)
    if s == 1:
        return ((image, 1, c), True) if c == 1 or channel == 1 else None
    if step == 1 and (c == 1 or channel >= s):
        return (image, channel if c > 1 else s, 1), False
    return ((image, 1, step), True) if c > 1 and channel == 1 and step >= c else None


def _like(x, strides_of_x):
    """an uninitialised gap-free map in x's layout, with its strides"""
    y = torch.empty_like(x)
    m = _map(y)
    return (y, m[0]) if m is not None and m[1] == strides_of_x[1] else (None, None)


def _readable(x):
    """x, or a gap-free copy where the kernels cannot walk it, its _map, and an output of the same layout with its strides"""
    m = _map(x)
    if m is not None:
        y, ys = _like(x, m)
        if y is not None:
            return x, m, y, ys
    x = x.clone(memory_format=torch.contiguous_format)
    m = _map(x)
    return (x, m) + _like(x, m)


def _check(x, num_groups, weight, bias, eps, act):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("group_norm_act: x must be a GPU tensor -- there is no CPU path")
    if x.dtype not in _TYPES:
        raise RuntimeError("group_norm_act: dtype %s not supported (fp32, bf16 or fp16)" % x.dtype)
    if x.dim() < 2:
        raise RuntimeError("group_norm_act: x must be [N, C, ...], got %s" % (tuple(x.shape),))
    c = x.shape[1]
    if not isinstance(num_groups, int) or num_groups < 1 or c == 0 or c % num_groups:
        raise RuntimeError("group_norm_act: %d channels do not split into %r groups" % (c, num_groups))
    for what, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (c,) or t.dtype not in _TYPES or t.device != x.device):
            raise RuntimeError("group_norm_act: %s must be a [%d] tensor of fp32, bf16 or fp16 on %s, got %s %s on %s"
                               % (what, c, x.device, tuple(t.shape), t.dtype, t.device))
    if not eps > 0:
        raise RuntimeError("group_norm_act: eps must be positive, got %r" % (eps,))
    if act not in _native.ACTS:
        raise RuntimeError("group_norm_act: act must be one of %s, got %r" % (sorted(_native.ACTS), act))


def _forward(x, weight, bias, num_groups, eps, act, slope):
    """(the map that was read, its _map, weight, bias, y, stats [2, N, groups])"""
    n, c = x.shape[:2]
    if x.numel() == 0:
        return x, None, weight, bias, torch.empty_like(x), torch.empty((2, n, num_groups), dtype=torch.float64, device=x.device)
    x, m, y, ys = _readable(x)
    weight, bias = (t if t is None or t.is_contiguous() else t.contiguous() for t in (weight, bias))
    stats = torch.empty((2, n, num_groups), dtype=torch.float64, device=x.device)
    _native.forward(x, m[0], y, ys, (n, c, x.numel() // (n * c)), weight, bias, stats, num_groups, eps, _native.ACTS[act], slope)
    return x, m, weight, bias, y, stats


class GroupNormActFunction(Function):
    """(x, weight, bias, num_groups, eps, act, slope) -> y; differentiable once in x, weight and bias"""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act, slope):
        x, ctx.map, weight, bias, y, stats = _forward(x.detach(), weight, bias, num_groups, eps, act, slope)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = num_groups, _native.ACTS[act], slope
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        groups, act, slope = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if x.numel() == 0:
            return (torch.empty_like(x) if need_x else None, torch.zeros_like(weight) if need_w else None,
                    torch.zeros_like(bias) if need_b else None) + (None,) * 4
        n, c = x.shape[:2]
        dx, dxs = _like(x, ctx.map) if need_x else (None, None)
        md = _map(dy)
        if md is None or md[1] != ctx.map[1]:           # another layout than x's: bring it into x's
            dy = _like(x, ctx.map)[0].copy_(dy)
            md = _map(dy)
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        _native.backward(x, ctx.map[0], dy, md[0], (n, c, x.numel() // (n * c)), weight, bias, stats, dx, dxs, dw, db, groups, act, slope)
        return dx, dw, db, None, None, None, None


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", slope=0.01):
    """act(group_norm(x, num_groups) * weight + bias) as one operator.

    x [N, C, space...] fp32, bf16 or fp16; channels last and channels first (the default) layouts are read as they lie, slices of
    either too, anything else is copied first; the result has x's type and layout.  weight, bias [C] or None, each fp32 or x's
    type or the other 16-bit one.  act: "none", "relu", "leaky_relu" (with `slope`), "silu".  Statistics (mean, biased variance of
    each image and group) are fp64.  A NaN or an infinity in a group makes that image's group NaN, and nothing else.
    Differentiable once (a WGAN-GP critic, whose penalty differentiates twice, keeps no norm, as in the reference)."""
    _check(x, num_groups, weight, bias, eps, act)
    eps, slope = float(eps), float(slope)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return GroupNormActFunction.apply(x, weight, bias, num_groups, eps, act, slope)
    return _forward(x.detach(), weight, bias, num_groups, eps, act, slope)[4]
