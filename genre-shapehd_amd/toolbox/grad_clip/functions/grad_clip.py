"""The norm of all gradients together, clipping by it, and the Adam step that takes the clip with it (csrc/grad_clip.hip).

Each is a handful of launches for the whole list of tensors, whatever its length, and waits for nothing: norm and factor stay on
the GPU.  Tensors are fp32, bf16 or fp16 (mixed lists too), on one GPU, gap-free in memory (any order of dimensions); no alignment
is asked for beyond the type's, so views into flat gradient buckets are fine.  (The reference steps its optimiser on the
gradients as they come, train.py:137-214.)"""
import math

import torch

from .._ext import Many, grad_lib as _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _list(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _gap_free(t):
    """whether t's values fill one block of memory, in some order of its dimensions"""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return t.numel() == 0
        expect *= size
    return True


def _check(op, tensors, dev=None, written=False):
    """the tensors on one GPU; gap-free ones as they are, others refused where they are `written`, else copied"""
    out = tensors
    for i, t in enumerate(tensors):
        if not t.is_cuda or (dev is not None and t.device != dev):
            raise RuntimeError("%s: tensor %d is on %s; all must be on one GPU -- there is no CPU path" % (op, i, t.device))
        dev = t.device
        if t.layout is not torch.strided or t.dtype not in _TYPES:
            raise RuntimeError("%s: tensor %d is %s %s; dense fp32, bf16 or fp16 tensors only" % (op, i, t.layout, t.dtype))
        if not t.is_contiguous() and not _gap_free(t):
            if written:
                raise RuntimeError("%s: tensor %d %s with strides %s has gaps or overlaps and cannot be written in place"
                                   % (op, i, tuple(t.shape), t.stride()))
            out = list(out) if out is tensors else out
            out[i] = t.contiguous()
    return out


def _kind(op, norm_type):
    p = float(norm_type)
    if p not in (2.0, math.inf):
        raise RuntimeError("%s: norm_type must be 2 or inf, got %r" % (op, norm_type))
    return 2 if p == 2.0 else 0


def _bound(op, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError("%s: max_norm must not be negative, got %r" % (op, max_norm))
    return max_norm


def grad_norm(tensors, norm_type=2.0):
    """norm of the vector of all the tensors' values (2: Euclidean, fp64 sums; inf: the largest magnitude) as an fp32 tensor of no
    dimensions on their GPU.  NaN where a value is NaN.  An empty list has the norm 0 (on the CPU, as nothing names a GPU)."""
    kind = _kind("grad_norm", norm_type)
    tensors = _list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    tensors = _check("grad_norm", tensors)
    out = torch.empty(2, dtype=torch.float32, device=tensors[0].device)
    _native.norm(Many(tensors), kind, math.inf, out)
    return out[0]


def clip_grads_(tensors, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """scale the tensors in place by min(1, max_norm / (norm + 1e-6)), norm = grad_norm(tensors, norm_type), and return the norm.
    A norm of infinity scales by 0 (infinities become NaN), NaN makes all NaN; error_if_nonfinite raises before anything is
    written instead, for which it waits for the GPU."""
    kind, max_norm = _kind("clip_grads_", norm_type), _bound("clip_grads_", max_norm)
    tensors = _list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    _check("clip_grads_", tensors, written=True)
    many = Many(tensors)
    out = torch.empty(2, dtype=torch.float32, device=many.device)
    _native.norm(many, kind, max_norm, out)
    if error_if_nonfinite and not math.isfinite(out[0].item()):
        raise RuntimeError("clip_grads_: the norm of the gradients is %r" % out[0].item())
    _native.scale(many, out[1:])
    torch.autograd.graph.increment_version(tensors)
    return out[0]


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """clip_grads_ on the gradients of `parameters` (a tensor, or any iterable of them; those without a gradient are passed over):
    what torch.nn.utils.clip_grad_norm_ does"""
    return clip_grads_([p.grad for p in _list(parameters) if p.grad is not None], max_norm, norm_type, error_if_nonfinite)


def clip_adam_step_(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False,
                    max_norm=None, norm_type=2.0):
    """one Adam step on `params` in place, `exp_avgs` and `exp_avg_sqs` with them, as if clip_grads_(grads, max_norm, norm_type) had
    run before -- without writing the gradients.  step counts from 1.  weight_decay is added to the gradient, or (decoupled) shrinks
    the weights by lr * weight_decay.  params[i] and grads[i] have one type and layout, the states are fp32 in that layout.
    Returns the norm of the gradients before the clip (None without max_norm)."""
    kind = _kind("clip_adam_step_", norm_type)
    lists = [_list(ts) for ts in (params, grads, exp_avgs, exp_avg_sqs)]
    if any(len(ts) != len(lists[0]) for ts in lists):
        raise RuntimeError("clip_adam_step_: the four lists have %s tensors" % [len(ts) for ts in lists])
    if max_norm is not None:
        max_norm = _bound("clip_adam_step_", max_norm)
    beta1, beta2 = map(float, betas)
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and lr >= 0 and eps >= 0 and weight_decay >= 0 and step >= 1):
        raise RuntimeError("clip_adam_step_: betas in [0, 1), lr, eps and weight_decay not negative and step from 1 are wanted, got %r"
                           % ((betas, lr, eps, weight_decay, step),))
    if not lists[0]:
        return None if max_norm is None else torch.tensor(0.0)
    dev = lists[0][0].device
    for ts in lists:
        _check("clip_adam_step_", ts, dev, written=True)
    for i, (p, g, m, v) in enumerate(zip(*lists)):
        if g.dtype != p.dtype or m.dtype != torch.float32 or v.dtype != torch.float32:
            raise RuntimeError("clip_adam_step_: tensor %d: gradient %s for %s, states %s and %s (fp32 is wanted)" % (i, g.dtype, p.dtype, m.dtype, v.dtype))
        if not (p.shape == g.shape == m.shape == v.shape and (p.stride() == g.stride() == m.stride() == v.stride()
                                                                  or (p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and v.is_contiguous()))):
            raise RuntimeError("clip_adam_step_: tensor %d: weight, gradient and states differ in shape or layout" % i)
    norm = factor = None
    if max_norm is not None:
        out = torch.empty(2, dtype=torch.float32, device=dev)
        _native.norm(Many(lists[1]), kind, max_norm, out)
        norm, factor = out[0], out[1:]
    _native.adam(Many(*lists), factor, int(step), float(lr), beta1, beta2, float(eps), float(weight_decay), decoupled)
    for ts in (lists[0], lists[2], lists[3]):
        torch.autograd.graph.increment_version(ts)
    return norm
