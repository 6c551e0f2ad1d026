"""The norm of all gradients together, clipping by it, and the Adam step that takes the clip with it (csrc/grad_clip.hip).

Each is a handful of launches for the whole list of tensors, whatever its length, and waits for nothing: norm and factor stay on
the GPU.  Tensors are fp32, bf16 or fp16 (mixed lists too), on one GPU, gap-free in memory (any order of dimensions); no alignment
is asked for beyond the type's, so views into flat gradient buckets are fine.  (The reference steps its optimiser on the
gradients as they come, train.py:137-214.)"""
import math

import torch

from .._ext import training_lib as _native


def _list(tensors):
    return tensors if isinstance(tensors, (list, tuple)) else [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _kind(op, norm_type):
    p = float(norm_type)
    if p != 2.0 and p != math.inf:
        raise RuntimeError("%s: norm_type must be 2 or inf, got %r" % (op, norm_type))
    return 2 if p == 2.0 else 0


def _bound(op, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError("%s: max_norm must not be negative, got %r" % (op, max_norm))
    return max_norm


def grad_norm(tensors, norm_type=2.0):
    """norm of the vector of all the tensors' values (2: Euclidean, fp64 sums; inf: the largest magnitude) as an fp32 tensor of no
    dimensions on their GPU.  NaN where a value is NaN.  It carries no gradient.  An empty list
    has the norm 0 (on the CPU, as nothing names a GPU)."""
    kind, tensors = _kind("grad_norm", norm_type), _list(tensors)
    return _native.grad_norm(tensors, math.inf, kind)[0] if tensors else torch.tensor(0.0)


def clip_grads_(tensors, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """scale the tensors in place by min(1, max_norm / (norm + 1e-6)), norm = grad_norm(tensors, norm_type), and return the norm.
    A norm of infinity scales by 0 (infinities become NaN), NaN makes all NaN; error_if_nonfinite raises before anything is
    written instead, for which it waits for the GPU.  Tensors that share memory, or one that is listed twice, are refused."""
    kind, max_norm, tensors = _kind("clip_grads_", norm_type), _bound("clip_grads_", max_norm), _list(tensors)
    if error_if_nonfinite:
        tensors = tuple(tensors)                                          # (other threads run while it waits: the list stays what it was)
    return _native.clip_grads(tensors, max_norm, kind, error_if_nonfinite) if tensors else torch.tensor(0.0)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """clip_grads_ on the gradients of `parameters` (a tensor, or any iterable of them; those without a gradient are passed over):
    what torch.nn.utils.clip_grad_norm_ does"""
    return clip_grads_([p.grad for p in _list(parameters) if p.grad is not None], max_norm, norm_type, error_if_nonfinite)


def clip_adam_step_(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False,
                    max_norm=None, norm_type=2.0, factor=None):
    """one Adam step on `params` in place, `exp_avgs` and `exp_avg_sqs` with them, as if clip_grads_(grads, max_norm, norm_type) had
    run before -- without writing the gradients.  step counts from 1 (a captured call replays with the one it was given).
    weight_decay is added to the gradient, or (decoupled) shrinks the weights by lr * weight_decay.  params[i] and grads[i]
    have one type and layout, the states are fp32 in that layout; tensors that share memory are refused (gradients may, with each
    other).  Returns the norm of the gradients before the clip (None without max_norm).
    factor (instead of max_norm): one fp32 value on the same GPU that the gradients are multiplied by -- for weights that are
    stepped in several calls under one clip."""
    kind = _kind("clip_adam_step_", norm_type)
    if factor is not None and max_norm is not None:
        raise RuntimeError("clip_adam_step_: max_norm or factor, not both")
    params, grads, exp_avgs, exp_avg_sqs = lists = [_list(ts) for ts in (params, grads, exp_avgs, exp_avg_sqs)]
    if any(len(ts) != len(params) for ts in lists):
        raise RuntimeError("clip_adam_step_: the four lists have %s tensors" % [len(ts) for ts in lists])
    if max_norm is not None:
        max_norm = _bound("clip_adam_step_", max_norm)
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1 and lr >= 0 and eps >= 0 and weight_decay >= 0 and step >= 1):
        raise RuntimeError("clip_adam_step_: betas in [0, 1), lr, eps and weight_decay not negative and step from 1 are wanted, got %r"
                           % ((betas, lr, eps, weight_decay, step),))
    if not params:
        return None if max_norm is None else torch.tensor(0.0)
    return _native.adam_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, beta1, beta2, eps, weight_decay, decoupled, max_norm, kind, factor)
