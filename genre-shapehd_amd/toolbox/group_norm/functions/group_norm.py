"""Group normalisation with the activation behind it, forward and backward (csrc/group_norm.hip, csrc/binding.cpp).

The reference's networks normalise over the batch (networks/networks.py:147-190); per-GPU batches of one to eight volumes, and
statistics that stay per rank, are what that serves worst (the refiner's innermost stage is 1^3: BatchNorm refuses to train on
one image).  Group statistics belong to one image: the result does not depend on the batch or on the ranks."""
from .._ext import training_lib as _native

ACTS = {"none": 0, "relu": 1, "leaky_relu": 2, "silu": 3}


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", slope=0.01):
    """act(group_norm(x, num_groups) * weight + bias) as one operator.

    x [N, C, space...] on a GPU, fp32, bf16 or fp16; channels last and channels first (the default) layouts are read as they lie,
    slices of either too, anything else is copied first; the result has x's type and layout.  weight, bias: [C] or None, of any of
    the three types.  act: "none", "relu", "leaky_relu" (with `slope`), "silu".  Statistics (mean and biased variance of each image
    and group) are fp64.  A NaN or an infinity makes its image's group NaN, and nothing else.  Differentiable once (a WGAN-GP
    critic, whose penalty differentiates twice, keeps no norm, as in the reference)."""
    code = ACTS.get(act)
    if code is None:
        raise RuntimeError("group_norm_act: act must be one of %s, got %r" % (sorted(ACTS), act))
    return _native.group_norm_act(x, num_groups, weight, bias, eps, code, slope)
