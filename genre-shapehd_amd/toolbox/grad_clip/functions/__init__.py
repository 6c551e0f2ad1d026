"""`from toolbox.grad_clip.functions import grad_norm, clip_grads_, clip_grad_norm_, clip_adam_step_`"""
from . import grad_clip as _m

__all__ = ["grad_norm", "clip_grads_", "clip_grad_norm_", "clip_adam_step_"]
globals().update({name: getattr(_m, name) for name in __all__})
