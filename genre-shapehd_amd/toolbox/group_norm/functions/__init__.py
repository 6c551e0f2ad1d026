"""`from toolbox.group_norm.functions import group_norm_act`"""
from . import group_norm as _m

GroupNormActFunction, group_norm_act = _m.GroupNormActFunction, _m.group_norm_act
__all__ = ["GroupNormActFunction", "group_norm_act"]
