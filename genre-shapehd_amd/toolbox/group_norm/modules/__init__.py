"""`from toolbox.group_norm.modules import GroupNormAct`"""
from . import group_norm as _m

GroupNormAct = _m.GroupNormAct
__all__ = ["GroupNormAct"]
