"""`from toolbox.group_norm.functions import group_norm_act`"""
from . import group_norm as _m

group_norm_act = _m.group_norm_act
__all__ = ["group_norm_act"]
