"""The native ops behind this package: the object of genre-shapehd_amd/_loader.py, located from this file's own path and shared
process-wide, so that it is the same one whether this tree is imported as `genre_shapehd_amd.toolbox...` or as `toolbox...`."""
import importlib.util
import os
import sys

_NAME = "_genre_shapehd_amd_loader"


def _loader():
    if _NAME in sys.modules:
        return sys.modules[_NAME]
    here = os.path.dirname(os.path.abspath(__file__))
    pkg = os.path.normpath(os.path.join(here, *([".."] * 3)))
    spec = importlib.util.spec_from_file_location(_NAME, os.path.join(pkg, "_loader.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules[_NAME] = mod
    try:
        spec.loader.exec_module(mod)
    except BaseException:
        del sys.modules[_NAME]
        raise
    return mod


training_lib = _loader().training_lib
