"""The C entries of the training-step ops on what the PyTorch binding never asks of them.  Bounds: test_gpu_group_norm.py's."""
import ctypes as C
import sys

import pytest
import torch

from test_gpu_group_norm import SLOPE, definition, make, near

pytestmark = pytest.mark.gpu
CODES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3, torch.float64: 4}


@pytest.fixture(scope="module")
def entry(genre):
    """call(name, tensors and None, scalars): a C entry on the current stream"""
    L = sys.modules["_genre_shapehd_amd_loader"]
    lib = C.CDLL(L.LIB_PATH)
    lib.genre_last_error.restype = C.c_char_p
    lib.genre_group_norm_workspace.restype = C.c_int64

    def desc(t):
        if t is None:
            return None
        d = L.GenreTensor()
        d.data, d.ndim, d.dtype = t.data_ptr(), t.dim(), CODES[t.dtype]
        for i in range(t.dim()):
            d.size[i], d.stride[i] = t.size(i), t.stride(i)
        return C.byref(d)

    def call(name, tensors, scalars):
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert getattr(lib, name)(*map(desc, tensors), *scalars, stream) == 1, lib.genre_last_error()

    call.scratch = lambda x, groups, back, dev: torch.empty(max(1, lib.genre_group_norm_workspace(desc(x), C.c_int(groups), C.c_int(back))), dtype=torch.float64, device=dev)
    return call


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
@pytest.mark.parametrize("n,c,groups,s", ((1, 12, 3, 20), (2, 12, 3, 20), (1, 12, 3, 6000), (2, 12, 3, 6000)))
def test_parameter_gradients_have_types_of_their_own(genre, dev, entry, n, c, groups, s, last):
    """whatever the types of weight and bias, or with none: dw and db are written in theirs, and nothing behind them"""
    x, dy, w, b = make(dev, n, c, (s,), torch.float32, last)
    types = (None, torch.float32, torch.bfloat16, torch.float16)
    for k, (wt, gt) in enumerate((wt, gt) for wt in types for gt in types[1:]):
        bt, ht = types[(k + 1) % 4], types[1 + k % 3]
        print("types", n, s, last, wt, gt, bt, ht, flush=True)
        weight, bias = None if wt is None else w.to(wt), None if bt is None else b.to(bt)
        y, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(2, n, groups, dtype=torch.float64, device=dev)
        dw, db = torch.full((c + 64,), 7.0, dtype=gt, device=dev), torch.full((c + 64,), 7.0, dtype=ht, device=dev)
        entry("genre_group_norm_forward", (x, y, weight, bias, stats, entry.scratch(x, groups, 0, dev)), (C.c_int(groups), C.c_double(1e-5), C.c_int(3), C.c_float(SLOPE)))
        entry("genre_group_norm_backward", (x, dy, weight, bias, stats, dx, dw[:c], db[:c], entry.scratch(x, groups, 1, dev)), (C.c_int(groups), C.c_int(3), C.c_float(SLOPE)))
        want = definition(x, dy, weight, bias, groups, "silu", 1e-5, SLOPE)
        for got, name in ((y, "y"), (dx, "dx"), (dw[:c], "dw"), (db[:c], "db")):
            near(got, want[name], name)
        assert bool((dw[c:] == 7).all()) and bool((db[c:] == 7).all())
