"""The training-step ops without a GPU: what the C entries refuse before any launch, what Python refuses, how networks are built."""
import ctypes as C
import math
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(genre):
    import sys
    L = sys.modules["_genre_shapehd_amd_loader"]
    lib = C.CDLL(L.LIB_PATH)
    lib.genre_last_error.restype = C.c_char_p
    for name in ("genre_group_norm_workspace", "genre_grad_workspace"):
        getattr(lib, name).restype = C.c_int64
    return L, lib


def desc(L, shape, stride=None, dtype=0, ptr=0x1000):
    d = L.GenreTensor()
    d.data, d.ndim, d.dtype = ptr, len(shape), dtype
    at = 1
    for i in reversed(range(len(shape))):
        d.size[i], d.stride[i] = shape[i], at if stride is None else stride[i]
        at *= shape[i]
    return C.byref(d)


F64 = 4


def test_group_norm_entries(lib):
    L, lib = lib

    def forward(x=None, y=None, w=None, b=None, stats=None, ws=None, groups=2, eps=1e-5, act=1):
        x = x or desc(L, (2, 6, 50000))
        return lib.genre_group_norm_forward(x, y or x, w, b, stats or desc(L, (2, 2, 2), dtype=F64), ws or desc(L, (1 << 20,), dtype=F64), C.c_int(groups),
                                            C.c_double(eps), C.c_int(act), C.c_float(0.1), None)

    def backward(x=None, dy=None, dx=None, dw=None, stats=None, ws=None, groups=2, act=1):
        x = x or desc(L, (2, 6, 50000))
        return lib.genre_group_norm_backward(x, dy or x, None, None, stats or desc(L, (2, 2, 2), dtype=F64), dx, dw, None, ws or desc(L, (1 << 20,), dtype=F64),
                                             C.c_int(groups), C.c_int(act), C.c_float(0.1), None)

    def refused(rc, word):
        assert rc == 0 and word in lib.genre_last_error(), lib.genre_last_error()

    for call in (forward, backward):
        refused(call(groups=4), b"split")
        refused(call(groups=0), b"split")
        refused(call(act=7), b"activation")
        refused(call(x=desc(L, (2, 6, 50000), dtype=1)), b"fp32, bf16 or fp16")
        refused(call(x=desc(L, (2, 6, 5, 10000))), b"[N,C,S]")
        refused(call(x=desc(L, (2, 6, 50000), stride=(600000, 100000, 2))), b"channels last")
        refused(call(stats=desc(L, (2, 2), dtype=F64)), b"stats")
        refused(call(stats=desc(L, (2, 2, 2))), b"stats")
        refused(call(ws=desc(L, (3,), dtype=F64)), b"ws")
        refused(call(ws=desc(L, (1 << 20,), dtype=F64, ptr=0x1008)), b"16 bytes")
    refused(forward(eps=0.0), b"eps")
    refused(forward(eps=math.nan), b"eps")
    refused(forward(y=desc(L, (2, 6, 50001))), b"shape")
    refused(forward(y=desc(L, (2, 6, 50000), dtype=2)), b"dtype")
    refused(forward(y=desc(L, (2, 6, 50000), stride=(300000, 1, 6))), b"all be channels last")
    refused(forward(w=desc(L, (5,))), b"weight")
    refused(forward(b=desc(L, (6,), stride=(2,))), b"bias")
    refused(backward(dx=desc(L, (2, 6, 49999))), b"shape")
    refused(backward(dw=desc(L, (6,), dtype=1)), b"dw")
    assert lib.genre_group_norm_workspace(desc(L, (2, 6, 50000)), 4, 0) == -1
    assert lib.genre_group_norm_workspace(desc(L, (2, 6, 50)), 2, 0) == 0                  # one workgroup a group: no scratch
    assert lib.genre_group_norm_workspace(desc(L, (2, 6, 50000)), 2, 0) > 0


@pytest.mark.parametrize("dtype", (0, 2))
@pytest.mark.parametrize("n,c,groups", ((1, 16, 4), (1, 640, 8), (2, 16, 4), (3, 5000, 2), (1, 20000, 1), (2, 40000, 2), (1, 70000, 2), (5, 99999, 3)))
def test_scratch_of_one_position_serves_both_layouts(lib, n, c, groups, dtype):
    """a [N, C, 1] map is channels last and channels first at once; which of them a call is, the other maps may decide"""
    L, lib = lib
    need = lambda stride, back: lib.genre_group_norm_workspace(desc(L, (n, c, 1), stride=stride, dtype=dtype), C.c_int(groups), C.c_int(back))
    for back in (0, 1):
        both, first = need((c, 1, 1), back), need((2 * c, 2, 1), back)
        assert both >= first >= 0


def test_list_entries(lib):
    L, lib = lib
    i64, i32, ptr = lambda *v: (C.c_int64 * len(v))(*v), lambda *v: (C.c_int32 * len(v))(*v), lambda *v: (C.c_void_p * len(v))(*v)
    out, ws = desc(L, (2,)), desc(L, (1 << 16,), dtype=F64)

    def norm(p=ptr(0x1000, 0x2000), n=i64(5, 6), t=i32(0, 2), count=2, kind=2, most=1.0, out=out, ws=ws):
        return lib.genre_grad_norm(p, n, t, C.c_int(count), C.c_int(kind), C.c_float(most), out, ws, None)

    def refused(rc, word):
        assert rc == 0 and word in lib.genre_last_error(), lib.genre_last_error()

    refused(norm(t=i32(0, 1)), b"fp32, bf16 or fp16")
    refused(norm(n=i64(5, -6)), b"values")
    refused(norm(n=i64(1 << 45, 1 << 45)), b"values")
    refused(norm(p=ptr(0x1000, None)), b"NULL")
    refused(norm(p=None), b"NULL")
    refused(norm(kind=3), b"norm_type")
    refused(norm(most=-1.0), b"max_norm")
    refused(norm(most=math.nan), b"max_norm")
    refused(norm(out=desc(L, (1,))), b"out")
    refused(norm(ws=desc(L, (1,), dtype=F64)), b"ws")
    refused(norm(count=-1), b"list")
    refused(lib.genre_grad_scale(ptr(0x1000), i64(3), i32(0), C.c_int(1), None, None), b"factor")
    four = [ptr(0x1000)] * 4

    def adam(lists=four, step=1, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0):
        return lib.genre_adam_step(*lists, i64(3), i32(0), C.c_int(1), None, C.c_int64(step), C.c_double(lr), C.c_double(b1), C.c_double(b2), C.c_double(eps),
                                   C.c_double(wd), C.c_int(0), None)

    refused(adam(step=0), b"step")
    refused(adam(b1=1.0), b"betas")
    refused(adam(b2=math.nan), b"betas")
    refused(adam(lr=-1.0), b"negative")
    refused(adam(wd=math.nan), b"negative")
    refused(adam(lists=four[:2] + [ptr(None)] + four[:1]), b"m of tensor 0")
    assert lib.genre_grad_workspace(i64(5, -1), 2) == -1


def test_no_cpu_path(genre):
    t = torch.zeros(2, 4, 3)
    for call in (lambda: genre.group_norm_act(t, 2), lambda: genre.grad_norm([t]), lambda: genre.clip_grads_([t], 1.0), lambda: genre.clip_adam_step_([t], [t], [t], [t], 1),
                 lambda: genre.GroupNormAct(2, 4)(t)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        genre.ClipAdam([p], max_grad_norm=1.0).step()


def test_arguments(genre):
    t = [torch.zeros(3)]
    for call in (lambda: genre.group_norm_act(t[0], 2, act="gelu"), lambda: genre.grad_norm(t, 1), lambda: genre.clip_grads_(t, -1.0), lambda: genre.clip_grads_(t, math.nan),
                 lambda: genre.clip_adam_step_(t, t, t, [], 1), lambda: genre.clip_adam_step_(t, t, t, t, 0), lambda: genre.clip_adam_step_(t, t, t, t, 1, betas=(0.9, 1.0)),
                 lambda: genre.clip_adam_step_(t, t, t, t, 1, max_norm=1.0, factor=t[0]), lambda: genre.grad_norm([1])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: genre.GroupNormAct(3, 4), lambda: genre.GroupNormAct(0, 4), lambda: genre.ClipAdam(t, max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            call()
    assert genre.grad_norm([]).item() == genre.clip_grads_([], 1.0).item() == genre.clip_grad_norm_([torch.nn.Parameter(t[0])], 1.0).item() == 0
    assert genre.clip_adam_step_([], [], [], [], 1) is None


def test_networks_with_group_norm(genre):
    from genre_shapehd_amd import networks as N
    from genre_shapehd_amd.models import GenReNet, GenReOptions
    for build in (lambda **k: N.Unet_3D(nf=4, **k), lambda **k: N.VoxelDecoder(n_dims=8, nf=32, **k), lambda **k: N.VoxelGenerator(nz=8, nf=4, **k)):
        batch, group = build(), build(norm="group")
        names = {k for k in batch.state_dict() if "running" not in k and "num_batches" not in k}
        assert set(group.state_dict()) == names
        assert all(group.state_dict()[k].shape == batch.state_dict()[k].shape for k in names)
        assert not any(isinstance(m, torch.nn.BatchNorm3d) for m in group.modules())
        group.load_state_dict(batch.state_dict(), strict=False)
        with pytest.raises(ValueError):
            build(norm="layer")
    assert any(isinstance(m, genre.GroupNormAct) for m in GenReNet(GenReOptions(norm="group")).refine_net.modules())


def test_the_plain_optimiser_stays_the_default(genre):
    from genre_shapehd_amd.optim import adam
    ps = [torch.nn.Parameter(torch.zeros(3))]
    assert type(adam(ps, 1e-3, (0.5, 0.9))) is torch.optim.Adam
    clip = adam(ps, 1e-3, (0.5, 0.9), 2.0)
    assert type(clip) is genre.ClipAdam and clip.max_grad_norm == 2.0 and clip.param_groups[0]["betas"] == (0.5, 0.9)


def test_copies_of_an_optimiser_keep_its_bound(genre):
    import copy
    import pickle
    opt = genre.ClipAdam([torch.nn.Parameter(torch.zeros(3))], lr=0.5, max_grad_norm=2.0)
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert again.max_grad_norm == 2.0 and again.grad_norm is None and again.param_groups[0]["lr"] == 0.5
        again.step()
