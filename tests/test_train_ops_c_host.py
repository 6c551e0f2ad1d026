"""The C entries of the training-step ops without a GPU: sizes that no tensor has are refused, and end no process."""
import ctypes as C

import pytest

from test_train_ops_host import F64, desc, lib  # noqa: F401

I64 = 1 << 62


def entries(L, lib, x, groups=2, act=1):
    """{name: the refusal of one map by every entry that takes one}"""
    big, stats = desc(L, (1 << 20,), dtype=F64), desc(L, (2, 2, 2), dtype=F64)
    g, a, s = C.c_int(groups), C.c_int(act), C.c_float(0.1)
    calls = {"workspace": lambda: lib.genre_group_norm_workspace(x, g, C.c_int(0)) + 1, "backward workspace": lambda: lib.genre_group_norm_workspace(x, g, C.c_int(1)) + 1,
             "forward": lambda: lib.genre_group_norm_forward(x, x, None, None, stats, big, g, C.c_double(1e-5), a, s, None),
             "backward": lambda: lib.genre_group_norm_backward(x, x, None, None, stats, x, None, None, big, g, a, s, None)}
    return {name: (call(), lib.genre_last_error()) for name, call in calls.items()}


@pytest.mark.parametrize("shape,stride,word", (
    ((2, 6, -5), (30, 5, 1), b"negative size"), ((-2, 6, 50000), (300000, 50000, 1), b"negative size"), ((-2, 6, -50000), (300000, 50000, 1), b"negative size"),
    ((2, -6, 50), (300, 50, 1), b"negative size"), ((2, 6, 50), (300, -50, 1), b"negative size or stride"),
    ((2, 6, I64), (0, I64, 1), b"2^60"), ((2, 6, I64 // 4 + 3), (0, I64, 1), b"2^60"), ((1, 1 << 20, 1 << 44), (0, 1 << 44, 1), b"2^60")))
def test_sizes_that_no_map_has(lib, shape, stride, word):  # noqa: F811
    L, lib = lib
    for name, (rc, error) in entries(L, lib, desc(L, shape, stride=stride)).items():
        assert rc == 0 and word in error, (name, error)


def test_more_threads_than_a_launch_holds(lib):  # noqa: F811
    """workgroups times threads of 2^32 or more, in the one-workgroup form and in two passes: refused before any launch, and before
    the caller allocates scratch"""
    L, lib = lib
    rows = lambda n: desc(L, (n, 8, 1), stride=(8, 1, 8))
    for name, (rc, error) in entries(L, lib, rows(1 << 26), groups=1).items():
        assert rc == 0 and b"too large for one launch" in error, (name, error)
    assert lib.genre_group_norm_workspace(rows((1 << 26) - 1), C.c_int(1), C.c_int(0)) == 0
    odd = lambda n: desc(L, (n, 4, 3), stride=(12, 3, 1))                  # (planes of an odd number of positions: the backward takes two passes)
    got = entries(L, lib, odd(1 << 24), groups=1)
    assert got["workspace"][0] == 1                                       # (0 values)
    for name in ("backward workspace", "backward"):
        rc, error = got[name]
        assert rc == 0 and b"too large for one launch" in error, (name, error)
    assert lib.genre_group_norm_workspace(odd((1 << 24) - 64), C.c_int(1), C.c_int(1)) > 0


@pytest.mark.parametrize("dtype", (0, 2, 3), ids=("fp32", "bf16", "fp16"))
def test_where_one_workgroup_ends(lib, dtype):  # noqa: F811
    """a call of one image that takes the one-workgroup form needs no scratch"""
    L, lib = lib

    def one(cg, s, last, back):
        d = desc(L, (1, 2 * cg, s), stride=(2 * cg * s, 1, 2 * cg) if last else (2 * cg * s, s, 1), dtype=dtype)
        return lib.genre_group_norm_workspace(d, C.c_int(2), C.c_int(back)) == 0

    for cg, s in ((1, 16384), (4, 4096), (64, 256), (1024, 16), (1023, 16)):
        for last in (False, True):
            assert one(cg, s, last, 0) and not one(cg, s + 1, last, 0), (cg, s, last)
            assert not one(cg, s, last, 1)
    for cg, s in ((1, 8192), (4, 2048), (64, 128), (512, 16)):
        assert one(cg, s, True, 1) and not one(cg, s + 1, True, 1) and not one(cg, s, False, 1), (cg, s)
    for cg, s in ((1, 4096), (4, 1024), (64, 64), (512, 8)):
        assert one(cg, s, False, 1) and not one(cg, s + 4, False, 1), (cg, s)
    for last in (False, True):
        assert one(1024, 4, last, 0) and not one(1025, 4, last, 0)
    assert not one(4, 1023, False, 1) and one(4, 1023, True, 1)            # (an odd number of positions: two passes backward)
