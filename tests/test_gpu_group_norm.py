"""group_norm_act against the definition in float64: forward, gradients, layouts, types, strides, and where it can go wrong.

Tolerances, before any run.  u = 2^-24 (half an fp32 step, relative), t = finfo(type).eps / 2.  Statistics and z are fp64 in the
kernels, so only what follows rounds:
  none, relu   y: z to fp32, then to the type: (u + t) |y|
  leaky_relu   one fp32 product with a slope that is itself rounded: (3 u + t) |y|
  silu         exp2(z log2 e): the constant and the product are off by |z| u each, exp2 and the reciprocal by 2 u, the sum, the
               last product and z itself by u (z's rounding moves the result by |z| u more): (8 u + 3 |z| u + t) |y|
  gradients    dz = dy act'(z) is off by E: 0 (none, relu), 2 u |dz| (leaky), and for silu s (1 + z (1 - s)) with s off by
               (6 + 3 |z|) u: E <= u (12 + 6 |z|) (1 + |z|) |dy|.  All sums are fp64:
               dx: r (|w| E + mean |w| E + |h| mean |w| E |h|) + (u + t) |dx|;  dw: sum E |h| + u-or-t |dw|;  db: sum E + ...
fp16 results below its normal range are off by up to 2^-25 absolutely (fp32's 2^-150 does not matter, nor does bf16's).  fp64 is
not exact either: every product and sum rounds by 2^-53 of ITS size, and the terms of dx may cancel (one value a group: dx = 0 =
r w dz - r m1), so D = 2^-47 -- 64 such roundings: the few of a term and those of a tree of sums over a map -- of the terms' sizes is added:
dx: D r (|w dz| + mean |w dz| + |h| mean |w dz h|);  dw: D sum |dz h|;  db: D sum |dz|;  y: D (|h w| + |b|).  The mean rounds by
2^-53 of itself, which moves h by up to d = D r |mean| and with it y by |w| d, silu's dz by |w dy| d (its slope's slope is below 1),
dx by r d (mean |w dz h| + |h| mean |w dz|) and dw by d sum |dz|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U, D = 2.0 ** -24, 2.0 ** -47
SLOPE = 0.2
ACTS = ("none", "relu", "leaky_relu", "silu")
TYPES = (torch.float32, torch.bfloat16, torch.float16)
LAST = {2: None, 3: None, 4: torch.channels_last, 5: torch.channels_last_3d}


def to_last(t):
    """the same values with the channels innermost in memory"""
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def make(dev, n, c, space, dtype, last, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, *space, generator=g) * (0.3 + torch.randn(1, c, *[1] * len(space), generator=g).abs()) + mean
    dy = torch.randn(n, c, *space, generator=g)
    w, b = 1 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    x, dy = x.to(dtype).to(dev), dy.to(dtype).to(dev)
    if last:
        x, dy = to_last(x), to_last(dy)
    return x, dy, w.to(dev), b.to(dev)


def definition(x, dy, w, b, groups, act, eps, slope):
    """y, dx, dw, db and their bounds, from the inputs' values in float64 on the host"""
    x, dy = x.detach().double().cpu(), dy.detach().double().cpu()
    n, c = x.shape[:2]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.detach().double().cpu()
    xs, dys = x.reshape(n, groups, -1), dy.reshape(n, c, -1)
    mean = xs.mean(2, keepdim=True)
    r = 1 / ((xs - mean).square().mean(2, keepdim=True) + eps).sqrt()
    h = ((xs - mean) * r).reshape(n, c, -1)
    z = h * w[:, None] + b[:, None]
    s = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp(min=0), "leaky_relu": torch.where(z > 0, z, z * slope), "silu": z * s}[act]
    d = {"none": torch.ones_like(z), "relu": (z > 0).double(), "leaky_relu": torch.where(z > 0, 1.0, slope).double(),
         "silu": s * (1 + z * (1 - s))}[act]
    dz = dys * d
    e = {"none": 0 * z, "relu": 0 * z, "leaky_relu": 2 * U * dz.abs(), "silu": U * (12 + 6 * z.abs()) * (1 + z.abs()) * dys.abs()}[act]

    off = D * (r * mean.abs()).expand(n, groups, c // groups).reshape(n, c, 1)
    if act == "silu":
        e = e + off * (w[:, None] * dys).abs()

    def group_mean(v):
        return v.reshape(n, groups, -1).mean(2, keepdim=True).expand(n, groups, c // groups).reshape(n, c, 1)

    rc = r.expand(n, groups, c // groups).reshape(n, c, 1)
    wz = w[:, None] * dz
    dx = rc * (wz - group_mean(wz) - h * group_mean(wz * h))
    we = w.abs()[:, None] * e
    we = we + D * wz.abs()
    dx_e = rc * (we + group_mean(we) + h.abs() * group_mean(we * h.abs()) + off * (group_mean((wz * h).abs()) + h.abs() * group_mean(wz.abs())))
    e = e + D * dz.abs()
    dw_e = (off * dz.abs()).sum((0, 2))
    y_e = {"none": 1, "relu": 1, "leaky_relu": 3, "silu": 8 + 3 * z.abs()}[act] * U * y.abs() + D * ((h * w[:, None]).abs() + b.abs()[:, None]) + off * w.abs()[:, None]
    return {"y": (y.reshape(x.shape), y_e.reshape(x.shape)), "dx": (dx.reshape(x.shape), dx_e.reshape(x.shape) + U * dx.abs().reshape(x.shape)),
            "dw": ((dz * h).sum((0, 2)), (e * h.abs()).sum((0, 2)) + dw_e), "db": (dz.sum((0, 2)), e.sum((0, 2)))}


def near(got, want, what):
    value, bound = want
    t = torch.finfo(got.dtype).eps / 2
    bound = bound + t * value.abs() + (2.0 ** -25 if got.dtype == torch.float16 else 0) + 1e-35
    off = (got.detach().double().cpu() - value).abs()
    assert got.shape == value.shape
    assert bool((off <= bound).all()), "%s: off by %g where %g is allowed" % (what, off.max(), bound.flatten()[(off - bound).argmax()])


def run(G, x, dy, w, b, groups, act, eps=1e-5, slope=SLOPE):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = G.group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=eps, act=act, slope=slope)
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    return {"y": y.detach(), "dx": next(grads), "dw": None if w is None else next(grads), "db": None if b is None else next(grads)}


def check(G, x, dy, w, b, groups, act, eps=1e-5, slope=SLOPE):
    got, want = run(G, x, dy, w, b, groups, act, eps, slope), definition(x, dy, w, b, groups, act, eps, slope)
    for k, v in got.items():
        if v is not None:
            near(v, want[k], "%s %s %s %s" % (k, tuple(x.shape), x.dtype, act))
    assert got["y"].dtype == got["dx"].dtype == x.dtype
    return got


SHAPES = [
    (1, 1, 1, (4,)), (2, 6, 3, (1, 1, 1)), (2, 8, 2, ()), (1, 5, 5, (33,)), (1, 640, 8, (1, 1, 1)), (2, 12, 12, (3, 3)),
    (3, 20, 4, (5, 7, 3)), (2, 45, 5, (23, 17)), (1, 1, 1, (70, 3)), (1, 1023, 3, (3, 5)), (2, 1030, 2, (9,)), (1, 4104, 8, (2, 3)),
    (1, 16, 1, (1, 2, 3)), (9, 3, 3, (2,)), (2, 80, 8, (16, 15, 14)),
    # groups of more values than one workgroup holds (65536 forward, 32768 backward), of more channels, and at the border
    # (the borders that the first kernels had; where they lie now, test_gpu_group_norm_borders.py has both sides of them)
    (2, 45, 1, (41, 40)), (1, 511, 1, (13, 11)), (1, 1030, 2, (9, 15)), (1, 1030, 1, (3,)), (1, 4104, 2, (5, 7)), (2, 7, 1, (101, 97)), (1, 3, 1, (40001,)),
    (1, 64, 2, (32, 32)), (1, 64, 2, (32, 33)), (1, 64, 1, (32, 32)), (1, 64, 1, (32, 33)), (1, 96, 1, (700,)),
    # more groups or channels than a second pass adds up itself; columns that run over a row's end; one channel
    (1, 40, 8, (64, 64, 20)), (1, 1500, 1, (40,)), (1, 45, 5, (91, 93)), (1, 1001, 1, (7, 5, 2)), (1, 300, 1, (15, 16)), (2, 1, 1, (257, 259)), (3, 65, 65, (210, 160)),
]


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
@pytest.mark.parametrize("dtype", TYPES, ids=("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("n,c,groups,space", SHAPES)
def test_against_the_definition(genre, dev, n, c, groups, space, dtype, last):
    for k, act in enumerate(ACTS):
        print("group norm", n, c, groups, space, dtype, last, act, flush=True)
        x, dy, w, b = make(dev, n, c, space, dtype, last, seed=k)
        got = check(genre, x, dy, w, b, groups, act)
        assert got["y"].stride() == x.stride() and got["dx"].stride() == x.stride()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16), ids=("fp32", "bf16"))
@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
def test_maps_of_many_workgroups(genre, dev, dtype, last):
    x, dy, w, b = make(dev, 2, 20, (48, 47, 46), dtype, last)
    check(genre, x, dy, w, b, 4, "leaky_relu")


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
@pytest.mark.parametrize("c,lo,hi", ((40, 8, 28), (41, 3, 18), (9, 2, 3)))
def test_slices_of_the_channels_are_read_where_they_lie(genre, dev, c, lo, hi, last):
    x, dy, w, b = make(dev, 2, c, (6, 5, 7), torch.float32, last)
    xs, dys = x[:, lo:hi], dy[:, lo:hi]
    before = x.clone()
    check(genre, xs, dys, w[lo:hi].contiguous(), b[lo:hi].contiguous(), 1 if hi - lo == 1 else 5, "relu")
    assert torch.equal(x, before)


def test_odd_addresses_and_orders(genre, dev):
    w, b = 1 + 0.1 * torch.randn(6, device=dev), 0.1 * torch.randn(6, device=dev)
    for dtype in TYPES:
        flat = torch.randn(2 * 6 * 35 + 1, device=dev).to(dtype)[1:]                       # one value off 16 bytes
        x = flat.view(2, 6, 5, 7)
        dy = torch.randn(2, 6, 5, 7, device=dev).to(dtype)
        check(genre, x, dy, w, b, 2, "silu")
        check(genre, flat.view(2, 5, 7, 6).permute(0, 3, 1, 2), dy, w, b, 2, "silu")       # channels last; dy channels first
        check(genre, flat.view(2, 6, 7, 5).transpose(2, 3), to_last(dy), w, b, 2, "silu")  # neither: copied
        check(genre, flat.view(6, 2, 5, 7).transpose(0, 1), dy, w, b, 2, "silu")           # images innermost but one
        check(genre, x[:, :, 1:4, ::2], dy[:, :, :3, :4], w, b, 3, "relu")
        check(genre, x[:1].expand(3, 6, 5, 7), torch.randn(3, 6, 5, 7, device=dev).to(dtype), w, b, 2, "relu")
        check(genre, x[:, :1].expand(2, 6, 5, 7), dy, w, b, 2, "none")
        check(genre, x.view(2, 6, 35)[:, :, 3], dy[:, :, 0, 0], w, b, 2, "none")


def test_expanded_output_gradient_and_missing_parameters(genre, dev):
    x, dy, w, b = make(dev, 2, 8, (5, 6), torch.float32, True)
    leaf = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
    genre.group_norm_act(leaf, 2, w, b, act="silu").sum().backward()                       # a gradient of strides 0
    near(leaf.grad, definition(x, torch.ones_like(x), w, b, 2, "silu", 1e-5, SLOPE)["dx"], "dx")
    check(genre, x, dy, None, None, 4, "relu")
    check(genre, x, dy, w, None, 4, "relu")
    check(genre, x, dy, None, b, 4, "relu")


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
def test_parameters_of_other_types(genre, dev, last):
    for dtype in TYPES:
        x, dy, w, b = make(dev, 2, 12, (5, 6), torch.bfloat16, last)
        check(genre, x, dy, w.to(dtype), b.to(dtype), 3, "silu")
        check(genre, x, dy, w.to(dtype).repeat(2).view(12, 2)[:, 0], b, 3, "none")         # strided


def test_gradients_that_are_not_wanted(genre, dev):
    x, dy, w, b = make(dev, 2, 12, (5, 6), torch.float32, True)
    want = definition(x, dy, w, b, 3, "relu", 1e-5, SLOPE)
    for needed in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(k)) for t, k in zip((x, w, b), needed)]
        genre.group_norm_act(*leaves[:1], 3, *leaves[1:], act="relu").backward(dy)
        for t, name, k in zip(leaves, ("dx", "dw", "db"), needed):
            assert (t.grad is not None) == bool(k)
            if k:
                near(t.grad, want[name], name)
    y = genre.group_norm_act(x, 3, w, b, act="relu")
    assert not y.requires_grad
    near(y, want["y"], "y")
    with torch.no_grad():
        assert torch.equal(genre.group_norm_act(x.requires_grad_(True), 3, w, b, act="relu"), y)
    with torch.inference_mode():
        assert torch.equal(genre.group_norm_act(x.detach(), 3, w, b, act="relu"), y)


def test_nothing_to_normalise(genre, dev):
    for shape in ((0, 6, 4, 4), (2, 6, 0, 4), (0, 6)):
        x = torch.empty(shape, device=dev, requires_grad=True)
        w, b = torch.ones(6, device=dev, requires_grad=True), torch.zeros(6, device=dev, requires_grad=True)
        y = genre.group_norm_act(x, 2, w, b, act="relu")
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()


def test_constant_groups_and_single_values(genre, dev):
    """a deviation of zero: h = 0 exactly, y = act(b), and no gradient reaches x"""
    for last in (False, True):
        x = torch.full((2, 6, 3, 5), 7.25, device=dev)
        x = to_last(x) if last else x
        _, dy, w, b = make(dev, 2, 6, (3, 5), torch.float32, last)
        got = check(genre, x, dy, w, b, 3, "silu")
        assert torch.equal(got["y"], to_last(got["y"])) and bool((got["dw"] == 0).all())
    x, dy, w, b = make(dev, 2, 6, (1, 1), torch.float32, False)                            # one value a group
    got = check(genre, x, dy, w, b, 6, "none")
    assert torch.equal(got["y"][0, :, 0, 0], b)


def test_levels_far_from_zero(genre, dev):
    """|mean| of 3e4 deviations: fp32 sums of squares would leave nothing of the variance"""
    for last in (False, True):
        x, dy, w, b = make(dev, 2, 8, (9, 11, 10), torch.float32, last, mean=3e4)
        check(genre, x, dy, w, b, 2, "relu")
    x, dy, w, b = make(dev, 1, 4, (50, 40), torch.float32, False)
    check(genre, x * 1e25, dy, w, b, 2, "none")                                            # squares beyond fp32's range
    check(genre, x * 1e-25, dy, w, b, 2, "none")


@pytest.mark.parametrize("bad", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
def test_one_bad_value_spoils_its_group_only(genre, dev, bad, last):
    x, dy, w, b = make(dev, 3, 10, (5, 9), torch.float32, last)
    clean = run(genre, x, dy, w, b, 5, "silu")
    x[1, 3, 2, 4] = bad                                                                    # image 1, group 1 (channels 2, 3)
    got = run(genre, x, dy, w, b, 5, "silu")
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, 2:4] = True
    for k in ("y", "dx"):
        assert bool(got[k][hit].isnan().all()) and torch.equal(got[k][~hit], clean[k][~hit])
    for k in ("dw", "db"):
        assert bool(got[k][2:4].isnan().all())
        assert torch.equal(got[k][[0, 1, 4, 5, 6, 7, 8, 9]], clean[k][[0, 1, 4, 5, 6, 7, 8, 9]])


@pytest.mark.parametrize("bad", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
def test_a_relu_that_is_off_passes_nothing_on(genre, dev, bad, last):
    """whatever the gradient holds there: the same bits as with zeros in its place (one workgroup a group, and two passes)"""
    for space in ((5, 9), (90, 91)):
        x, dy, w, b = make(dev, 2, 8, space, torch.float32, last)
        off = run(genre, x, dy, w, b, 2, "relu")["y"] == 0
        want = run(genre, x, dy.masked_fill(off, 0.0), w, b, 2, "relu")
        got = run(genre, x, dy.masked_fill(off, bad), w, b, 2, "relu")
        for k in got:
            assert bool(got[k].isfinite().all()) and torch.equal(got[k], want[k])


def test_gradients_against_differences(genre, dev):
    """the smooth activation, central differences of the operator's own fp32 forward summed in float64: the step h = 2^-6 leaves a
    truncation of h^2 / 6 times the third derivative of the loss (below 40 here: |r| <= 4, |dy| <= 3, few terms) = 2e-3 and a rounding of
    sum |dy| u |y| / h <= 1e-3"""
    x, dy, w, b = make(dev, 1, 4, (3, 5), torch.float32, True, seed=3)
    got = run(genre, x, dy, w, b, 2, "silu")

    def loss(x, w, b):
        return (genre.group_norm_act(x, 2, w, b, act="silu").double() * dy.double()).sum().item()

    h = 2.0 ** -6
    for name, t in (("dx", x), ("dw", w), ("db", b)):
        for at in range(0, t.numel(), 3):
            idx = tuple(int(i) for i in torch.unravel_index(torch.tensor(at), t.shape))
            args = {"x": x.clone(), "w": w.clone(), "b": b.clone()}
            args[name[1]][idx] = t[idx] + h
            up = loss(**args)
            args[name[1]][idx] = t[idx] - h
            assert abs((up - loss(**args)) / (2 * h) - got[name][idx].item()) <= 3e-3, (name, idx)


def test_same_inputs_same_bits_on_another_stream(genre, dev):
    for last in (False, True):
        x, dy, w, b = make(dev, 2, 40, (20, 21, 22), torch.float32, last)
        first = run(genre, x, dy, w, b, 8, "leaky_relu")
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            second = run(genre, x, dy, w, b, 8, "leaky_relu")
        third = run(genre, x, dy, w, b, 8, "leaky_relu")                                   # at once with it
        torch.cuda.synchronize()
        for k in first:
            assert torch.equal(first[k], second[k]) and torch.equal(first[k], third[k])


def test_captured_and_replayed(genre, dev):
    """two graphs of forward + backward replayed in turn, with eager calls and synchronisations between, on new inputs each time"""
    shapes = ((2, 20, (6, 7, 8), True), (3, 8, (9, 10), False))
    graphs = []
    for n, c, space, last in shapes:
        x, dy, w, b = make(dev, n, c, space, torch.float32, last)
        leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(True) for t in (x, w, b)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                torch.autograd.grad(genre.group_norm_act(leaves[0], 4, *leaves[1:], act="silu"), leaves, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = genre.group_norm_act(leaves[0], 4, *leaves[1:], act="silu")
            grads = torch.autograd.grad(y, leaves, dy)
            y = y.detach()
        graphs.append((graph, leaves, dy, y, grads))
    for turn in range(3):
        wants = []
        for graph, leaves, dy, y, grads in graphs:
            with torch.no_grad():
                leaves[0].normal_()
                dy.normal_()
            wants.append(run(genre, leaves[0], dy, *leaves[1:], 4, "silu"))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (graph, leaves, dy, y, grads), want in zip(graphs, wants):
            assert torch.equal(y, want["y"])
            for got, k in zip(grads, ("dx", "dw", "db")):
                assert torch.equal(got, want[k])


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
def test_maps_of_more_than_2_31_values(genre, dev, last):
    """channels of +1 and -1: mean 0, deviation 1, so r = 1 / sqrt(1 + eps), y = +-r, dx = r (1 - r^2) dy for dy = x, dw = r S, db = +-S"""
    s = 2 ** 30 + 40
    x = torch.ones((1, s, 2) if last else (1, 2, s), dtype=torch.bfloat16, device=dev)
    x = x.transpose(1, 2) if last else x
    x[:, 1].neg_()
    w, b = torch.ones(2, device=dev, requires_grad=True), torch.zeros(2, device=dev, requires_grad=True)
    dy, leaf = x.clone(), x.requires_grad_(True)
    y = genre.group_norm_act(leaf, 1, w, b, eps=0.25)
    dx, dw, db = torch.autograd.grad(y, (leaf, w, b), dy)
    r = 1 / math.sqrt(1.25)
    for got, value in ((y.detach(), r), (dx, r * (1 - r * r))):
        for c, sign in ((0, 1), (1, -1)):
            lo, hi = got[0, c].min().item(), got[0, c].max().item()
            assert lo == hi and abs(lo - sign * value) <= (2.0 ** -9 + U) * value
    assert abs(dw[0].item() / (r * s) - 1) <= 2 * U and abs(dw[1].item() / (r * s) - 1) <= 2 * U
    assert abs(db[0].item() / s - 1) <= 2 * U and abs(db[1].item() / s + 1) <= 2 * U


def test_under_autocast(genre, dev):
    """types are what is given: a bf16 map with fp32 parameters, inside autocast as outside"""
    x, dy, w, b = make(dev, 2, 12, (5, 6), torch.bfloat16, True)
    want = run(genre, x, dy, w, b, 3, "silu")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = run(genre, x, dy, w, b, 3, "silu")
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_as_torch_has_it(genre, dev):
    """the layers that GroupNormAct replaces, in float64 (nn.GroupNorm behind a state_dict of the same keys)"""
    ours = genre.GroupNormAct(4, 20, act="leaky_relu", slope=0.01).to(dev)
    with torch.no_grad():
        ours.weight.normal_()
        ours.bias.normal_()
    stock = torch.nn.GroupNorm(4, 20).double().to(dev)
    stock.load_state_dict(ours.state_dict())
    x = torch.randn(2, 20, 5, 6, 7, device=dev)
    want = torch.nn.functional.leaky_relu(stock(x.double()), 0.01)
    off = (ours(x).double() - want).abs()
    assert bool((off <= 4 * U * want.abs() + 1e-12).all())


def test_second_derivatives_are_refused(genre, dev):
    x = torch.randn(1, 4, 3, device=dev, requires_grad=True)
    g, = torch.autograd.grad(genre.group_norm_act(x, 2, act="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals(genre, dev):
    x, w = torch.zeros(2, 6, 4, device=dev), torch.ones(6, device=dev)
    for bad in (lambda: genre.group_norm_act(x, 4), lambda: genre.group_norm_act(x, 0), lambda: genre.group_norm_act(x.double(), 2),
                lambda: genre.group_norm_act(x, 2, w[:5]), lambda: genre.group_norm_act(x, 2, w.double()), lambda: genre.group_norm_act(x, 2, w.cpu()),
                lambda: genre.group_norm_act(x, 2, act="tanh"), lambda: genre.group_norm_act(x, 2, eps=0.0), lambda: genre.group_norm_act(x[0, 0], 2),
                lambda: genre.group_norm_act(x.cpu(), 2)):
        with pytest.raises(RuntimeError):
            bad()
