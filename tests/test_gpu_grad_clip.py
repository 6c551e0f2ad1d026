"""grad_norm, clip_grads_, clip_adam_step_ against the definitions in float64.

Tolerances, before any run.  u = 2^-24 (half an fp32 step), t = finfo(type).eps / 2.
  norm      fp64 sums, one rounding: u |norm| (and 1e-12 for the sums)
  factor    norm + 1e-6, the quotient, max_norm and 1e-6 as fp32: 4 u, and the norm's own u: 5 u relative
  clipped   the product: (6 u + t) |g|, fp16 below its normal range 2^-25
  Adam      g' = g f + wd p: 6 u |g f| + 3 u |wd p|, call it G.  m: b1 and 1 - b1 rounded, two products and a sum (fused once):
            3 u |b1 m| + (1 - b1) (4 u |g'| + G);  v: the same, 3 u b2 v + (1 - b2) (5 u g'^2 + 2 |g'| G)
            p: the quotient q = m / (sqrt(v) k + eps): relative 7 u + dm / |m| + dv / (2 v), times the step size's 2 u:
            step |q| (10 u) + step dm / den + step |q| dv / (2 v) + (2 u + t) |p|, with step |q| <= lr sqrt-bounded by the values at hand"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tensors(dev, sizes, dtype=torch.float32, seed=0, scale=1.0, bucket=False):
    g = torch.Generator().manual_seed(seed)
    host = [(scale * torch.randn(s, generator=g)).to(dtype) for s in sizes]
    if not bucket:
        return [t.to(dev) for t in host]
    flat = torch.cat([t.flatten() for t in host]).to(dev)                # views one behind the other: no alignment
    return [v.view(s) for v, s in zip(flat.split([t.numel() for t in host]), sizes)]


def norm64(ts, kind=2.0):
    vs = [t.detach().double().cpu().flatten() for t in ts]
    v = torch.cat(vs) if vs else torch.zeros(1, dtype=torch.float64)
    return (v.norm() if kind == 2.0 else v.abs().max() if v.numel() else torch.tensor(0.0, dtype=torch.float64)).item()


LISTS = {
    "one value": [(1,)], "no values": [(0,), (3, 0)], "odd": [(1,), (7,), (0,), (33, 5), (4097,), (3, 1, 5)], "scalar": [()],
    "exact chunks": [(16384,), (4096,), (8192, 2)], "many": [(i % 7 + 1, i % 13 + 1) for i in range(450)], "large": [(64, 64, 8, 8, 8), (3,), (1000003,)],
}


@pytest.mark.parametrize("dtype", TYPES, ids=("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("name", LISTS)
def test_norms(genre, dev, name, dtype):
    for bucket in (False, True):
        ts = tensors(dev, LISTS[name], dtype, bucket=bucket)
        for kind in (2.0, math.inf):
            print("norm", name, dtype, bucket, kind, flush=True)
            want = norm64(ts, kind)
            got = genre.grad_norm(ts, norm_type=kind)
            assert got.dtype == torch.float32 and got.dim() == 0 and got.device == dev
            assert abs(got.item() - want) <= (U + 1e-12) * want


def test_norm_of_lists_of_several_types_and_of_one_tensor(genre, dev):
    ts = tensors(dev, [(100,), (5000,)]) + tensors(dev, [(3000,), (17,)], torch.bfloat16, 1) + tensors(dev, [(4100,)], torch.float16, 2)
    ts = [ts[i] for i in (4, 0, 2, 1, 3)]
    assert abs(genre.grad_norm(ts).item() - norm64(ts)) <= 1.1 * U * norm64(ts)
    assert genre.grad_norm(ts, "inf").item() == norm64(ts, math.inf)
    assert abs(genre.grad_norm(ts[0]).item() - norm64(ts[:1])) <= 1.1 * U * norm64(ts[:1])
    assert genre.grad_norm([]).item() == 0
    gap = ts[1][::3]                                                     # copied: only read
    assert abs(genre.grad_norm([gap]).item() - norm64([gap])) <= 1.1 * U * norm64([gap])
    assert abs(genre.grad_norm(t for t in ts).item() - norm64(ts)) <= 1.1 * U * norm64(ts)


def test_norms_at_the_ends_of_the_range(genre, dev):
    big = [torch.full((1000,), 1e30, device=dev), torch.full((10,), 1e-30, device=dev)]
    assert abs(genre.grad_norm(big).item() / (1e30 * math.sqrt(1000)) - 1) <= 2 * U      # squares beyond fp32
    tiny = [torch.full((1000,), 1e-30, device=dev)]
    assert abs(genre.grad_norm(tiny).item() / (1e-30 * math.sqrt(1000)) - 1) <= 2 * U
    for kind in (2.0, math.inf):
        ts = tensors(dev, [(5000,), (300,)])
        ts[1][7] = math.inf
        assert genre.grad_norm(ts, kind).item() == math.inf
        ts[0][4321] = math.nan
        assert math.isnan(genre.grad_norm(ts, kind).item())


def test_a_tensor_of_more_than_2_31_values(genre, dev):
    n = 2 ** 31 + 12345
    t = torch.full((n,), 2.0, dtype=torch.bfloat16, device=dev)
    t[-1] = -5
    want = math.sqrt(4.0 * (n - 1) + 25)
    assert genre.grad_norm([t], math.inf).item() == 5
    assert abs(genre.clip_grads_([t], want / 2).item() / want - 1) <= 2 * U          # a factor of 1/2 but for 1e-11
    assert t[-1].item() == -2.5 and t[:-1].min().item() == t[:-1].max().item() == 1


def factor64(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


@pytest.mark.parametrize("dtype", TYPES, ids=("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("name", ("odd", "many", "large", "one value", "no values"))
@pytest.mark.parametrize("max_norm,kind", ((0.5, 2.0), (1e9, 2.0), (0.25, math.inf), (0.0, 2.0)))
def test_clip(genre, dev, name, dtype, max_norm, kind):
    ts = tensors(dev, LISTS[name], dtype, bucket=True)
    before = [t.clone() for t in ts]
    want, versions = norm64(ts, kind), [t._version for t in ts]
    got = genre.clip_grads_(ts, max_norm, norm_type=kind)
    assert abs(got.item() - want) <= (U + 1e-12) * want
    f = factor64(want, max_norm)
    for t, b in zip(ts, before):
        if f == 1:
            assert torch.equal(t, b)
        off = (t.double() - f * b.double()).abs()
        assert bool((off <= (6 * U + half(dtype)) * f * b.double().abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-40)).all())
    assert all(t._version > v for t, v in zip(ts, versions))


def test_clip_of_a_model_as_torch_does_it(genre, dev):
    net = torch.nn.Sequential(torch.nn.Conv3d(2, 20, 4), torch.nn.BatchNorm3d(20), torch.nn.Linear(5, 3)).to(dev).to(memory_format=torch.channels_last_3d)
    ps = list(net.parameters())
    for p in ps[:-1]:
        p.grad = torch.randn_like(p)                                      # (the conv's gradient is channels last)
    copies = [p.detach().double().requires_grad_(True) for p in ps]
    for c, p in zip(copies, ps):
        c.grad = None if p.grad is None else p.grad.double()
    want = torch.nn.utils.clip_grad_norm_(copies, 0.7)
    got = genre.clip_grad_norm_(net.parameters(), 0.7)
    assert abs(got.item() / want.item() - 1) <= 2 * U
    for c, p in zip(copies[:-1], ps[:-1]):
        assert bool(((p.grad.double() - c.grad).abs() <= 7 * U * c.grad.abs()).all())
    assert ps[-1].grad is None
    assert genre.clip_grad_norm_(ps[-1], 1.0).item() == 0


def test_clip_with_infinities_and_nan(genre, dev):
    ts = tensors(dev, [(500,), (40,)])
    ts[0][3] = math.inf
    assert genre.clip_grads_(ts, 1.0).item() == math.inf
    assert math.isnan(ts[0][3].item()) and not ts[1].any()                # factor 0
    ts = tensors(dev, [(500,), (40,)])
    ts[0][3] = math.nan
    kept = [t.clone() for t in ts]
    with pytest.raises(RuntimeError):
        genre.clip_grads_(ts, 1.0, error_if_nonfinite=True)
    assert torch.equal(ts[1], kept[1])
    assert math.isnan(genre.clip_grads_(ts, 1.0).item()) and bool(ts[1].isnan().all())


def adam64(p, g, m, v, step, lr, betas, eps, wd, decoupled, f, dtype):
    p, g, m, v = (t.double().cpu() for t in (p, g, m, v))
    b1, b2 = betas
    ge = 6 * U * (g * f).abs() + (0 if decoupled else 3 * U * (wd * p).abs())
    gs = g * f + (0 if decoupled else wd * p)
    m2, v2 = b1 * m + (1 - b1) * gs, b2 * v + (1 - b2) * gs * gs
    me = 3 * U * (b1 * m).abs() + (1 - b1) * (4 * U * gs.abs() + ge)
    ve = 3 * U * b2 * v + (1 - b2) * (5 * U * gs * gs + 2 * gs.abs() * ge)
    size, root = lr / (1 - b1 ** step), math.sqrt(1 - b2 ** step)
    den = v2.sqrt() / root + eps
    q = m2 / den
    keep = 1 - lr * wd if decoupled else 1.0
    pe = size * (10 * U * q.abs() + me / den + q.abs() * ve / (2 * v2).clamp(min=1e-300)) + 2 * U * (p * keep).abs()
    p2 = p * keep - size * q
    return (p2, pe + half(dtype) * p2.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)), (m2, me + U * m2.abs()), (v2, ve + U * v2.abs())


@pytest.mark.parametrize("dtype", TYPES, ids=("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("name", ("odd", "many", "large"))
@pytest.mark.parametrize("step,wd,decoupled,max_norm", ((1, 0.0, False, None), (7, 0.1, False, 1.0), (1000, 0.1, True, 1e9), (3, 0.0, False, 0.0)))
def test_adam(genre, dev, name, dtype, step, wd, decoupled, max_norm):
    sizes = LISTS[name]
    p, g = tensors(dev, sizes, dtype, 1, 0.1, bucket=True), tensors(dev, sizes, dtype, 2, 0.3, bucket=True)
    m, v = tensors(dev, sizes, seed=3, scale=0.1), [t.square() + 1e-3 for t in tensors(dev, sizes, seed=4, scale=0.3)]
    norm = norm64(g)
    f = 1.0 if max_norm is None else factor64(norm, max_norm)
    args = dict(lr=1e-2, betas=(0.5, 0.9), eps=1e-8)
    want = [adam64(*t, step, 1e-2, (0.5, 0.9), 1e-8, wd, decoupled, f, dtype) for t in zip(p, g, m, v)]
    kept, versions = [t.clone() for t in g], [t._version for t in p + m + v]
    got = genre.clip_adam_step_(p, g, m, v, step, weight_decay=wd, decoupled=decoupled, max_norm=max_norm, **args)
    assert (got is None) == (max_norm is None)
    if got is not None:
        assert abs(got.item() - norm) <= 1.1 * U * norm
    assert all(torch.equal(a, b) for a, b in zip(g, kept))
    assert all(t._version > k for t, k in zip(p + m + v, versions))
    for i, w in enumerate(want):
        for t, (value, bound), what in zip((p[i], m[i], v[i]), w, "pmv"):
            off = (t.double().cpu() - value).abs()
            assert bool((off <= bound + 1e-38).all()), (what, i, off.max() if off.numel() else 0)


def test_adam_as_torch_does_it(genre, dev):
    """five steps of clip + Adam in float64 by torch: the errors of single steps (above) add up, 5 x (10 + 8) u of the update and of p"""
    sizes = [(40, 20, 4, 4, 4), (40,), (1,), (640, 64)]
    p, m, v = tensors(dev, sizes, seed=1, scale=0.1), [torch.zeros(s, device=dev) for s in sizes], [torch.zeros(s, device=dev) for s in sizes]
    ref = [t.double().requires_grad_(True) for t in p]
    opt = torch.optim.Adam(ref, lr=1e-2, betas=(0.5, 0.9))
    for step in range(1, 6):
        g = tensors(dev, sizes, seed=10 + step, scale=0.2)
        for r, t in zip(ref, g):
            r.grad = t.double()
        torch.nn.utils.clip_grad_norm_(ref, 3.0)
        opt.step()
        genre.clip_adam_step_(p, g, m, v, step, lr=1e-2, betas=(0.5, 0.9), max_norm=3.0)
    for t, r in zip(p, ref):
        # (a first step's quotient is +-1; a later one is m / sqrt(v) with m of either sign: its error is that of |m| before cancelling, <= 1)
        assert bool(((t.double() - r.detach()).abs() <= 5 * (20 * U * 1e-2 * 4 + 2 * U * r.detach().abs())).all())


def test_layouts_of_weights_and_states(genre, dev):
    shape = (6, 5, 4, 4, 4)
    p = torch.randn(shape, device=dev).to(memory_format=torch.channels_last_3d)
    g, m, v = torch.randn_like(p), torch.zeros_like(p), torch.zeros_like(p)
    q, h = p.clone(memory_format=torch.contiguous_format), g.clone(memory_format=torch.contiguous_format)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    genre.clip_adam_step_([p], [g], [m], [v], 1, max_norm=1.0)
    genre.clip_adam_step_([q], [h], [a], [b], 1, max_norm=1.0)
    # (the norm's partial sums are cut along memory: its last bit may differ, and with it m, v; a first step's quotient is +-1)
    assert bool(((p - q).abs() <= 4 * U * q.abs() + 20 * U * 1e-3).all()) and bool(((m - a).abs() <= 8 * U * a.abs()).all())
    with pytest.raises(RuntimeError):
        genre.clip_adam_step_([p], [h], [m], [v], 2)                      # gradient in another layout
    with pytest.raises(RuntimeError):
        genre.clip_grads_([torch.ones(1, device=dev).expand(5)], 1.0)
    with pytest.raises(RuntimeError):
        genre.clip_grads_([torch.ones(10, device=dev)[::2]], 1.0)


def test_strides_of_dimensions_of_one_value_do_not_matter(genre, dev):
    """the gradient of a channels-last weight with one output channel may come with any stride there"""
    p, g = (torch.randn(1, 8, 4, 4, 4, device=dev).to(memory_format=torch.channels_last_3d) for _ in range(2))
    m, v, q = torch.zeros_like(p), torch.zeros_like(p), p.clone()
    other = g.as_strided(g.shape, (1, *g.stride()[1:]))
    assert other.stride() != p.stride() and torch.equal(other, g)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    genre.clip_adam_step_([p], [other], [m], [v], 1, max_norm=1.0)
    genre.clip_adam_step_([q], [g], [a], [b], 1, max_norm=1.0)
    assert torch.equal(p, q) and torch.equal(m, a) and torch.equal(v, b)


def test_weights_that_are_no_numbers_keep_their_moments_clean(genre, dev):
    """without weight decay a gradient does not depend on its weight; an infinite weight stays one"""
    for dtype in TYPES:
        p, g = tensors(dev, [(37,)], dtype, 1)[0], tensors(dev, [(37,)], dtype, 2)[0]
        q = p.clone()
        p[3], p[36], p[20] = math.inf, -math.inf, math.nan
        a, b, c, d = (torch.zeros(37, device=dev) for _ in range(4))
        genre.clip_adam_step_([p], [g], [a], [b], 1, max_norm=1.0)
        genre.clip_adam_step_([q], [g], [c], [d], 1, max_norm=1.0)
        assert torch.equal(a, c) and torch.equal(b, d)
        assert p[3].item() == math.inf and p[36].item() == -math.inf and math.isnan(p[20].item())
        p[3], p[36], p[20] = q[3], q[36], q[20]
        assert torch.equal(p, q)


def test_refusals(genre, dev):
    t, s = [torch.zeros(4, device=dev)], [torch.zeros(4, device=dev)]
    for bad in (lambda: genre.grad_norm(t, 1.0), lambda: genre.grad_norm([torch.zeros(3)]), lambda: genre.grad_norm([t[0].double()]),
                lambda: genre.clip_grads_(t, -1.0), lambda: genre.clip_grads_(t, math.nan), lambda: genre.grad_norm(t + [torch.zeros(2)]),
                lambda: genre.grad_norm([torch.zeros(4, device=dev).to_sparse()]), lambda: genre.clip_adam_step_(t, t, s, [], 1),
                lambda: genre.clip_adam_step_(t, s, s, s, 0), lambda: genre.clip_adam_step_(t, s, s, s, 1, betas=(1.0, 0.9)),
                lambda: genre.clip_adam_step_(t, [s[0].half()], s, s, 1), lambda: genre.clip_adam_step_([t[0].half()], [s[0].half()], [s[0].half()], s, 1),
                lambda: genre.clip_adam_step_(t, [s[0][:3]], s, s, 1), lambda: genre.clip_adam_step_(t, s, s, s, 1, lr=-1.0)):
        with pytest.raises(RuntimeError):
            bad()


def test_tensors_that_share_memory_are_refused(genre, dev):
    """before anything is written; gradients may be the same tensor, as nothing writes them"""
    flat = torch.ones(5000, device=dev)
    a, b = flat[:3000], flat[2999:]
    for ts in ([a, b], [b, a], [a, a], [flat, flat[7:8]], [a, flat[3000:], a.view(60, 50)]):
        with pytest.raises(RuntimeError, match="shares memory"):
            genre.clip_grads_(ts, 1.0)
    p, m, v = (tensors(dev, [(3000,), (3000,)], seed=s, scale=0.1) for s in (1, 2, 3))
    v = [t.abs() for t in v]
    g = tensors(dev, [(3000,)], seed=4)
    kept = [t.clone() for t in p + m + v]
    for lists in (([p[0], p[0]], g * 2, m, v), (p, g * 2, [m[0]] * 2, v), (p, g * 2, m, m), (p, [g[0], p[0]], m, v), (p, g * 2, m, [v[0], m[1]])):
        with pytest.raises(RuntimeError, match="shares memory"):
            genre.clip_adam_step_(*lists, 1, max_norm=1.0)
    assert bool((flat == 1).all()) and all(torch.equal(t, k) for t, k in zip(p + m + v, kept))
    genre.clip_grads_([flat[:3000], flat[3000:], flat[9:9]], 1e9)
    genre.clip_adam_step_(p, g * 2, m, v, 1)
    assert not torch.equal(p[0], kept[0])


def test_streams_and_graphs(genre, dev):
    """captured norm + clip and clip + Adam, replayed with eager work and synchronisations between: the same bits as eager calls"""
    sizes = LISTS["odd"] + LISTS["many"][:250]
    g, p = tensors(dev, sizes, seed=1, bucket=True), tensors(dev, sizes, seed=2)
    m, v = [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]
    flat = g[0]._base
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        genre.clip_grads_([t.clone() for t in g], 1.0)
    torch.cuda.current_stream().wait_stream(side)
    clip, adam = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(clip):
        norm1 = genre.clip_grads_(g, 1.0)
    with torch.cuda.graph(adam):
        norm2 = genre.clip_adam_step_(p, g, m, v, 3, max_norm=0.5)
    for turn in range(3):
        flat.normal_()
        eg = [t.clone() for t in g]
        ep, em, ev = ([t.clone() for t in ts] for ts in (p, m, v))
        n1 = genre.clip_grads_(eg, 1.0)
        n2 = genre.clip_adam_step_(ep, eg, em, ev, 3, max_norm=0.5)
        torch.cuda.synchronize()
        clip.replay()
        adam.replay()
        torch.cuda.synchronize()
        assert norm1.item() == n1.item() and norm2.item() == n2.item()
        for a, b in zip(g + p + m + v, eg + ep + em + ev):
            assert torch.equal(a, b)
    a = genre.grad_norm(g)
    with torch.cuda.stream(side):
        b = genre.grad_norm(g)
    torch.cuda.synchronize()
    assert a.item() == b.item()
