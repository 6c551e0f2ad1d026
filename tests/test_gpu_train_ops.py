"""Group norm, clip and Adam as the training step uses them together: networks with norm="group", ClipAdam, the training command.
Bounds are those of test_gpu_group_norm.py and test_gpu_grad_clip.py, held by every operator on what it was really given."""
import pytest
import torch

from test_gpu_grad_clip import U, adam64, factor64, norm64
from test_gpu_group_norm import LAST, definition, near

pytestmark = pytest.mark.gpu


def networks(genre):
    from genre_shapehd_amd import networks
    return networks


def watch(net, genre):
    """{module: what its group norm read, gave and received} of the next forward and backward"""
    seen, hooks = {}, []

    def forward(m, args, y):
        x, s = args[0], seen.setdefault(m, {})
        s["x"], s["y"] = x.detach().clone(), y.detach().clone()
        x.register_hook(lambda g, s=s: s.__setitem__("dx", g.detach().clone()))
        y.register_hook(lambda g, s=s: s.__setitem__("dy", g.detach().clone()))

    for m in net.modules():
        if isinstance(m, genre.GroupNormAct):
            hooks.append(m.register_forward_hook(forward))
    return seen, hooks


@pytest.mark.parametrize("layout", ("first", "last"))
@pytest.mark.parametrize("kind", ("decoder", "generator"))
def test_a_training_step_of_a_decoder(genre, dev, kind, layout):
    torch.manual_seed(0)
    N = networks(genre)
    net = (N.VoxelDecoder(n_dims=12, nf=32, norm="group") if kind == "decoder" else N.VoxelGenerator(nz=12, nf=4, res=64, norm="group")).to(dev)
    if layout == "last":
        net = net.to(memory_format=LAST[5])
    opt = genre.ClipAdam(net.parameters(), lr=1e-3, betas=(0.5, 0.9), max_grad_norm=1e-3)
    for step in (1, 2):
        seen, hooks = watch(net, genre)
        code = torch.randn(2, 12, 1, 1, 1, device=dev)
        opt.zero_grad(set_to_none=True)
        out = net(code)
        torch.nn.functional.mse_loss(out, torch.rand_like(out)).backward()
        for h in hooks:
            h.remove()
        assert len(seen) == (5 if kind == "decoder" else 4)
        for m, s in seen.items():
            want = definition(s["x"], s["dy"], m.weight, m.bias, m.num_groups, m.act, m.eps, m.slope)
            for got, k in ((s["y"], "y"), (s["dx"], "dx"), (m.weight.grad, "dw"), (m.bias.grad, "db")):
                near(got, want[k], "%s of %s" % (k, tuple(s["x"].shape)))
        ps = list(net.parameters())
        grads, before = [p.grad.clone() for p in ps], [p.detach().clone() for p in ps]
        states = [(opt.state[p].get("exp_avg", torch.zeros_like(p)).clone(), opt.state[p].get("exp_avg_sq", torch.zeros_like(p)).clone()) for p in ps]
        opt.step()
        norm = norm64(grads)
        f = factor64(norm, 1e-3)
        assert abs(opt.grad_norm.item() - norm) <= 1.1 * U * norm and f < 1
        for p, b, g, (m, v) in zip(ps, before, grads, states):
            assert torch.equal(p.grad, g)
            for got, (value, bound) in zip((p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"]), adam64(b, g, m, v, step, 1e-3, (0.5, 0.9), 1e-8, 0.0, False, f, p.dtype)):
                assert bool(((got.detach().double().cpu() - value).abs() <= bound + 1e-38).all())
            assert float(opt.state[p]["step"]) == step


def test_the_refiner_trains_on_one_image(genre, dev):
    """its innermost map is 1^3: batch statistics of one image do not exist, group statistics do"""
    N = networks(genre)
    x = torch.rand(1, 2, 128, 128, 128, device=dev)
    with pytest.raises(ValueError):
        N.Unet_3D(nf=2).to(dev)(x)
    net = N.Unet_3D(nf=2, norm="group").to(dev)
    seen, hooks = watch(net, genre)
    net(x).square().mean().backward()
    assert len(seen) == 11
    for m, s in seen.items():
        want = definition(s["x"], s["dy"], m.weight, m.bias, m.num_groups, m.act, m.eps, m.slope)
        near(s["y"], want["y"], "y")
        near(s["dx"], want["dx"], "dx")
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in net.parameters())


def test_an_image_does_not_depend_on_its_batch(genre, dev):
    x, w, b = torch.randn(4, 40, 9, 10, 11, device=dev), torch.randn(40, device=dev), torch.randn(40, device=dev)
    for last in (False, True):
        x = x.contiguous(memory_format=LAST[5] if last else torch.contiguous_format)
        whole = genre.group_norm_act(x, 8, w, b, act="silu")
        for i in range(4):
            near(genre.group_norm_act(x[i:i + 1], 8, w, b, act="silu"),
                 definition(x[i:i + 1], torch.zeros_like(x[i:i + 1]), w, b, 8, "silu", 1e-5, 0.01)["y"], "alone")
            near(whole[i:i + 1], definition(x[i:i + 1], torch.zeros_like(x[i:i + 1]), w, b, 8, "silu", 1e-5, 0.01)["y"], "in the batch")


# ---- ClipAdam ---------------------------------------------------------------------------------------------------
def weights(dev, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(dtype).to(dev)) for s in ((20, 7, 3, 3), (20,), (1,), (33, 65))]


def test_steps_with_parameters_that_come_and_go(genre, dev):
    """a parameter without a gradient keeps its moments and its count; the others go on: torch.optim.Adam in float64 says where to.
    Bound: each of 4 steps adds that of test_gpu_grad_clip's five, 20 u lr 4 + 2 u |p|"""
    ps = weights(dev)
    ref = [p.detach().double().requires_grad_(True) for p in ps]
    opt = genre.ClipAdam([{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3, "weight_decay": 0.01}], lr=1e-2, betas=(0.5, 0.9), max_grad_norm=2.0)
    stock = torch.optim.Adam([{"params": ref[:2]}, {"params": ref[2:], "lr": 5e-3, "weight_decay": 0.01}], lr=1e-2, betas=(0.5, 0.9))
    for step in range(4):
        g = torch.Generator().manual_seed(100 + step)
        for i, (p, r) in enumerate(zip(ps, ref)):
            p.grad = None if (step + i) % 3 == 0 else torch.randn(p.shape, generator=g).to(dev)
            r.grad = None if p.grad is None else p.grad.double()
        torch.nn.utils.clip_grad_norm_(ref, 2.0)
        stock.step()
        opt.step()
    for p, r in zip(ps, ref):
        assert float(opt.state[p]["step"]) == float(stock.state[r]["step"])
        assert bool(((p.double() - r).abs() <= 4 * (20 * U * 1e-2 * 4 + 2 * U * r.abs())).all())


def test_states_go_to_torch_and_back(genre, dev, tmp_path):
    from genre_shapehd_amd.models import checkpoint
    for dtype in (torch.float32, torch.bfloat16):
        ps = weights(dev, 1, dtype)
        opt = genre.ClipAdam(ps, lr=1e-2, betas=(0.5, 0.9), max_grad_norm=1.0)
        for p in ps:
            p.grad = torch.randn_like(p)
        opt.step()
        net = torch.nn.Module()
        net.ps = torch.nn.ParameterList(ps)
        path = str(tmp_path / "c.pt")
        checkpoint.save_state_dict(path, [net], [opt], epoch=3)
        others = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        again = genre.ClipAdam(others, lr=1e-2, betas=(0.5, 0.9), max_grad_norm=1.0)
        stock = torch.optim.Adam([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1e-2, betas=(0.5, 0.9))
        net2 = torch.nn.Module()
        net2.ps = torch.nn.ParameterList(others)
        assert checkpoint.load_state_dict(path, [net2], [again])["epoch"] == 3
        stock.load_state_dict(opt.state_dict())
        for p, o, s in zip(ps, others, stock.param_groups[0]["params"]):
            assert float(stock.state[s]["step"]) == float(again.state[o]["step"]) == 1
            o.grad = p.grad.clone()
        if dtype == torch.float32:                                        # (torch keeps bf16 moments: rounded on the way)
            opt.step()
            again.step()
            assert all(torch.equal(p, o) for p, o in zip(ps, others))
        # a state that torch's Adam wrote
        third = genre.ClipAdam([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1e-2, betas=(0.5, 0.9))
        third.load_state_dict(stock.state_dict())
        for p, q in zip(third.param_groups[0]["params"], ps):
            p.grad = torch.ones_like(p)
        third.step()
        assert all(st["exp_avg"].dtype == torch.float32 and float(st["step"]) == 2 for st in third.state.values())


def test_gradients_and_moments_in_another_layout(genre, dev):
    """the same bits (no bound: no sum whose order a layout changes) when gradients, or weights after the first step, change it"""
    def build():
        torch.manual_seed(5)
        ps = [torch.nn.Parameter(torch.randn(s, device=dev)) for s in ((6, 5, 4, 4, 4), (1, 3, 2, 2, 2), (7,))]
        return ps, genre.ClipAdam(ps, lr=1e-2)

    last = lambda t: t.to(memory_format=torch.channels_last_3d) if t.dim() == 5 else t
    plain, opt = build()
    other, opt2 = build()
    for step in range(3):
        g = torch.Generator().manual_seed(step)
        if step == 1:
            for p in other:
                p.data = last(p.data)
        for p, q in zip(plain, other):
            p.grad = torch.randn(p.shape, generator=g).to(dev)
            q.grad = p.grad.clone() if step == 2 else last(p.grad)
        opt.step()
        opt2.step()
        assert all(torch.equal(p, q) for p, q in zip(plain, other))
        assert all(torch.equal(opt.state[p][k], opt2.state[q][k]) for p, q in zip(plain, other) for k in ("exp_avg", "exp_avg_sq"))
    assert other[0].is_contiguous(memory_format=torch.channels_last_3d) and opt2.state[other[0]]["exp_avg"].stride() == other[0].stride()


def test_a_step_without_a_bound_and_one_without_gradients(genre, dev):
    ps = weights(dev, 2)
    opt = genre.ClipAdam(ps, lr=1e-2)
    before = [p.detach().clone() for p in ps]
    assert opt.step(lambda: 3.0) == 3.0
    assert all(torch.equal(p, b) for p, b in zip(ps, before)) and opt.grad_norm is None
    for p in ps:
        p.grad = 5 * torch.ones_like(p)
    opt.step()
    assert opt.grad_norm is None
    # a first step of constant gradients: m / sqrt(v) = 1, so p falls by lr (g / (g + eps)): 12 u lr + 2 u |p|
    assert all(bool(((p - (b - 1e-2)).abs() <= 12 * U * 1e-2 + 3 * U * b.abs() + 1e-10).all()) for p, b in zip(ps, before))


def test_weights_that_a_graph_still_needs_are_seen_to_change(genre, dev):
    """in-place steps count as such: a backward through what a step has overwritten raises, as after torch's optimisers"""
    p = torch.nn.Parameter(torch.randn(5, device=dev))
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    genre.ClipAdam([p]).step()
    with pytest.raises(RuntimeError):
        loss.backward()


def test_a_step_is_not_captured(genre, dev):
    p = torch.nn.Parameter(torch.ones(5, device=dev))
    p.grad = torch.ones_like(p)
    opt = genre.ClipAdam([p], max_grad_norm=1.0)
    opt.step()
    graph, kept = torch.cuda.CUDAGraph(), p.detach().clone()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    assert torch.equal(p, kept) and float(opt.state[p]["step"]) == 1


def test_what_autograd_guards(genre, dev):
    """a map changed between forward and backward raises; a result changed in place does not matter, as the map is what is kept;
    a second backward through a retained graph gives the same"""
    x, w = torch.randn(2, 8, 4, 4, device=dev, requires_grad=True), torch.ones(8, device=dev, requires_grad=True)
    leaf = x * 1
    y = genre.group_norm_act(leaf, 2, w, act="silu")
    first = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    again = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    z = y.mul_(2)
    assert all(torch.equal(2 * a, b) for a, b in zip(first, torch.autograd.grad(z.sum(), (x, w), retain_graph=True)))
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_broadcast_inputs(genre, dev):
    """one image for a whole batch, one weight for all channels: their gradients are the sums of what each copy gets, which are those
    of the copies laid out (bits; the sums over four and eight fp32 terms are torch's, (n - 1) u of the terms' magnitudes apart at most)"""
    for shape in ((1, 8, 5, 9), (1, 8, 60, 71)):
        x, w, b, dy = torch.randn(shape, device=dev), torch.randn(1, device=dev), torch.randn(8, device=dev), torch.randn(4, *shape[1:], device=dev)
        one = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = genre.group_norm_act(one[0].expand(4, -1, -1, -1), 2, one[1].expand(8), one[2], act="silu")
        dx, dw, db = torch.autograd.grad(y, one, dy)
        all_ = [t.clone().requires_grad_(True) for t in (x.repeat(4, 1, 1, 1), w.repeat(8), b)]
        z = genre.group_norm_act(all_[0], 2, all_[1], all_[2], act="silu")
        ex, ew, eb = torch.autograd.grad(z, all_, dy)
        assert torch.equal(y, z) and torch.equal(db, eb)
        for got, each in ((dx, ex), (dw, ew.unsqueeze(1))):
            off = (got.double() - each.double().sum(0, keepdim=True).view(got.shape)).abs()
            assert bool((off <= 8 * U * each.double().abs().sum(0, keepdim=True).view(got.shape)).all())


def test_two_passes_captured_and_replayed(genre, dev):
    """maps that take scratch memory: two graphs with an eager call between their replays, each result the eager one's bits"""
    graphs = []
    for fmt, shape in ((torch.channels_last_3d, (2, 40, 20, 21, 22)), (torch.contiguous_format, (2, 24, 30, 31, 9))):
        x, dy = (torch.randn(shape, device=dev).contiguous(memory_format=fmt) for _ in range(2))
        leaves = [t.clone().requires_grad_(True) for t in (x, torch.randn(shape[1], device=dev), torch.randn(shape[1], device=dev))]
        step = lambda leaves=leaves, dy=dy: [(y := genre.group_norm_act(leaves[0], 8, *leaves[1:], act="relu")).detach(), *torch.autograd.grad(y, leaves, dy)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, leaves, dy, step, got))
    for turn in range(3):
        wants = []
        for graph, leaves, dy, step, got in graphs:
            with torch.no_grad():
                leaves[0].normal_()
                dy.normal_()
            wants.append([t.clone() for t in step()])
        for graph, *_ in graphs:
            graph.replay()
            graphs[0][3]()
        torch.cuda.synchronize()
        for (*_, got), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_threads_at_once(genre, dev):
    """each on a stream of its own, as data-parallel programs call: the bits of one after the other"""
    import threading
    x = torch.randn(2, 40, 20, 21, 22, device=dev)
    lists = [[torch.randn(s, device=dev) for s in ((5000,), (33, 7), (1,))] for _ in range(2)]
    want = [(genre.group_norm_act(x, 8, act="silu"), genre.grad_norm(ts)) for ts in lists]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                y, norm = genre.group_norm_act(x, 8, act="silu"), genre.grad_norm(lists[i])
            torch.cuda.current_stream().synchronize()
        got[i] = (y, norm)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_views_of_negatives(genre, dev):
    """torch's lazy negation (of a conjugate's imaginary part) is a flag on the tensor, not in its memory"""
    x, dy, w = (torch.randn(s, device=dev) for s in ((2, 8, 4, 4), (2, 8, 4, 4), (8,)))
    neg = lambda t: torch._neg_view(-t)

    def run(x, dy, w):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w)]
        y = genre.group_norm_act(leaves[0], 2, leaves[1], act="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = run(x, dy, w)
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    assert torch.equal(genre.group_norm_act(neg(x), 2, neg(w), act="silu"), want[0])
    assert all(torch.equal(a, b) for a, b in zip(run(x, neg(dy), w), want))
    leaf = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(genre.group_norm_act(torch._neg_view(leaf), 2, w, act="silu"), leaf, dy)[0], -run(-x, dy, w)[1])
    assert genre.grad_norm([neg(x), dy]).item() == genre.grad_norm([x, dy]).item()
    with pytest.raises(RuntimeError):
        genre.clip_grads_([neg(x)], 1e-3)
    m, v, p, q = torch.zeros_like(x), torch.zeros_like(x), torch.nn.Parameter(x.clone()), torch.nn.Parameter(x.clone())
    with pytest.raises(RuntimeError):
        genre.clip_adam_step_([p.detach()], [neg(dy)], [m], [v], 1)
    for t, g in ((p, dy), (q, neg(dy))):
        t.grad = g
        genre.ClipAdam([t], max_grad_norm=1.0).step()
    assert torch.equal(p, q)


def test_forward_mode_is_refused(genre, dev):
    """rather than a result without its tangent"""
    from torch.autograd import forward_ad
    x, w = torch.randn(2, 8, 4, device=dev), torch.randn(8, device=dev)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x), 2), (x, 2, forward_ad.make_dual(w, w)), (x, 2, w, forward_ad.make_dual(w, w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                genre.group_norm_act(*args)


@pytest.mark.parametrize("config", ("shapehd", "wgangp", "genre"))
def test_the_training_command(genre, dev, config, monkeypatch, capsys, tmp_path):
    """two steps of train.py with both options, on narrow networks (and without MIOpen's search, which takes minutes for new shapes)"""
    from functools import partial
    from genre_shapehd_amd import networks, train
    from genre_shapehd_amd.models import genre as M_genre, shapehd as M_shapehd
    made = []

    def watched(*args):
        made.append(optim(*args))
        return made[-1]

    optim = train.adam

    class Quiet:                                                          # (what is set on it does not reach torch)
        def __getattr__(self, name, real=torch.backends.cudnn):
            return getattr(real, name)

    monkeypatch.setattr(torch.backends, "cudnn", Quiet())
    monkeypatch.setattr(train, "adam", watched)
    monkeypatch.setattr(M_shapehd, "adam", watched)
    monkeypatch.setattr(M_shapehd, "ShapeHDNet", partial(M_shapehd.ShapeHDNet, nf=32, d_nf=2))
    monkeypatch.setattr(M_shapehd, "VoxelGenerator", partial(networks.VoxelGenerator, nf=2))
    monkeypatch.setattr(M_shapehd, "VoxelDiscriminator", partial(networks.VoxelDiscriminator, nf=2))
    monkeypatch.setattr(M_genre, "Unet_3D", partial(networks.Unet_3D, nf=2))
    path = str(tmp_path / "c.pt")
    args = ["--config", config, "--norm", "group", "--clip_grad", "0.5", "--batch", "2", "--steps", "2", "--save", path]
    train.main(args)
    train.main(args + ["--resume", path])
    lines = [line.split() for line in capsys.readouterr().out.splitlines() if line.startswith("step")]
    assert [line[1] for line in lines] == ["0", "1", "2", "3"]
    nets = 2 if config == "wgangp" else 1
    assert len(made) == 2 * nets and all(type(o) is genre.ClipAdam and float(o.grad_norm) > 0 for o in made)
    for first, again in zip(made[:nets], made[nets:]):
        assert {float(s["step"]) for s in first.state.values()} == {2.0} and {float(s["step"]) for s in again.state.values()} == {4.0}
