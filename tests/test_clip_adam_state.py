"""ClipAdam's state on its way through files and into torch.optim.Adam, on the CPU: the kernels' part of a step is a plain one here."""
import copy
import io

import pytest
import torch


class _Native:
    """the two native calls of ClipAdam.step"""

    @staticmethod
    def grad_norm(tensors, max_norm, kind):
        norm = torch.stack([t.float().norm() for t in tensors]).norm()
        return torch.stack([norm, (max_norm / (norm + 1e-6)).clamp(max=1)])

    @staticmethod
    def laid_otherwise(weights, others):
        return []


def _plain_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr, betas, eps, weight_decay, decoupled, factor):
    for p, g, m, v in zip(params, grads, exp_avgs, exp_avg_sqs):
        assert m.dtype == v.dtype == torch.float32
        g = g.float() * (1 if factor is None else factor)
        m.mul_(betas[0]).add_((1 - betas[0]) * g)
        v.mul_(betas[1]).add_((1 - betas[1]) * g * g)
        p.copy_(p.float() - lr / (1 - betas[0] ** step) * m / (v.sqrt() / (1 - betas[1] ** step) ** 0.5 + eps))


@pytest.fixture
def optim(genre, monkeypatch):
    from genre_shapehd_amd import optim
    monkeypatch.setattr(optim, "_native", _Native)
    monkeypatch.setattr(optim, "clip_adam_step_", _plain_step)
    return optim


def _weights(dtype=torch.float32):
    g = torch.Generator().manual_seed(3)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in ((4, 3), (5,), (1,), (2, 2, 2))]


def _grads(params, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (scale * torch.randn(p.shape, generator=g)).to(p.dtype)


def _through_a_file(sd):
    f = io.BytesIO()
    torch.save(sd, f)
    f.seek(0)
    return torch.load(f)


@pytest.mark.parametrize("foreach", (False, True))
@pytest.mark.parametrize("way", (_through_a_file, copy.deepcopy, lambda sd: sd), ids=("file", "copy", "as it is"))
def test_adam_goes_on_counting_each_parameter_once(optim, way, foreach):
    """torch.optim.Adam from a ClipAdam's state: the bits of one whose state was put together parameter by parameter"""
    ps = _weights()
    opt = optim.ClipAdam(ps, lr=1e-2, betas=(0.5, 0.9), max_grad_norm=1.0)
    _grads(ps, 0)
    opt.step()
    got, want = [torch.nn.Parameter(p.detach().clone()) for p in ps], [torch.nn.Parameter(p.detach().clone()) for p in ps]
    adams = [torch.optim.Adam(qs, lr=1e-2, betas=(0.5, 0.9), foreach=foreach) for qs in (got, want)]
    options = {"lr": 1e-2, "betas": (0.5, 0.9), "foreach": foreach}
    sd = way(opt.state_dict())
    adams[0].load_state_dict(dict(sd, param_groups=[dict(sd["param_groups"][0], **options)]))
    for p, q in zip(ps, want):
        adams[1].state[q] = {"step": torch.tensor(1.0), "exp_avg": opt.state[p]["exp_avg"].clone(), "exp_avg_sq": opt.state[p]["exp_avg_sq"].clone()}
    for step in (2, 3):
        for qs, adam in zip((got, want), adams):
            _grads(qs, step)
            adam.step()
        assert [float(adams[0].state[q]["step"]) for q in got] == [float(step)] * 4
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {float(opt.state[p]["step"]) for p in ps} == {1.0}             # (theirs, not ours)


@pytest.mark.parametrize("foreach", (False, True))
def test_files_with_a_shared_count_load_as_well(genre, foreach, tmp_path):
    """what models.checkpoint reads, whoever wrote it"""
    from genre_shapehd_amd.models import checkpoint
    net = torch.nn.Module()
    net.ps = torch.nn.ParameterList(_weights())
    one, params = torch.tensor(4.0), list(net.parameters())
    adam = torch.optim.Adam(params, lr=1e-2, foreach=foreach)
    for p in params:
        adam.state[p] = {"step": one, "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p)}
    path = str(tmp_path / "c.pt")
    checkpoint.save_state_dict(path, [net], [adam])
    again = torch.optim.Adam(params, lr=1e-2, foreach=foreach)
    checkpoint.load_state_dict(path, [net], [again])
    _grads(params, 1)
    again.step()
    assert [float(again.state[p]["step"]) for p in params] == [5.0] * 4


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=("fp32", "bf16", "fp16"))
def test_a_resumed_run_is_the_one_that_was_saved(optim, dtype):
    """bits, with gradients so small that an fp16 second moment would be zero (1e-4 squared), through a file, a copy and a pickle"""
    import pickle
    ps = _weights(dtype)
    opt = optim.ClipAdam(ps, lr=1e-2, betas=(0.5, 0.9))
    _grads(ps, 0, 1e-4)
    opt.step()
    runs = [(ps, opt)]
    for way in (_through_a_file, copy.deepcopy):
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        again = optim.ClipAdam(qs, lr=1e-2, betas=(0.5, 0.9))
        again.load_state_dict(way(opt.state_dict()))
        runs.append((qs, again))
    whole = pickle.loads(pickle.dumps(opt))
    runs.append((whole.param_groups[0]["params"], whole))
    for step in (2, 3):
        for qs, o in runs:
            _grads(qs, step, 1e-4)
            o.step()
    for qs, o in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        for p, q in zip(ps, qs):
            assert all(torch.equal(opt.state[p][k], o.state[q][k]) and o.state[q][k].dtype == torch.float32 for k in ("step", "exp_avg", "exp_avg_sq"))


def test_loaded_moments_are_the_ones_that_the_hooks_leave(optim):
    """and no memory of the state that was loaded"""
    ps = _weights(torch.float16)
    opt = optim.ClipAdam(ps, lr=1e-2)
    _grads(ps, 0)
    opt.step()
    again = optim.ClipAdam([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1e-2)
    half = lambda o, sd: dict(sd, state={k: dict(st, exp_avg=st["exp_avg"] / 2) for k, st in sd["state"].items()})
    again.register_load_state_dict_pre_hook(half)
    sd = opt.state_dict()
    again.load_state_dict(sd)
    for p, q in zip(ps, again.param_groups[0]["params"]):
        assert torch.equal(again.state[q]["exp_avg"], opt.state[p]["exp_avg"] / 2)
        again.state[q]["exp_avg_sq"].zero_()
        assert bool((opt.state[p]["exp_avg_sq"] > 0).all())
    again.load_state_dict(sd)                                             # (no hook of the first load is left)
    again.load_state_dict(optim.ClipAdam(ps).state_dict())                # no state at all
    assert not again.state


def test_a_state_that_half_precision_adam_wrote(optim):
    """its moments, which are half precision there"""
    ps = _weights(torch.bfloat16)
    adam = torch.optim.Adam(ps, lr=1e-2)
    _grads(ps, 0)
    adam.step()
    opt = optim.ClipAdam([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=1e-2)
    opt.load_state_dict(adam.state_dict())
    qs = opt.param_groups[0]["params"]
    for p, q in zip(ps, qs):
        assert all(opt.state[q][k].dtype == torch.float32 and torch.equal(opt.state[q][k], adam.state[p][k].float()) for k in ("exp_avg", "exp_avg_sq"))
    _grads(qs, 1)
    opt.step()
    assert {float(opt.state[q]["step"]) for q in qs} == {2.0}
