"""ClipAdam's state through the framework's checkpoints, on the kernels (test_clip_adam_state.py has it without them)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def network(dev, dtype, like=None):
    g = torch.Generator().manual_seed(3)
    net = torch.nn.Module()
    net.ps = torch.nn.ParameterList([torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).to(dev)) for s in ((20, 7, 3, 3), (20,), (1,), (33, 65))])
    if like is not None:
        net.load_state_dict(like.state_dict())
    return net


def give(net, seed, scale):
    g = torch.Generator().manual_seed(seed)
    for p in net.ps:
        p.grad = (scale * torch.randn(p.shape, generator=g)).to(p.dtype).to(p.device)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16), ids=("fp32", "bf16", "fp16"))
def test_a_resumed_run_is_the_one_that_was_saved(genre, dev, dtype, tmp_path):
    """bits, with gradients whose squares an fp16 second moment would lose"""
    from genre_shapehd_amd.models import checkpoint
    net = network(dev, dtype)
    opt = genre.ClipAdam(net.parameters(), lr=1e-2, betas=(0.5, 0.9), max_grad_norm=2e-3)
    give(net, 0, 1e-4)
    opt.step()
    path = str(tmp_path / "c.pt")
    checkpoint.save_state_dict(path, [net], [opt])
    other = network(dev, dtype)
    again = genre.ClipAdam(other.parameters(), lr=1e-2, betas=(0.5, 0.9), max_grad_norm=2e-3)
    checkpoint.load_state_dict(path, [other], [again])
    for step in (2, 3):
        for n, o in ((net, opt), (other, again)):
            give(n, step, 1e-4)
            o.step()
    for p, q in zip(net.ps, other.ps):
        assert torch.equal(p, q) and float(again.state[q]["step"]) == 3
        assert all(torch.equal(opt.state[p][k], again.state[q][k]) for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("options", ({"foreach": False}, {"foreach": True}, {"fused": True}), ids=("plain", "foreach", "fused"))
def test_a_run_that_goes_on_without_the_bound(genre, dev, options, tmp_path):
    """torch.optim.Adam from a checkpoint of ClipAdam's: the bits of one whose state was put together parameter by parameter"""
    from genre_shapehd_amd.models import checkpoint
    net = network(dev, torch.float32)
    opt = genre.ClipAdam(net.parameters(), lr=1e-2, betas=(0.5, 0.9), max_grad_norm=1.0)
    give(net, 0, 1.0)
    opt.step()
    path = str(tmp_path / "c.pt")
    checkpoint.save_state_dict(path, [net], [opt])
    nets = [network(dev, torch.float32, net) for _ in range(2)]
    adams = [torch.optim.Adam(n.parameters(), lr=1e-2, betas=(0.5, 0.9), **options) for n in nets]
    checkpoint.load_state_dict(path, nets[:1], adams[:1])
    where = dev if "fused" in options else "cpu"
    for p, q in zip(net.ps, nets[1].ps):
        adams[1].state[q] = {"step": torch.tensor(1.0, device=where), "exp_avg": opt.state[p]["exp_avg"].clone(), "exp_avg_sq": opt.state[p]["exp_avg_sq"].clone()}
    for step in (2, 3):
        for n, adam in zip(nets, adams):
            give(n, step, 1.0)
            adam.step()
        assert [float(adams[0].state[q]["step"]) for q in nets[0].ps] == [float(step)] * 4
        assert all(torch.equal(a, b) for a, b in zip(nets[0].ps, nets[1].ps))
