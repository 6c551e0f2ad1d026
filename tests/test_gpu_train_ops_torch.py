"""The training-step ops under what torch lays over autograd: saved tensors on the host, recomputation, function transforms."""
import pytest
import torch

from test_gpu_group_norm import definition, make, near, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("last", (False, True), ids=("first", "last"))
@pytest.mark.parametrize("space", ((5, 9), (90, 91)), ids=("one workgroup", "two passes"))
def test_maps_that_are_kept_on_the_host(genre, dev, space, last):
    """they come back channels first, whatever they were: the gradients are those of the definition all the same"""
    x, dy, w, b = make(dev, 2, 8, space, torch.float32, last)
    with torch.autograd.graph.save_on_cpu():
        got = run(genre, x, dy, w, b, 2, "silu")
    want = definition(x, dy, w, b, 2, "silu", 1e-5, 0.2)
    for k in got:
        near(got[k], want[k], k)


@pytest.mark.parametrize("reentrant", (False, True))
def test_recomputed_in_the_backward(genre, dev, reentrant):
    from torch.utils.checkpoint import checkpoint
    net = genre.GroupNormAct(2, 8, act="silu").to(dev)
    x, dy, _, _ = make(dev, 2, 8, (20, 21), torch.float32, True)
    leaves = [x.requires_grad_(True), *net.parameters()]
    want = torch.autograd.grad(net(x), leaves, dy)
    x.grad = None
    checkpoint(net, x, use_reentrant=reentrant).backward(dy)
    assert all(torch.equal(t.grad, v) for t, v in zip(leaves, want))


def test_function_transforms_are_refused(genre, dev):
    """whose tensors hold no memory of their own"""
    x, w = torch.randn(3, 2, 8, 4, device=dev), torch.ones(8, device=dev)
    for call in (lambda: torch.func.vmap(lambda t: genre.group_norm_act(t, 2, w))(x), lambda: torch.func.grad(lambda t: genre.group_norm_act(t, 2, w).sum())(x[0]),
                 lambda: torch.func.vmap(lambda t: genre.grad_norm([t]))(x), lambda: torch.func.vmap(lambda t: genre.clip_grads_([t], 1.0))(x),
                 lambda: torch.func.jvp(lambda t: genre.group_norm_act(t, 2, w), (x[0],), (x[0],))):
        with pytest.raises(RuntimeError):
            call()


def test_a_refiner_with_group_norm_is_captured_and_replayed(genre, dev):
    """as GenReInference(graph=True) does with the whole model: every replay is what the eager forward gives, to the convolutions' rounding"""
    from genre_shapehd_amd.networks import Unet_3D
    torch.manual_seed(2)
    net = Unet_3D(norm="group").to(dev).eval()
    x = torch.rand(1, 2, 128, 128, 128, device=dev)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                net(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = net(x)
        for _ in range(3):
            x.uniform_()
            want = net(x)
            graph.replay()
            torch.cuda.synchronize()
            assert (y - want).abs().max() <= 1e-4 * max(1.0, want.abs().max())
