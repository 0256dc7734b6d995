"""A backward pass captured into a graph whose forward pass ran before the capture: every replay gives the
same gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def replayed(run, stream, times=3):
    """The results of `run` captured on `stream`, after some replays."""
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    seen = []
    for _ in range(times):
        graph.replay()
        torch.cuda.synchronize()
        seen.append([t.clone() for t in out])
    return seen


@pytest.mark.parametrize("factor", [1.0, 0.5])
@pytest.mark.parametrize("shape,O", [((2, 20, 30, 40), 5), ((2, 20, 30, 40), 40), ((400, 70), 300)], ids=lambda v: str(v).replace(" ", ""))
def test_backward_alone(cuda_device, shape, O, factor):
    from test_losses_gpu import make

    from msd_pytorch_b200 import linear_cross_entropy

    x, w, b, y = make(shape, O, torch.float32, 70, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    upstream = torch.full((), factor, device=cuda_device)
    want = torch.autograd.grad(linear_cross_entropy(*leaves, y), leaves, upstream)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        loss = linear_cross_entropy(*leaves, y)
    side.synchronize()
    for grads in replayed(lambda: torch.autograd.grad(loss, leaves, upstream), side):
        for g, e in zip(grads, want):
            assert float((g - e).abs().max()) <= 1e-5 * float(e.abs().max())


def test_module_backward_alone(cuda_device):
    from msd_pytorch_b200 import MSDModule

    torch.manual_seed(6)
    net = MSDModule(1, 5, 4, 1, [1, 2], ndim=2).to(cuda_device)
    with torch.no_grad():
        net.final_layer.linear.weight.normal_(0, 0.5)
    params = list(net.parameters())
    x, y = torch.randn(2, 1, 32, 64, device=cuda_device), torch.randint(0, 5, (2, 32, 64), device=cuda_device)
    upstream = torch.full((), 0.5, device=cuda_device)
    want = torch.autograd.grad(net.cross_entropy(x, y), params, upstream)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        torch.autograd.grad(net.cross_entropy(x, y), params, upstream)  # scratch memory of this stream
        loss = net.cross_entropy(x, y)
    side.synchronize()
    for grads in replayed(lambda: torch.autograd.grad(loss, params, upstream), side):
        for g, e in zip(grads, want):
            assert float((g - e).abs().max()) <= 1e-4 * float(e.abs().max())
