"""More tokens, or more labels, than are worked on at a time, with a weight for every token (bounds of
test_loss_ranges_gpu.py)."""
import pytest
import torch

from test_loss_ranges_gpu import check
from test_losses_gpu import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape,O", [((2, 6, 600001), 70), ((3, 5, 100, 1001), 250), ((4000, 24), 30000)], ids=lambda v: str(v).replace(" ", ""))
def test_weighted_tokens(cuda_device, shape, O, dtype):
    x, w, b, y = make(shape, O, dtype, 60, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(61)
    weights = torch.rand(y.shape, device=cuda_device, generator=g) * 1e-2
    check(x, w, b, y, weights, 2.0 ** -25 if dtype == torch.float16 else 0.0)


def test_peak_memory(cuda_device):
    """A step over 128^3 voxels, 12 channels and 256 labels stays far below the 2 GB that the logits would take."""
    from msd_pytorch_b200 import linear_cross_entropy

    dev = cuda_device
    x = torch.randn(1, 12, 128, 128, 128, device=dev, requires_grad=True)
    w, b = torch.randn(256, 12, device=dev, requires_grad=True), torch.randn(256, device=dev, requires_grad=True)
    y = torch.randint(0, 256, (1, 128, 128, 128), device=dev)
    torch.cuda.reset_peak_memory_stats(dev)
    before = torch.cuda.memory_allocated(dev)
    linear_cross_entropy(x, w, b, y).backward()
    assert torch.cuda.max_memory_allocated(dev) - before <= (101 + 15 + 600) << 20


def test_more_than_65536_labels_in_one_sum(cuda_device):
    """Labels that the gradient of the features adds up in several sums of the tensor core: half a bfloat16 step in
    every G and in the result, and 10 % for the sums (as in test_losses_gpu.test_large_weights)."""
    from msd_pytorch_b200 import linear_cross_entropy

    T, C, O = 1500, 2048, 89000
    x, w, b, y = make((T, C), O, torch.bfloat16, 62, cuda_device)
    leaf = x.detach().requires_grad_(True)
    (gx,) = torch.autograd.grad(linear_cross_entropy(leaf, w, b, y, reduction="sum"), leaf)
    keep = y != -100
    rows, label = torch.where(keep[:, None], x.double(), 0.0), torch.where(keep, y, 0)
    step = 10000
    lse = torch.full((T,), float("-inf"), dtype=torch.float64, device=x.device)
    for o in range(0, O, step):
        lse = torch.logaddexp(lse, torch.logsumexp(rows @ w[o:o + step].double().t() + b[o:o + step].double(), 1))
    dx, size = torch.zeros_like(rows), torch.zeros_like(rows)
    for o in range(0, O, step):
        wo = w[o:o + step].double()
        G = torch.exp(rows @ wo.t() + b[o:o + step].double() - lse[:, None])
        here = keep & (label >= o) & (label < o + step)
        G[here.nonzero()[:, 0], label[here] - o] -= 1
        G = G * keep[:, None]
        dx += G @ wo
        size += G.abs() @ wo.abs()
    assert bool(((gx.double() - dx).abs() <= 2.0 ** -7 * 1.1 * size).all())
