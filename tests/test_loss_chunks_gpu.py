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
