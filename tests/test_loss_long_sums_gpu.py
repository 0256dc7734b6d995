"""Logits over very many channels of 16 bits: sums may not drift with their length.

All products are positive, where an adder that truncates drifts most.  1024 products at a time go through
64 additions that may each be off by 2^-23 of the sum so far, and C / 1024 + 4 more round (2^-24): a
logit is off by (128 + C / 1024 + 4) 2^-24 of itself.  (One truncating sum over 262144 channels: 16384 additions.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,C,O", [(40, 262144, 50), (200, 65536, 300), (6, 1000003, 17)])
def test_long_contraction(cuda_device, T, C, O, dtype):
    from msd_pytorch_b200 import _lib, linear_cross_entropy

    g = torch.Generator(device=cuda_device).manual_seed(C)
    x = (torch.rand(T, C, device=cuda_device, generator=g) * 4 + 1).to(dtype)
    w = (torch.linspace(1, 8, O, device=cuda_device)[:, None] * (torch.rand(O, C, device=cuda_device, generator=g) + 0.5) * (4.0 / C)).to(dtype)
    y = torch.randint(0, O, (T,), device=cuda_device, generator=g)
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]
    # a float16 weight may be subnormal: its products are exact all the same
    bound = 2 * (128 + C / 1024 + 4) * U * z.max(1).values + (O + 16) * 2 * U + 4 * U * want
    for grad in (False, True):
        leaves = [x.detach().requires_grad_(grad), w.detach().requires_grad_(grad)]
        each = linear_cross_entropy(*leaves, None, y, reduction="none").detach().double()
        assert bool(((each - want).abs() <= bound).all())
    assert _lib.device_status(cuda_device) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("T,C,O", [(61, 1000, 5003), (300, 8192, 1000), (150, 65536, 500)])
def test_small_loss_alone(cuda_device, T, C, O, dtype):
    """Logits have standard deviation 2, a stretch of 256 products 2 / sqrt(n) with n = C / 256.  Its 16 additions
    truncate by half a step, 2^-24 of the partial sum, in the mean: at most 16 x 2^-24 x 2 / sqrt(n) per stretch, and as
    the stretches' signs are random 2^-19 for all n of them, whatever n.  Losses are 9 in the mean: 2^-22 of them."""
    from msd_pytorch_b200 import linear_cross_entropy

    g = torch.Generator(device=cuda_device).manual_seed(C + 1)
    x = torch.randn(T, C, device=cuda_device, generator=g).to(dtype)
    w = (torch.randn(O, C, device=cuda_device, generator=g) * (2 / C ** 0.5)).to(dtype)
    y = torch.randint(0, O, (T,), device=cuda_device, generator=g)
    want = torch.nn.functional.cross_entropy(x.double() @ w.double().t(), y, reduction="none")
    with torch.no_grad():
        each = linear_cross_entropy(x, w, None, y, reduction="none").double()
    assert float((each - want).norm()) <= 2.0 ** -22 * float(want.norm())
