"""Clipping at the ends of float32's range, and what autograd learns of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64], ids=str)
@pytest.mark.parametrize("max_norm", [1e-3, 1e-6, 1.0])
def test_factors_below_the_smallest_normal_number(cuda_device, dtype, max_norm):
    """Values near 1e38 clipped to a small norm: the factor is a subnormal float32, the results are not.
    Norm and factor: 3 2^-24 (float32 sums of 32 bytes) and 2^-24; the result one rounding more."""
    from msd_pytorch_b200 import clip_norm_

    g = torch.Generator(device=cuda_device).manual_seed(1)
    t = (torch.rand(5000, device=cuda_device, generator=g) * 2e38 + 1e38).to(dtype)
    want = t.double()
    norm = want.norm()
    want = want * (max_norm / (norm + 1e-6))
    tensors = [t[:1237], t[1237:]]
    got = clip_norm_(tensors, max_norm)
    if dtype == torch.float64:
        assert abs(float(got) - float(norm)) <= 1e-14 * float(norm)
    half = torch.finfo(dtype).eps / 2
    relative = half + (2.0 ** -50 if dtype == torch.float64 else 5 * 2.0 ** -24)
    assert bool(((t.double() - want).abs() <= relative * want.abs()).all())
