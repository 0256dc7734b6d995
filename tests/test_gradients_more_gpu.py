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


def test_autograd_sees_the_change(cuda_device):
    """A graph that saved a tensor refuses to go backward after the tensor was clipped, as after any operation
    in place; outputs count as written, inputs beside them do not."""
    from msd_pytorch_b200 import clip_norm_

    for strided in (False, True):
        base = torch.randn(8, 6, device=cuda_device)
        a, b = (base[:, ::2], torch.randn(5, device=cuda_device)) if strided else (base, torch.randn(5, device=cuda_device))
        leaf = torch.randn(a.shape, device=cuda_device, requires_grad=True)
        loss = (leaf * a).sum()
        versions = a._version, b._version
        clip_norm_([a, b], 0.1)
        assert a._version > versions[0] and b._version > versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        out = [torch.empty_like(a), torch.empty_like(b)]
        versions = a._version, b._version, out[0]._version, out[1]._version
        clip_norm_([a, b], 0.1, out=out)
        assert (a._version, b._version) == versions[:2]
        assert out[0]._version > versions[2] and out[1]._version > versions[3]
    with torch.inference_mode():  # tensors without a version
        t = torch.ones(100, device=cuda_device)
        clip_norm_([t], 1.0)
        assert abs(float(t[0]) - 0.1) <= 1e-7
