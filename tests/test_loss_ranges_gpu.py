"""Values of very different sizes in one call: float32 products keep float32's accuracy for each of them.

Bounds as in test_losses_gpu.py, without any term that goes by the largest value of a tensor: sums of K
products are off by (2 K + 8) 2^-24 times the sum of the products' magnitudes, token by token, channel by
channel and label by label.  Only float32's own smallest numbers are a limit: an operand's last piece has
bfloat16's exponents, so what lies below the smallest normal number 2^-126 of it may count as zero, and an
operand is off by 2^-126 at most beside its rounding."""
import pytest
import torch

from test_losses_gpu import make

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -126
SHAPES = [((300, 70), 130), ((2, 30, 16, 16), 40), ((1, 20, 10, 10), 300), ((3, 33), 50), ((2, 20, 9, 11), 5), ((1, 140, 8, 12), 16)]


def rows_of(x):
    return x.double() if x.dim() == 2 else x.double().flatten(2).transpose(1, 2).reshape(-1, x.shape[1])


def formulas(x, w, b, y, weights):
    """(value, bound) of the losses and the gradients of sum(weights * losses)."""
    half = torch.finfo(x.dtype).eps / 2
    X, W, B, t, g = rows_of(x), w.double(), b.double(), y.reshape(-1), weights.double().reshape(-1)
    T, C, O = X.shape[0], X.shape[1], W.shape[0]
    keep = t != -100
    X = torch.where(keep[:, None], X, 0.0)
    z = X @ W.t() + B
    dz = (2 * C + 8) * U * (X.abs() @ W.abs().t() + B.abs()) + TINY * (X.abs().sum(1, keepdim=True) + W.abs().sum(1))
    dz = dz.max(1, keepdim=True).values
    lse = torch.logsumexp(z, 1, keepdim=True)
    rel = 2 * dz + (O + 16) * 2 * U
    label = torch.where(keep, t, 0)
    losses = torch.where(keep, (lse - z.gather(1, label[:, None]))[:, 0], 0.0)
    loss_bound = torch.where(keep, rel[:, 0] + 4 * U * losses, 0.0)
    g = torch.where(keep, g, 0.0)
    p = torch.exp(z - lse)
    hot = torch.nn.functional.one_hot(label, O).double()
    G = (p - hot) * g[:, None]
    dp = torch.where(rel < 1, p * rel * 2, 1.0)  # nothing is known of p where rel is large, but 0 <= p <= 1
    dG = (dp + hot * 2 * U) * g[:, None].abs() + (8 * U + (0 if x.dtype == torch.float32 else half)) * G.abs()
    out = [(losses, loss_bound)]
    for a, da, m, k in ((G, dG, W, O), (G.t(), dG.t(), X, T)):
        v = a @ m
        out.append((v, (da @ m.abs() + (2 * k + 8) * U * (a.abs() @ m.abs()) + TINY * (m.abs().sum(0) + a.abs().sum(1, keepdim=True))) * (1 + half) + half * v.abs()))
    v = G.sum(0)
    out.append((v, (dG.sum(0) + (2 * T + 8) * U * G.abs().sum(0)) * (1 + half) + half * v.abs()))
    return out


def check(x, w, b, y, weights, floor=0.0):
    from msd_pytorch_b200 import _lib, linear_cross_entropy

    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    each = linear_cross_entropy(*leaves, y, reduction="none")
    gx, gw, gb = torch.autograd.grad(each, leaves, weights)
    want = formulas(x, w, b, y, weights)
    for name, got, (value, bound) in zip(("loss", "grad_x", "grad_weight", "grad_bias"), (each.reshape(-1), rows_of(gx), gw, gb), want):
        ok = (got.detach().double() - value).abs() <= bound + floor
        assert bool(ok.all()), "%s: %d of %d outside" % (name, int((~ok).sum()), ok.numel())
    assert _lib.device_status(x.device) == 0


@pytest.mark.parametrize("shape,O", SHAPES, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("size", [1e4, 1e9])
def test_one_large_token(cuda_device, shape, O, size):
    """A token far larger than the others takes nothing from them.  Its own weights are small, so that its
    logits stay in range; the other tokens do not have its channels."""
    x, w, b, y = make(shape, O, torch.float32, 50, cuda_device, ignored=0.1)
    C = shape[1]
    x[:, :C // 2] = 0
    first = x[0, :, ...].reshape(C, -1)[:, 0] if x.dim() > 2 else x[0]
    first[:C // 2] = torch.randn(C // 2, device=cuda_device) * size
    w[:, :C // 2] /= size
    assert float(x.abs().max()) > size / 2
    check(x, w, b, y, torch.ones(y.shape, device=cuda_device))


@pytest.mark.parametrize("shape,O", SHAPES, ids=lambda v: str(v).replace(" ", ""))
def test_channels_of_all_sizes(cuda_device, shape, O):
    """Channels from 1e-9 to 1e9 with weights that make up for them."""
    x, w, b, y = make(shape, O, torch.float32, 51, cuda_device, ignored=0.1)
    size = 10.0 ** torch.linspace(-9, 9, shape[1], device=cuda_device)
    check(x * size.view(1, -1, *[1] * (x.dim() - 2)), w / size, b, y, torch.ones(y.shape, device=cuda_device))


@pytest.mark.parametrize("shape,O", SHAPES, ids=lambda v: str(v).replace(" ", ""))
def test_token_weights_of_all_sizes(cuda_device, shape, O):
    """Upstream gradients from 1e-9 to 1e9, each token's features' gradient to its own accuracy."""
    x, w, b, y = make(shape, O, torch.float32, 52, cuda_device, ignored=0.1)
    weights = 10.0 ** torch.linspace(-9, 9, y.numel(), device=cuda_device).view(y.shape)
    check(x, w, b, y, weights)
    check(x, w, b, y, torch.flip(weights, [0]))


@pytest.mark.parametrize("size", [3.4028e38, 1e-30])
def test_ends_of_the_range(cuda_device, size):
    """Features up to the largest float32 (which no bfloat16 is as large as), and close to the smallest."""
    x, w, b, y = make((150, 40), 70, torch.float32, 53, cuda_device, ignored=0.1)
    x = x.clamp(-1, 1) * size
    check(x, w / size, b, y, torch.ones(y.shape, device=cuda_device)) if size < 1 else check(x, w * 1e-38, b, y, torch.full(y.shape, 2.0 ** -60, device=cuda_device))


@pytest.mark.parametrize("dtype,lo,hi", [(torch.bfloat16, -9, 9), (torch.float16, -6, 2)], ids=str)
@pytest.mark.parametrize("shape,O", SHAPES, ids=lambda v: str(v).replace(" ", ""))
def test_token_weights_in_16_bits(cuda_device, shape, O, dtype, lo, hi):
    """The same with 16-bit features (float16's own smallest step beside the bound)."""
    x, w, b, y = make(shape, O, dtype, 54, cuda_device, ignored=0.1)
    weights = 10.0 ** torch.linspace(lo, hi, y.numel(), device=cuda_device).view(y.shape)
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    check(x, w, b, y, weights, floor)
    check(x, w, b, y, torch.flip(weights, [0]), floor)


@pytest.mark.parametrize("T,C,O", [(1500, 300, 700), (40, 24, 150001), (5000, 24, 9)])
def test_token_weights_in_float16_by_size(cuda_device, T, C, O):
    """Several splits of the contraction, several pieces of the labels, few labels over rows."""
    x, w, b, y = make((T, C), O, torch.float16, 55, cuda_device, ignored=0.1)
    weights = 10.0 ** torch.linspace(-6, 0, T, device=cuda_device)
    check(x, w, b, y, weights, 2.0 ** -25)


@pytest.mark.parametrize("shape,O", SHAPES, ids=lambda v: str(v).replace(" ", ""))
def test_one_heavy_token_in_float16(cuda_device, shape, O):
    """A token of weight 6e4 takes nothing from the features' gradients of tokens of weight 1e-4."""
    x, w, b, y = make(shape, O, torch.float16, 56, cuda_device, ignored=0.0)
    first = x[0, :, ...].reshape(shape[1], -1)[:, 0] if x.dim() > 2 else x[0]
    first.mul_(0.1)
    weights = torch.full(y.shape, 1e-4, device=cuda_device)
    weights.view(-1)[0] = 6e4
    check(x, w, b, y, weights, 2.0 ** -25)
