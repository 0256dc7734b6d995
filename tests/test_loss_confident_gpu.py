"""Confident tokens: the target's logit stands far above the others, so loss and 1 - p are small
beside the logits.  All inputs are small integers, so that every logit is exact in float32 in any order.

Bounds.  With s = 1 + sum over the other labels of exp(z - m), at most 16 + O / 16 additions round a sum in
[1, 2) (U = 2^-24 each), whatever the kernel; the terms behind the 1 are off by 2^-22 (exponential) and
4 U 1.5 |z| (a logit in units of log 2, and the difference of two) relative.  log s, loss and 1 - p are
off by as much, and by one step of their own size.  p of the other labels is off relatively by all of it
together; sums of n equal gradients round n times."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LAYOUTS = [  # shape of the features, labels
    ((2, 12, 8, 20), 4), ((2, 12, 8, 20), 7), ((1, 24, 9, 11), 11), ((1, 24, 9, 11), 16), ((1, 150, 10, 10), 3),  # few labels
    ((2, 24, 9, 12), 40), ((64, 64), 300), ((300, 40), 1000), ((1, 16), 50), ((3, 16), 700),
]


def confident(shape, O, offset, margin, dtype, dev):
    """Token t has channel t % C alone; label o has weight `margin` there if it is that token's target."""
    C = shape[1]
    T = 1
    for s in (shape[0], *shape[2:]):
        T *= s
    channel = torch.arange(T, device=dev) % C
    rows = torch.nn.functional.one_hot(channel, C).to(dtype)
    x = rows if len(shape) == 2 else rows.view(shape[0], -1, C).transpose(1, 2).reshape(shape).contiguous()
    o = torch.arange(O, device=dev)
    target_of = torch.arange(C, device=dev) * 7 % O
    w = torch.where(o[:, None] == target_of, margin, -(o % 3)[:, None]).to(dtype)
    b = torch.full((O,), offset, device=dev, dtype=dtype)
    y = target_of[channel].view(shape[0], *shape[2:])
    z = w.double() + b.double()[:, None]  # of a token with channel c
    return x, w, b, y, z, target_of, torch.bincount(channel, minlength=C).double()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("offset", [0, 96, -96, 1000])
@pytest.mark.parametrize("shape,O", LAYOUTS, ids=lambda v: str(v).replace(" ", ""))
def test_confident_tokens(cuda_device, shape, O, offset, dtype):
    from msd_pytorch_b200 import linear_cross_entropy

    for margin in (9, 12):
        x, w, b, y, z, target_of, n = confident(shape, O, offset, margin, dtype, cuda_device)
        C = shape[1]
        lse = torch.logsumexp(z, 0)
        log_s = torch.log1p(torch.exp(z - z.gather(0, target_of[None])).sum(0) - 1.0)
        exact = log_s  # the target is the largest
        big = float(z.abs().max())
        relative = 2.0 ** -22 + 4 * U * 1.5 * big + 4 * U
        bound = (16 + O / 16) * U + relative * exact + 2 * U * exact
        for grad in (False, True):
            leaves = [t.detach().requires_grad_(grad) for t in (x, w, b)]
            each = linear_cross_entropy(*leaves, y, reduction="none").detach().double().reshape(-1)
            channel = torch.arange(each.numel(), device=x.device) % C
            assert bool(((each - exact[channel]).abs() <= bound[channel]).all()), (margin, grad)
            total = linear_cross_entropy(*leaves, y, reduction="sum")
            assert abs(float(total.detach()) - float((exact * n).sum())) <= float((bound * n).sum()) + 4 * U * float((exact * n).sum())
        grads = torch.autograd.grad(total, leaves)
        half = torch.finfo(dtype).eps / 2
        G = torch.exp(z - lse)
        dG = G * (relative + (16 + O / 16) * U)
        hot = torch.nn.functional.one_hot(target_of, O).t().bool()
        G = torch.where(hot, torch.expm1(-log_s)[None], G)
        dG = torch.where(hot, bound[None], dG)
        if dtype != torch.float32:
            dG = dG + half * (G.abs() + dG)
        if dtype == torch.float16:
            dG = dG + 2.0 ** -39  # G is held as a float16 in units of 2^-14 of the upstream gradient
        want = G * n
        tolerance = dG * n * (1 + half) + (half + 2 * U * (n + 8)) * want.abs() + 2.0 ** -38 * n
        if dtype == torch.float16:
            tolerance = tolerance + 2.0 ** -25
        assert bool(((grads[1].double() - want).abs() <= tolerance).all()), margin
        assert bool(((grads[2].double() - want.sum(1)).abs() <= tolerance.sum(1) + half * want.sum(1).abs()).all()), margin
