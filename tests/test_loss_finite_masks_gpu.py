"""Labels masked by a bias of the type's lowest value, the largest number that is no infinity: a token whose
labels are all masked like that has equal logits, and one whose target is masked a finite loss.

Products are sums of small integers, so logits are exact up to their one rounding to float32; the bounds
are those of test_loss_confident_gpu.py with differences of logits d instead of logits: exp(-d) is off by
2^-22 + 4 U d relative."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("masked", ["all", "target", "all_but_one"])
@pytest.mark.parametrize("shape,O", [((2, 6, 9, 12), 4), ((2, 6, 9, 12), 11), ((1, 6, 9, 12), 16), ((2, 6, 9, 12), 40), ((70, 24), 300), ((1, 24), 50), ((4, 24), 700)],
                         ids=lambda v: str(v).replace(" ", ""))
def test_lowest_value(cuda_device, shape, O, masked, dtype):
    from msd_pytorch_b200 import linear_cross_entropy

    dev, C = cuda_device, shape[1]
    g = torch.Generator(device=dev).manual_seed(O)
    x = torch.randint(-1, 2, shape, device=dev, generator=g).to(dtype)
    w = torch.randint(-1, 2, (O, C), device=dev, generator=g).to(dtype)
    b = torch.randint(-3, 4, (O,), device=dev, generator=g).to(dtype)
    lowest = torch.finfo(dtype).min
    y = torch.full((shape[0], *shape[2:]), O // 2, dtype=torch.int64, device=dev)
    if masked == "target":
        b[O // 2] = lowest
    else:
        keep = b[0].clone()
        b.fill_(lowest)
        if masked == "all_but_one":
            b[0] = keep
    rows = x.double() if x.dim() == 2 else x.double().flatten(2).transpose(1, 2).reshape(-1, C)
    z = ((rows @ w.double().t()).float() + b.float()).double()
    top = z.max(1, keepdim=True).values
    p = torch.softmax(z, 1)
    gap = (top[:, 0] - z[:, O // 2])
    loss = gap + torch.log(torch.exp(z - top).sum(1))
    d = torch.where(p > 0, top - z, 0.0)
    relative = (2.0 ** -22 + 4 * U * d.max()) + (O + 16) * 2 * U
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    for alone in (True, False):
        with torch.set_grad_enabled(not alone):
            each = linear_cross_entropy(*leaves, y, reduction="none")
        assert bool(torch.isfinite(each).all())
        assert bool(((each.detach().double().reshape(-1) - loss).abs() <= relative + 4 * U * loss).all())
    total = linear_cross_entropy(*leaves, y, reduction="none").sum() if dtype == torch.float16 else linear_cross_entropy(*leaves, y, reduction="sum")
    gx, gw, gb = torch.autograd.grad(total, leaves)
    half = torch.finfo(dtype).eps / 2
    G = p.clone()
    G[:, O // 2] -= 1
    dG = p * relative + 4 * U * G.abs() + (half * G.abs() if dtype != torch.float32 else 0) + (2.0 ** -38)
    for got, want, bound in ((gw, G.t() @ rows, dG.t() @ rows.abs() + 2 * U * (len(rows) + 8) * (G.abs().t() @ rows.abs())),
                             (gb, G.sum(0), dG.sum(0) + 2 * U * (len(rows) + 8) * G.abs().sum(0))):
        ok = (got.double() - want).abs() <= bound * (1 + half) + half * want.abs() + 2.0 ** -25
        assert bool(ok.all())
    tokens = gx.double() if x.dim() == 2 else gx.double().flatten(2).transpose(1, 2).reshape(-1, C)
    bound = dG @ w.double().abs() + 2 * U * (O + 8) * (G.abs() @ w.double().abs())
    want = G @ w.double()
    assert bool(((tokens - want).abs() <= bound * (1 + half) + half * want.abs() + 2.0 ** -25).all())
