"""What hooks on saved tensors hand back to the loss's backward pass: the geometry that the library gets
is that of the tensors at hand, not that of the forward call's."""
import pytest
import torch

from msd_pytorch_b200 import losses


@pytest.fixture
def calls(monkeypatch):
    """The library calls replaced: forward leaves a mark, backward records what it was given."""
    record = []

    def forward(x, geometry, weight, bias, target, ignore_index, reduction, keep):
        record.append(("forward", x, geometry))
        return torch.zeros(()), torch.full((8,), len(record), dtype=torch.uint8)

    def backward(x, geometry, weight, bias, target, ignore_index, reduction, saved, grad_loss, grad_x, grad_x_geometry, grad_weight, grad_bias):
        record.append(("backward", x, geometry, weight, saved, grad_x, grad_x_geometry))
        for g in (grad_x, grad_weight, grad_bias):
            g.zero_()

    monkeypatch.setattr(losses, "_check", lambda *a: None)
    monkeypatch.setattr(losses, "xent_forward_", forward)
    monkeypatch.setattr(losses, "xent_backward_", backward)
    return record


def last_element(x, geometry):
    n, c, v, sn, sc, sv = geometry
    return x.storage_offset() + (n - 1) * sn + (c - 1) * sc + (v - 1) * sv


HOOKS = {
    "dense": lambda t: t.clone(memory_format=torch.contiguous_format),
    "channels_last": lambda t: t.contiguous(memory_format=torch.channels_last) if t.dim() == 4 else t.clone(),
    "same": lambda t: t,
}


@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("layout", ["slice", "channels_last", "cropped"])
def test_layouts_from_hooks(calls, hook, layout):
    wide = torch.randn(2, 20, 10, 16)
    x = {"slice": wide[:, 3:15], "channels_last": wide[:, 3:15].contiguous(memory_format=torch.channels_last), "cropped": wide[:, 3:15, :, :12]}[layout]
    leaves = [x.detach().requires_grad_(True), torch.randn(30, 12, requires_grad=True), torch.randn(30, requires_grad=True)]
    y = torch.zeros(x.shape[0], *x.shape[2:], dtype=torch.int64)
    with torch.autograd.graph.saved_tensors_hooks(HOOKS[hook], lambda t: t):
        loss = losses.linear_cross_entropy(*leaves, y)
    loss.backward()
    first, (_, got, geometry, _, saved, grad_x, grad_geometry) = calls[0], calls[-1]
    assert geometry == losses._features(got) and torch.equal(got, x)
    assert last_element(got, geometry) < got.untyped_storage().nbytes() // 4
    assert grad_geometry == losses._features(grad_x) and last_element(grad_x, grad_geometry) < grad_x.numel()
    # what forward left serves the backward call only in the layout that it was made for
    again = [c for c in calls if c[0] == "forward"]
    assert len(again) == (1 if geometry == first[2] else 2)
    assert int(saved[0]) == len(again)


def test_weight_of_another_alignment(calls):
    """A 16-bit weight is read where it lies or packed, by its alignment, and what forward leaves follows."""
    x, y = torch.randn(40, 16).bfloat16(), torch.zeros(40, dtype=torch.int64)
    flat = torch.randn(30 * 16 + 1).bfloat16()
    w = flat[1:].view(30, 16)
    if w.data_ptr() % 16 == 0:
        w = flat[:-1].view(30, 16)
    leaves = [x.requires_grad_(True), w.detach().requires_grad_(True), torch.zeros(30).bfloat16().requires_grad_(True)]
    for hook, forwards in ((lambda t: t, 1), (lambda t: t.clone(), 3)):
        with torch.autograd.graph.saved_tensors_hooks(hook, lambda t: t):
            loss = losses.linear_cross_entropy(*leaves, y)
        loss.backward()
        assert len([c for c in calls if c[0] == "forward"]) == forwards
