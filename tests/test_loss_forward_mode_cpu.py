"""Forward-mode derivatives are not offered by the loss and the clipping: a tangent is refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from msd_pytorch_b200 import losses


@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
@pytest.mark.parametrize("which", [0, 1, 2], ids=["input", "weight", "bias"])
def test_tangents_are_refused(monkeypatch, which, grad):
    monkeypatch.setattr(losses, "_check", lambda *a: None)
    monkeypatch.setattr(losses, "xent_forward_", lambda *a: (torch.zeros(()), torch.zeros(8, dtype=torch.uint8)))
    monkeypatch.setattr(losses, "xent_step_", lambda *a: (torch.zeros(()), torch.zeros(8, dtype=torch.uint8)))
    operands = [torch.randn(40, 12), torch.randn(30, 12), torch.randn(30)]
    y = torch.zeros(40, dtype=torch.int64)
    with torch.set_grad_enabled(grad):
        with fwAD.dual_level():
            assert losses.linear_cross_entropy(*operands, y).shape == ()  # no tangent: as anywhere
            operands[which] = fwAD.make_dual(operands[which], torch.ones_like(operands[which]))
            with pytest.raises(RuntimeError, match="jvp"):
                losses.linear_cross_entropy(*operands, y)


def test_tangents_of_gradients_are_refused():
    from msd_pytorch_b200 import clip_norm_, total_norm

    t = torch.ones(3)
    with fwAD.dual_level():
        dual = fwAD.make_dual(t, torch.ones(3))
        for call in (lambda: total_norm([t, dual]), lambda: clip_norm_([dual], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):
            total_norm([t])
