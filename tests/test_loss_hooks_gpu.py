"""The loss's gradients with saved tensors that travel through the host and come back in another layout
(tolerances of test_losses_gpu.py)."""
import pytest
import torch

from test_losses_gpu import check, expected, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pin", [False, True], ids=["pageable", "pinned"])
@pytest.mark.parametrize("dtype,labels,reduction", [(torch.float32, 6, "sum"), (torch.float32, 6, "none"), (torch.float32, 40, "sum"), (torch.bfloat16, 6, "sum"),
                                                    (torch.float16, 40, "sum")], ids=str)
def test_save_on_cpu(cuda_device, dtype, labels, reduction, pin):
    from msd_pytorch_b200 import _lib, linear_cross_entropy

    x, w, b, y = make((2, 12, 10, 16), labels, dtype, 40, cuda_device)
    wide = torch.full((2, 20, 10, 16), float("nan"), dtype=dtype, device=cuda_device)
    wide[:, 3:15] = x
    want = expected(x, w, b, y, -100, reduction)
    for v in (wide[:, 3:15], x.contiguous(memory_format=torch.channels_last)):
        leaves = [t.detach().requires_grad_(True) for t in (v, w, b)]
        with torch.autograd.graph.save_on_cpu(pin_memory=pin):
            loss = linear_cross_entropy(*leaves, y, reduction=reduction)
        check("loss", loss, want["loss"])
        for _ in range(2):  # the second pass of a kept graph computes everything from the saved tensors
            grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss), retain_graph=True)
            for name, g in zip(("grad_x", "grad_weight", "grad_bias"), grads):
                check(name, g, want[name])
    assert _lib.device_status(cuda_device) == 0
