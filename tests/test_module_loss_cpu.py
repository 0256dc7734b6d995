"""Refusals of ``MSDModule.cross_entropy`` that need no GPU: the block's kernels take its parameters by
address."""
import pytest
import torch

from msd_pytorch_b200 import MSDModule


def make():
    net = MSDModule(1, 4, 3, 1, [1, 2], ndim=2)
    return net, torch.randn(1, 1, 8, 8), torch.zeros(1, 8, 8, dtype=torch.int64)


def test_strided_weights():
    net, x, y = make()
    net.to(memory_format=torch.channels_last)
    assert not net.msd_block.weight1.is_contiguous()
    with pytest.raises(RuntimeError, match="weight1 to be contiguous"):
        net.cross_entropy(x, y)


def test_another_device():
    for name in ("bias", "weight0", "weight2"):
        net, x, y = make()
        old = getattr(net.msd_block, name)
        setattr(net.msd_block, name, torch.nn.Parameter(torch.empty_like(old, device="meta")))
        with pytest.raises(RuntimeError, match="on cpu, got one on meta"):
            net.cross_entropy(x, y)


def test_depth():
    net, x, y = make()
    net.msd_block.dilations = [1, 2]
    with pytest.raises(RuntimeError, match="3 dilations, got 2"):
        net.cross_entropy(x, y)


def test_shapes():
    """A 2D network's kernels hold 9 taps, a volume's layers read 27."""
    net, _, _ = make()
    with pytest.raises(RuntimeError, match="weight0 of shape"):
        net.cross_entropy(torch.randn(1, 1, 8, 8, 8), torch.zeros(1, 8, 8, 8, dtype=torch.int64))
    net, x, y = make()
    net.msd_block.bias = torch.nn.Parameter(torch.zeros(2))
    with pytest.raises(RuntimeError, match="3 block biases"):
        net.cross_entropy(x, y)


@pytest.mark.parametrize("ignore", [2 ** 63, -2 ** 63 - 1, 2 ** 64 + 5])
def test_ignore_index_out_of_range(monkeypatch, ignore):
    """An index past 64 bits is refused instead of losing its high bits on the way to the library."""
    from msd_pytorch_b200 import linear_cross_entropy, losses

    monkeypatch.setattr(losses, "_check", lambda *a: None)
    net, x, y = make()
    with pytest.raises(ValueError, match="ignore_index"):
        net.cross_entropy(x, y, ignore_index=ignore)
    with pytest.raises(ValueError, match="ignore_index"):
        linear_cross_entropy(torch.zeros(4, 3), torch.zeros(5, 3), None, torch.zeros(4, dtype=torch.int64), ignore_index=ignore)
