"""Sizes that the library asks for, without a GPU: what a call needs beside its tensors is bounded."""
import pytest

from msd_pytorch_b200 import _lib

MB = 1 << 20


def sizes(dtype, batch, channels, voxels, labels):
    f = _lib.MsdFeatures()
    f.data, f.batch, f.channels, f.voxels = 256, batch, channels, voxels
    f.stride_batch, f.stride_channel, f.stride_voxel = channels * voxels, voxels, 1
    L = _lib.lib
    return (L.msd_linear_xent_saved_bytes(dtype, f, 256, labels), L.msd_linear_xent_workspace_bytes(dtype, f, 256, labels, 0),
            L.msd_linear_xent_workspace_bytes(dtype, f, 256, labels, 1))


@pytest.mark.parametrize("dtype,channels,voxels,labels", [
    (_lib.MSD_F32, 12, 128 ** 3, 256), (_lib.MSD_F32, 51, 128 ** 3, 20), (_lib.MSD_F32, 101, 2 * 1024 ** 2, 17), (_lib.MSD_BF16, 5, 30000000, 256),
    (_lib.MSD_F16, 5, 30000000, 256), (_lib.MSD_F32, 2, 100000000, 100), (_lib.MSD_F32, 40, 50000000, 1000), (_lib.MSD_F32, 300, 10000000, 65),
])
def test_work_space_is_bounded(dtype, channels, voxels, labels):
    """256 MB of G, 512 MB of packed features, and a half more for sums and edges; 7 bytes per voxel, and
    up to 256 MB of packed operands, from forward to backward."""
    saved, forward, backward = sizes(dtype, 1, channels, voxels, labels)
    assert backward <= 1152 * MB and forward <= 1152 * MB
    assert saved <= 7 * voxels + 256 * MB + 4096
    logits = 4 * voxels * labels
    if logits > 2048 * MB:
        assert max(forward, backward) < logits / 2


@pytest.mark.parametrize("dtype", [_lib.MSD_F32, _lib.MSD_BF16, _lib.MSD_F16])
def test_few_labels_keep_nothing_per_voxel(dtype):
    """The backward pass of few labels computes its statistics again."""
    for voxels in (64, 128 ** 3):
        assert sizes(dtype, 2, 51, voxels, 11)[0] <= 256
