import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (ROOT, os.path.join(ROOT, "tests", "golden")):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a CUDA device (run on a B200)")
    config.addinivalue_line("markers", "slow: long-running test")


def pytest_collection_modifyitems(items):
    """Comparisons with the reference's own build, which exists only where its checkout does, come last: a run
    that stops at the first failure reaches everything else before them."""
    items.sort(key=lambda item: item.fspath.basename == "test_parity_configs_gpu.py")


@pytest.fixture(scope="session")
def cuda_device():
    import torch

    if not torch.cuda.is_available():
        pytest.fail("test is marked gpu but no CUDA device is visible")
    return torch.device("cuda:0")
