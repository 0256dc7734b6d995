"""Calls of several host threads at once: what is set up per kernel holds for all of them."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_few_tokens_of_different_widths(cuda_device):
    """Four tokens of 8192 channels take 128 KB of shared memory, of 256 channels 4 KB: one thread's calls must
    not lower the limit that the other's launch."""
    from msd_pytorch_b200 import linear_cross_entropy

    cases, failures = [], []
    for k, C in enumerate((8192, 256, 4096, 64)):
        g = torch.Generator(device=cuda_device).manual_seed(k)
        x = torch.randn(4, C, device=cuda_device, generator=g).bfloat16()
        w = torch.randn(200, C, device=cuda_device, generator=g).mul_(C ** -0.5).bfloat16()
        y = torch.randint(0, 200, (4,), device=cuda_device, generator=g)
        cases.append((x, w, y, linear_cross_entropy(x, w, None, y, reduction="none")))
    torch.cuda.synchronize(cuda_device)

    def work(x, w, y, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
                for _ in range(400):
                    got = linear_cross_entropy(x, w, None, y, reduction="none")
                torch.cuda.current_stream(cuda_device).synchronize()
                assert torch.equal(got, want)
        except BaseException as e:  # reported by the test's own thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
