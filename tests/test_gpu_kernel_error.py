"""vc_kernel_error on the GPU: what the units report, and what a call costs."""
from __future__ import annotations

import statistics
import time

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_reported_until_cleared(gpu):
    """A kernel's error stays until a call clears it."""
    c = gpu.kv8_cache(*(torch.zeros(4096, dtype=torch.uint8, device="cuda") for _ in range(4)), 2, 1, 16, 64)
    x = torch.zeros(1, 64, device="cuda").half()
    one = torch.tensor([0, 9], dtype=torch.int32, device="cuda")
    assert gpu.kernel_error(True) == 0
    assert gpu.kv8_append(c, x, x, 1, one[1:], 1, one, 1, 1, gpu.Dtype.F16) == 0  # page 9 of 2
    torch.cuda.synchronize()
    assert [gpu.kernel_error(False), gpu.kernel_error(False), gpu.kernel_error(True), gpu.kernel_error(True)] == [4, 4, 4, 0]


def test_costs_no_more_than_five_small_copies(gpu, dev):
    """As many synchronous copies of a word as there were units before the serving kernels'."""
    word, host = dev.alloc(256), np.zeros(1, np.uint32)

    def median(f):
        times = []
        for _ in range(300):
            t = time.perf_counter()
            f()
            times.append(time.perf_counter() - t)
        return statistics.median(times)

    torch.cuda.synchronize()
    ask = median(lambda: gpu.kernel_error(True))
    copy = median(lambda: [gpu.vcMemcpy(host, word.ptr, 4, gpu.VCMemcpyKind.DeviceToHost) for _ in range(5)])
    assert ask < copy, (ask, copy)
