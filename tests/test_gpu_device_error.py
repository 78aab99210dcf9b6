"""vox_cuda_device_error() as a status call that a serving loop can make every step: its cost, and that it gathers the flags of
every kernel family and clears them."""

from __future__ import annotations

import statistics
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def _median_s(fn, n=200):
    for _ in range(20):
        fn()
    t = []
    for _ in range(n):
        t0 = time.perf_counter()
        fn()
        t.append(time.perf_counter() - t0)
    return statistics.median(t)


def test_status_call_costs_one_launch_and_one_copy(vox):
    """However many translation units hold a flag, the call is one launch and one blocking copy: allowed are three times what
    torch takes for a one-element kernel and reading its result."""
    x = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = _median_s(lambda: x.add_(1).item())
    call = _median_s(vox.device_error)
    assert call <= 3 * one, f"device_error {call * 1e6:.1f} us, one launch and one copy {one * 1e6:.1f} us"
