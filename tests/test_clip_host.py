"""CPU: what the C ABI of gradient norm and clipping refuses before any CUDA call."""
import ctypes

import pytest

from mappedconvolutions_b200 import _lib


def lists(numel, dtype=0):
    n = len(numel)
    return (ctypes.c_void_p * n)(*[256] * n), (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*[dtype] * n)


@pytest.mark.parametrize("numel", [[(1 << 63) - 1], [1 << 62], [8192 << 30], [8192 << 29] * 2, [1 << 55] * 300, [(1 << 63) - 8192, 5]])
def test_more_elements_than_can_be_counted(numel):
    p, n, t = lists(numel)
    ws = 1 << 30
    assert _lib.lib().mc_grad_norm(len(numel), p, n, t, 2.0, 8, None, 4096, ws, None) == -6
    assert _lib.lib().mc_grad_clip(len(numel), p, t, p, t, n, 2.0, 1.0, 8, None, 4096, ws, None) == -6


def test_bad_tensors_are_reported_before_large_ones():
    L = _lib.lib()
    p, n, t = lists([(1 << 63) - 1, -1])
    assert L.mc_grad_norm(2, p, n, t, 2.0, 8, None, 4096, 1 << 30, None) == -1
    p, n, t = lists([5])
    assert L.mc_grad_norm(1, p, n, t, 2.0, 8, None, None, 1 << 30, None) == -3  # (and a small list gets as far as its workspace)
