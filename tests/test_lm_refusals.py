"""The recurrence refuses what it cannot address before it launches anything (no GPU needed: a launch would report that there is
none, not that the call is too large)."""
import pytest

from dnatok_amd import _lib

P = 4096                                # an address that is never looked at
TOO_LARGE = -3
TOTAL = 100000                          # several tiles, so that words would have to be filled first


def scan(x_stride, gate_stride, dtype=0):
    L = _lib.lib()
    need = L.dnatok_gated_scan_work_bytes(TOTAL, 8)
    assert need > 0
    return L.dnatok_gated_scan(P, x_stride, P, gate_stride, dtype, None, 1, TOTAL, 8, 0, None, P, None, None, P, need, None)


def backward(x_stride, gate_stride, dy_stride, dtype=0):
    L = _lib.lib()
    need = L.dnatok_gated_scan_work_bytes(TOTAL, 8)
    return L.dnatok_gated_scan_backward(P, x_stride, P, gate_stride, dtype, None, 1, TOTAL, 8, 0, None, P, dy_stride, None, P, P, P,
                                        None, P, need, None)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("far", [2 ** 31 // 2 // 25 + 1, 2 ** 40, 2 ** 58, 2 ** 61, 2 ** 62 + 2 ** 40])
def test_tokens_too_far_apart(far, dtype):
    calls = [scan(far, 8, dtype), scan(8, far, dtype), backward(far, 8, 8, dtype), backward(8, far, 8, dtype),
             backward(8, 8, far, dtype)]
    assert calls == [TOO_LARGE] * 5
