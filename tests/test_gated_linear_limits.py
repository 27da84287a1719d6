"""The longest sequence that the gated linear recurrence takes (refused before anything is launched: no GPU)."""
import ctypes

import pytest

from elman_b200 import _lib

P = 1 << 20


@pytest.mark.parametrize("T,message", [(2 ** 31 - 1, b"too long"), (2 ** 31 - 1024, b"too long"), (2 ** 31 - 1025, b"workspace is NULL")])
def test_steps_counted_past_the_end_stay_within_32_bits(T, message):
    lib = _lib.load()
    strides = (ctypes.c_long * 14)(*[1, 1] * 7)
    assert lib.elman_gated_linear_workspace(_lib.ELMAN_BF16, T, 1, 1) > 0
    assert lib.elman_gated_linear_forward(_lib.ELMAN_BF16, 0, T, 1, 1, P, P, P, None, None, strides, 2 * P, P, None, None, 0, None) == 1
    assert message in lib.elman_b200_last_error()
    far = [P + (k << 34) for k in range(3)]
    assert lib.elman_gated_linear_backward(_lib.ELMAN_BF16, T, 1, 1, P, P, P, P, P, None, None, strides, *far, P, None, 0, None) == 1
    assert message in lib.elman_b200_last_error()
