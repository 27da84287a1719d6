"""What the gated linear recurrence refuses, at the C entry and in Python (nothing is launched: no GPU)."""
import ctypes

import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H


def _strides(*v):
    return (ctypes.c_long * len(v))(*v)


def _forward(lib, dtype=_lib.ELMAN_F32, training=0, T=4, B=2, d=8, f=1 << 20, h_last=1 << 20, saved=None, strides=None,
             y=1 << 20):
    strides = strides if strides is not None else _strides(*[16, 8] * 4)
    return lib.elman_gated_linear_forward(dtype, training, T, B, d, f, f, f, None, None, strides, y, h_last, saved,
                                          None, 0, None)


@pytest.mark.parametrize("kw,message", [
    (dict(dtype=7), b"dtype"), (dict(T=-1), b"negative size"), (dict(f=None), b"NULL"), (dict(y=None), b"NULL"),
    (dict(h_last=None), b"NULL"), (dict(training=1), b"saved"),
    (dict(strides=_strides(16, 8, 16, -8, 16, 8, 16, 8)), b"negative stride"),
    (dict(strides=_strides(16, 8, 16, 8, 16, 8, 0, 8)), b"overlap"),
    (dict(strides=_strides(16, 8, 16, 8, 16, 8, 16, 7)), b"overlap"),
    (dict(strides=_strides(16, 8, 16, 8, 16, 8, 12, 8)), b"overlap"),
])
def test_c_entry_refuses(kw, message):
    lib = _lib.load()
    assert _forward(lib, **kw) == 1
    assert message in lib.elman_b200_last_error()


def test_c_backward_refuses_overlapping_gradients_and_missing_pointers():
    lib = _lib.load()
    p = 1 << 20
    call = lambda s, saved=p: lib.elman_gated_linear_backward(_lib.ELMAN_BF16, 4, 2, 8, p, p, p, saved, p, None, None, s, p, p, p, p,  # noqa: E731
                                                              None, 0, None)
    assert call(_strides(*[16, 8] * 6, 16, 4)) == 1 and b"overlap" in lib.elman_b200_last_error()
    assert call(_strides(*[16, 8] * 7), saved=None) == 1 and b"saved" in lib.elman_b200_last_error()
    assert call(None) == 1


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert _forward(lib, B=0, f=None, y=None, h_last=None) == 0
    assert _forward(lib, d=0, f=None, y=None, h_last=None) == 0


def test_workspace_is_a_host_function():
    lib = _lib.load()
    for T in (0, 1, 100, 70000):
        assert lib.elman_gated_linear_workspace(_lib.ELMAN_BF16, T, 2, 64) < (1 << 30)
    assert lib.elman_gated_linear_workspace(_lib.ELMAN_BF16, -1, 2, 64) == 0


def test_python_refuses():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        H.gated_linear_forward(False, x, x, x)
    with pytest.raises(TypeError):
        H.gated_linear_forward(False, x.tolist(), x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        H.gated_linear_backward(x, x, x, x, x)


@pytest.mark.parametrize("dc,dz,strides,refused", [
    (8, 16, (48, 24), False), (8, 24, (48, 24), True), (8, 12, (48, 24), True), (0, 16, (48, 24), True),
    (48, 16, (48, 24), True), (16, 8, (24, 1680), False), (8, 16, (50, 24), True), (4096, 8192, (50, 24), False)])
def test_c_backward_refuses_gradients_among_one_another(dc, dz, strides, refused):
    """df, dc, dz at these elements of one buffer.  What is apart gets as far as the missing workspace."""
    lib = _lib.load()
    p = 1 << 20
    assert lib.elman_gated_linear_workspace(_lib.ELMAN_F32, 70, 2, 8) > 0
    assert lib.elman_gated_linear_backward(_lib.ELMAN_F32, 70, 2, 8, p, p, p, p, p, None, None,
                                           _strides(*[48, 24] * 4, *strides * 3), p, p + 4 * dc, p + 4 * dz, p, None, 0, None) == 1
    assert (b"df, dc and dz overlap" if refused else b"workspace is NULL") in lib.elman_b200_last_error()


@pytest.mark.parametrize("kw,message", [(dict(f=(1 << 20) + 2), b"misaligned tensor"), (dict(y=(1 << 20) + 1), b"misaligned tensor"),
                                        (dict(h_last=(1 << 20) + 2), b"misaligned state"),
                                        (dict(training=1, saved=(1 << 20) + 1), b"misaligned state")])
def test_c_entry_refuses_pointers_between_elements(kw, message):
    lib = _lib.load()
    assert _forward(lib, **kw) == 1
    assert message in lib.elman_b200_last_error()


def test_c_entry_refuses_a_workspace_off_its_boundary():
    lib = _lib.load()
    p, need = 1 << 20, lib.elman_gated_linear_workspace(_lib.ELMAN_F32, 70, 2, 8)
    s = _strides(*[16, 8] * 4)
    assert lib.elman_gated_linear_forward(_lib.ELMAN_F32, 0, 70, 2, 8, p, p, p, None, None, s, 2 * p, p, None, p + 8, need, None) == 1
    assert b"16-byte" in lib.elman_b200_last_error()
