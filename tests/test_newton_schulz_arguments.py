"""What the orthogonalisation and the Muon step refuse (nothing is launched: no GPU)."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H

P = 1 << 20


def _call(lib, dtype=_lib.ELMAN_BF16, count=1, m=4, n=4, steps=5, abc=H.NEWTON_SCHULZ_COEFFICIENTS, eps=1e-7, G=P, out=P, ws=P, ws_bytes=1 << 30):
    return lib.elman_newton_schulz(dtype, count, m, n, G, out, steps, *abc, eps, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,rc,message", [
    (dict(dtype=5), 1, b"dtype"), (dict(m=-1), 1, b"negative size"), (dict(count=70000), 1, b"too large"), (dict(steps=0), 1, b"steps"),
    (dict(steps=101), 1, b"steps"), (dict(eps=-1.0), 1, b"eps"), (dict(abc=(10.0, 0.0, 0.0)), 1, b"beyond 3.5"),
    (dict(abc=(2.0, 70.0, -70.0), steps=1), 1, b"beyond"), (dict(abc=(float("nan"), 0.0, 0.0)), 1, b"beyond"),
    (dict(G=None), 1, b"NULL"), (dict(out=None), 1, b"NULL"), (dict(ws=None), 1, b"NULL"), (dict(ws_bytes=100), 4, b"workspace"),
    (dict(ws=P + 8), 1, b"aligned"), (dict(G=P + 1), 1, b"misaligned"), (dict(out=P + 2, dtype=_lib.ELMAN_F32), 1, b"misaligned"),
])
def test_c_entry_refuses(kw, rc, message):
    lib = _lib.load()
    assert _call(lib, **kw) == rc
    assert message in lib.elman_b200_last_error()


def test_growth_over_the_steps_is_what_counts():
    lib = _lib.load()
    assert _call(lib, abc=(1.2, 0.0, 0.0), steps=6, G=None) == 1 and b"NULL" in lib.elman_b200_last_error()       # 1.2^6 < 3.5
    assert _call(lib, abc=(1.2, 0.0, 0.0), steps=7, G=None) == 1 and b"beyond" in lib.elman_b200_last_error()


def test_muon_entry_refuses():
    lib = _lib.load()
    call = lambda offsets=P, params=P, grads=P, mom=P, ws=P: lib.elman_muon_step(  # noqa: E731
        _lib.ELMAN_F32, 1, 4, 4, offsets, params, grads, mom, 0.1, 0.9, 1, 0.0, 1.0, None, 5, *H.NEWTON_SCHULZ_COEFFICIENTS, 1e-7, ws, 1 << 30, None)
    for name in ("offsets", "params", "grads", "mom", "ws"):
        assert call(**{name: None}) == 1 and b"NULL" in lib.elman_b200_last_error()
    for name in ("offsets", "params", "grads", "mom"):
        assert call(**{name: P + (4 if name == "offsets" else 2)}) == 1 and b"misaligned" in lib.elman_b200_last_error()


def test_nothing_to_do_is_no_error_and_needs_no_workspace():
    lib = _lib.load()
    for kw in (dict(count=0), dict(m=0), dict(n=0)):
        assert _call(lib, G=None, out=None, ws=None, ws_bytes=0, **kw) == 0
    assert lib.elman_newton_schulz_workspace(_lib.ELMAN_BF16, 0, 4, 4) == 0
    assert lib.elman_newton_schulz_workspace(_lib.ELMAN_BF16, 3, 100, 50) % 256 == 0


def test_python_refuses():
    with pytest.raises(RuntimeError, match="CUDA"):
        H.newton_schulz(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        H.newton_schulz([[1.0]])
