"""Which tiles a call of given sizes takes is a host function (no GPU)."""
import pytest

from elman_b200 import _lib


@pytest.mark.parametrize("count,m,n,tile", [(18, 1280, 1280, 256), (6, 2560, 1280, 256), (6, 1280, 2560, 256), (1, 4096, 4096, 256),
                                            (1, 256, 256, 128), (18, 512, 512, 128), (12, 270, 1536, 128), (2, 200, 9000, 128)])
def test_many_or_large_matrices_take_pairs(count, m, n, tile):
    lib = _lib.load()
    assert lib.elman_newton_schulz_tile(_lib.ELMAN_BF16, count, m, n) == tile
    assert lib.elman_newton_schulz_tile(_lib.ELMAN_F32, count, m, n) == 128


def test_nothing_to_do():
    lib = _lib.load()
    for dtype, count, m, n in [(7, 1, 8, 8), (_lib.ELMAN_BF16, 0, 8, 8), (_lib.ELMAN_BF16, 1, 0, 8), (_lib.ELMAN_BF16, 1, 8, -1)]:
        assert lib.elman_newton_schulz_tile(dtype, count, m, n) == 0
