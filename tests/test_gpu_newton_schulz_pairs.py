"""Tiles of 256 x 256 on pairs of blocks at ragged sizes: a symmetric product of several blocks whose last one is partial, or
whose second half lies past the last row, wide and tall; elman_newton_schulz_tile says which kind a call takes."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests.test_gpu_newton_schulz import TOL, make, reference, rel
from tests.test_gpu_newton_schulz_precision import after_rounding

pytestmark = pytest.mark.gpu

PAIRS = [(6, 1300, 1310), (12, 700, 700), (12, 690, 1100), (12, 1100, 690), (4, 2570, 1290), (4, 1290, 2570), (30, 520, 1030), (30, 1030, 520),
         (3, 1500, 1601), (18, 1280, 1280), (1, 2048, 4096)]
SINGLE = [(18, 512, 512), (1, 1300, 1310), (12, 270, 1536), (2, 200, 9000)]


@pytest.mark.parametrize("kind", ["noise", "lowrank"])
@pytest.mark.parametrize("count,m,n", PAIRS)
def test_pairs_against_definition(count, m, n, kind):
    assert _lib.load().elman_newton_schulz_tile(_lib.ELMAN_BF16, count, m, n) == 256
    G = make(count, m, n, torch.bfloat16, kind=kind, seed=n)
    X, want = H.newton_schulz(G), reference(G)
    for k in range(count):
        assert rel(X[k], want[k]) < TOL[torch.bfloat16] and rel(X[k], want[k].bfloat16().double()) < after_rounding(max(m, n)), k
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("count,m,n", SINGLE)
def test_single_blocks_against_definition(count, m, n):
    assert _lib.load().elman_newton_schulz_tile(_lib.ELMAN_BF16, count, m, n) == 128
    G = make(count, m, n, torch.bfloat16, seed=n)
    X, want = H.newton_schulz(G), reference(G)
    for k in range(count):
        assert rel(X[k], want[k].bfloat16().double()) < after_rounding(max(m, n)), k
