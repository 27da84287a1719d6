"""Newton-Schulz products of matrices whose norm is far below eps, and which the division by it leaves small."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests.test_gpu_newton_schulz import TOL, reference, rel
from tests.test_gpu_newton_schulz_norms import of_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norm", [1e-6, 1e-9, 1e-11, 1e-13, 1e-16, 1e-24])
@pytest.mark.parametrize("m,n", [(256, 256), (100, 300), (300, 40)])
def test_gradients_far_below_eps(m, n, norm, dtype):
    """The start is G / eps then, and the result about a^5 of that: as many bits as for any other matrix."""
    G = of_norm(norm, 2, m, n, dtype)
    X, want = H.newton_schulz(G), reference(G)
    for k in range(2):
        assert rel(X[k], want[k]) < TOL[dtype]
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [1, 3, 12, 30])
def test_small_starts_grow_to_one(steps, dtype):
    """Steps enough to bring a start of 1e-9 up to one: every step's values stay where the products hold them."""
    G = of_norm(1e-16, 2, 90, 140, dtype, seed=1)
    abc = (1.875, -1.25, 0.375)
    assert rel(H.newton_schulz(G, steps, abc), reference(G, steps, abc)) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_and_ordinary_matrices_in_one_call(dtype):
    G = torch.cat([of_norm(x, 1, 140, 150, dtype, seed=k) for k, x in enumerate((1.0, 1e-12, 3e-8, 1e-20, 5.0))])
    X, want = H.newton_schulz(G), reference(G)
    for k in range(5):
        assert rel(X[k], want[k]) < TOL[dtype], k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("abc,steps", [((0.5, 0.0, 0.0), 20), ((0.6, -0.3, 0.1), 40), ((-0.4, 0.2, 0.1), 9)])
@pytest.mark.parametrize("norm", [1.0, 1e-12])
def test_coefficients_that_shrink(norm, abc, steps, dtype):
    """Every step halves the values, or nearly: none is lost on the way down."""
    G = of_norm(norm, 2, 90, 140, dtype, seed=2)
    assert rel(H.newton_schulz(G, steps, abc), reference(G, steps, abc)) < TOL[dtype]
