"""Newton-Schulz products without eps: zero matrices, and norms at the ends of the type's range."""
import pytest
import torch

from elman_b200 import hasty_pytorch_lib as H
from elman_b200.train_step import FlatGradients, FlatMuon
from tests.test_gpu_newton_schulz import TOL, make, reference, rel

pytestmark = pytest.mark.gpu


def of_norm(norm, count, m, n, dtype, seed=0):
    G = make(count, m, n, torch.float32, seed=seed).double()
    return (G * (norm / G.pow(2).sum((-2, -1), keepdim=True).sqrt())).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_eps(dtype):
    """eps = 0: a zero matrix stays zero, and the smallest and the largest norms are as good as any."""
    zero = torch.zeros(1, 50, 60, dtype=dtype, device="cuda")
    norms = (1e-36, 1e-38, 1.0, 1e38) + ((1e-41,) if dtype == torch.float32 else ())     # (bfloat16 has nothing below 9e-41)
    G = torch.cat([zero] + [of_norm(x, 1, 50, 60, dtype, seed=3) for x in norms])
    assert torch.isfinite(G).all() and (G[1:] != 0).any(-1).any(-1).all()
    X, want = H.newton_schulz(G, eps=0.0), reference(G[1:], eps=0.0)
    assert (X[0] == 0).all()
    for k in range(len(norms)):
        assert rel(X[1 + k], want[k]) < TOL[dtype], k


def test_muon_without_eps_leaves_parameters_without_a_gradient_alone():
    p = torch.nn.Parameter(torch.randn(40, 60, device="cuda"))
    keep = p.detach().clone()
    opt = FlatMuon(FlatGradients([[p]]), [p], eps=0.0)
    opt.step()
    assert torch.equal(p.detach(), keep)
