"""What the Newton-Schulz products keep of their operands: results of bfloat16 matrices are those of 32-bit products, rounded
once, and so are parameters that a Muon step moves."""
import math

import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from elman_b200.train_step import FlatGradients, FlatMuon
from tests.test_gpu_newton_schulz import make, reference, rel

pytestmark = pytest.mark.gpu

BF16_STEP = 2.0 ** -7          # between neighbours, relative to the value, at most


def before_rounding(q):
    """Norm-wise error of the result before it is rounded: operands of 22 bits and what small singular values grow by, as for
    float32 matrices (2e-5), and sums that are cut off, not rounded: 3 q / 16 additions to a sum, half of 2^-24 lost a
    time on average, half of that over a sum that grows, with a factor of up to two in each of five steps."""
    return 2e-5 + 10 * (3 * q / 16) * 2.0 ** -26


def after_rounding(q):
    """An element comes out at the other neighbour where the rounding border lies within its error: |error| / step of
    them, each a step off, so that the squared distance is the sum of |error| * step <= |error| |step| (norms)."""
    return math.sqrt(before_rounding(q) * BF16_STEP)


SIZES = [(1, 64, 64), (3, 100, 70), (2, 24, 800), (1, 256, 256), (2, 270, 1536), (4, 1000, 257), (1, 1280, 1280), (6, 1300, 1310), (2, 2570, 1290),
         (2, 1290, 2570)]


@pytest.mark.parametrize("kind", ["noise", "lowrank"])
@pytest.mark.parametrize("count,m,n", SIZES)
def test_bf16_results_are_the_exact_ones_rounded(count, m, n, kind):
    G = make(count, m, n, torch.bfloat16, kind=kind, seed=m)
    X, want = H.newton_schulz(G), reference(G)
    for k in range(count):
        assert rel(X[k], want[k].bfloat16().double()) < after_rounding(max(m, n)), k
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("m,n", [(256, 256), (300, 130), (640, 1300)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_rounds_bf16_parameters_once(m, n, nesterov):
    """Large steps: the update is most of the new value, and nothing of it but the parameter is rounded to 16 bits."""
    g = torch.Generator(device="cuda").manual_seed(m)
    p = torch.nn.Parameter((0.01 * torch.randn(m, n, generator=g, device="cuda")).bfloat16())
    grads = FlatGradients([[p]])
    opt = FlatMuon(grads, [p], lr=0.5, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    momentum = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for it in range(3):
        p.grad.copy_(torch.randn(m, n, generator=g, device="cuda"))
        d = p.grad.double()
        before = p.detach().double()
        momentum += (1 - 0.9) * (d - momentum)
        opt.step()
        X = reference(d + 0.9 * (momentum - d) if nesterov else momentum)
        want = before * (1 - 0.5 * 0.1) - 0.5 * max(1.0, m / n) ** 0.5 * X
        assert rel(p.detach(), want.bfloat16().double()) < after_rounding(max(m, n)), it
