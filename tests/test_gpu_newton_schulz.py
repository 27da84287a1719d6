"""Newton-Schulz orthogonalisation (elman_newton_schulz) against its definition in 64 bits."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H

pytestmark = pytest.mark.gpu

# bf16: the output is rounded once (half a step: 2^-8 relative).  Inside, X, A and B are rounded to fp16 (half a
# step: 2^-11) once a step.  What the last two steps round (6 times 2^-11) enters with factors around one; what earlier steps
# round is in the second part of X that a X takes, 2^-22 off, except where it enters through A and B, whose products with the
# small singular directions are small themselves.  6 * 2^-11 + 2^-8 < 2^-7 + 2^-9.
# fp32: 22 bits an operand, 15 such roundings and the fp32 sums: 15 * 2^-22 = 3.6e-6 where nothing grows; singular values at
# the noise floor grow by up to 3.44^5 / 30 = 16 relative to the strong ones they are rounded beside, in the first step only.
TOL = {torch.float32: 2e-5, torch.bfloat16: 2 ** -7 + 2 ** -9}
COEFFICIENTS = H.NEWTON_SCHULZ_COEFFICIENTS


def reference(G, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    X = G.double()
    X = X / (X.pow(2).sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        if G.shape[-2] <= G.shape[-1]:
            A = X @ X.mT
            X = a * X + b * (A @ X) + c * (A @ (A @ X))
        else:
            A = X.mT @ X
            X = a * X + b * (X @ A) + c * ((X @ A) @ A)
    return X


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


def make(count, m, n, dtype, kind="noise", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    G = torch.randn(count, m, n, generator=g, device="cuda")
    if kind == "lowrank":
        G = 0.01 * G + 0.1 * torch.randn(count, m, 16, generator=g, device="cuda") @ torch.randn(count, 16, n, generator=g, device="cuda")
    return (1e-3 * G).to(dtype)


SIZES = [(1, 1, 1), (1, 1, 5), (2, 5, 1), (3, 2, 3), (1, 8, 8), (2, 63, 65), (1, 64, 64), (2, 127, 129), (1, 128, 128), (1, 129, 127), (3, 130, 70),
         (2, 257, 1000), (1, 300, 41), (2, 512, 1280), (1, 384, 384), (5, 256, 512), (1, 33, 2000), (1, 2000, 33), (1, 700, 700)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count,m,n", SIZES)
def test_against_definition(count, m, n, dtype):
    G = make(count, m, n, dtype, seed=m + n)
    keep = G.clone()
    X = H.newton_schulz(G)
    want = reference(G)
    assert X.dtype == dtype and X.shape == G.shape and torch.equal(G, keep)
    for k in range(count):
        assert rel(X[k], want[k]) < TOL[dtype], (k, rel(X[k], want[k]))
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(512, 512), (1280, 640), (270, 1536)])
def test_strong_directions_above_noise(m, n, dtype):
    G = make(2, m, n, dtype, kind="lowrank", seed=3)
    assert rel(H.newton_schulz(G), reference(G)) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_singular_values_end_near_one(dtype):
    X = H.newton_schulz(make(1, 200, 320, dtype, seed=1))[0]
    s = torch.linalg.svdvals(X.double())
    assert 0.65 < float(s[:150].min()) and float(s.max()) < 1.25


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7, 10])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_and_coefficients(steps, dtype):
    coefficients = (1.875, -1.25, 0.375)      # the quintic that converges to one
    G = make(2, 90, 150, dtype, seed=steps)
    assert rel(H.newton_schulz(G, steps, coefficients), reference(G, steps, coefficients)) < TOL[dtype]
    coefficients = (1.5, -0.5, 0.0)           # the cubic
    assert rel(H.newton_schulz(G, steps, coefficients), reference(G, steps, coefficients)) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scale_of_the_gradient_does_not_matter(dtype):
    G = make(1, 100, 140, dtype, seed=2)
    for scale in (2.0 ** -90, 2.0 ** 90):
        X = H.newton_schulz(G * scale, eps=0.0)
        assert rel(X, reference(G, eps=0.0)) < TOL[dtype]
    one = torch.zeros(1, 50, 80, device="cuda", dtype=dtype)     # a single entry: a singular value of one
    one[0, 7, 9] = -3e-4
    X = H.newton_schulz(one)
    assert rel(X, reference(one)) < TOL[dtype] and int((X != 0).sum()) == 1


def test_zero_and_non_finite_matrices_stay_among_themselves():
    G = make(5, 150, 140, torch.bfloat16, seed=4)
    want = H.newton_schulz(G)
    G[1] = 0
    G[2, 3, 5] = float("nan")
    G[3, 140, 139] = float("inf")
    X = H.newton_schulz(G)
    assert torch.equal(X[0], want[0]) and torch.equal(X[4], want[4])
    assert (X[1] == 0).all() and torch.isnan(X[2]).all() and torch.isnan(X[3]).all()


def test_leading_dimensions_and_plain_matrices():
    G = make(6, 40, 30, torch.float32)
    X = H.newton_schulz(G)
    assert torch.equal(H.newton_schulz(G.view(2, 3, 40, 30)).view(6, 40, 30), X)
    assert torch.equal(H.newton_schulz(G[2]), X[2])
    assert H.newton_schulz(G[:0]).shape == (0, 40, 30) and H.newton_schulz(G[:, :0]).shape == (6, 0, 30)


def test_two_runs_and_two_batches_give_the_same_bits():
    G = make(7, 300, 500, torch.bfloat16, seed=6)
    X = H.newton_schulz(G)
    assert torch.equal(H.newton_schulz(G), X)
    assert torch.equal(torch.stack([H.newton_schulz(g) for g in G]), X)


def test_calls_on_two_streams_at_once():
    """Launches that share the device: none waits for another's blocks."""
    sets = [make(6, 640, 700, torch.bfloat16, seed=1), make(2, 1100, 1024, torch.bfloat16, seed=2), make(3, 300, 400, torch.float32, seed=3)]
    want = [H.newton_schulz(G) for G in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for G, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(H.newton_schulz(G))
    torch.cuda.synchronize()
    assert all(torch.equal(X, want[k % 3]) for k, X in enumerate(got))
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("count,m,n", [(18, 512, 512), (3, 1280, 1280), (4, 2560, 1024), (1, 2048, 4096)])
def test_tiles_of_block_pairs(count, m, n):
    """Sizes at which pairs of blocks make tiles of 256 x 256."""
    G = make(count, m, n, torch.bfloat16, kind="lowrank", seed=m)
    assert rel(H.newton_schulz(G), reference(G)) < TOL[torch.bfloat16]


def test_captured_on_another_stream():
    a, b = make(2, 200, 300, torch.bfloat16, seed=7), make(1, 330, 130, torch.bfloat16, seed=8)
    side, graphs, outs, pool = torch.cuda.Stream(), [], [], None
    with torch.cuda.stream(side):
        H.newton_schulz(a), H.newton_schulz(b)
    torch.cuda.synchronize()
    for G in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool, stream=side):
            outs.append(H.newton_schulz(G))
        pool = g.pool()
        graphs.append(g)
    for seed in (1, 2):
        for G, g, X in zip((a, b), graphs, outs):
            G.copy_(make(*G.shape, torch.bfloat16, seed=seed))
            g.replay()
            torch.cuda.synchronize()
            got = X.clone()
            assert torch.equal(got, H.newton_schulz(G))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(64, 9000), (9000, 100), (200, 9000)])
def test_long_and_narrow_matrices(m, n, dtype):
    """The tile's shape follows both extents: these are where the longer one, q, decides.  The fp32 sums are cut off, not
    rounded: each of the q / 48 additions to one of the three sums loses 2^-24 of it on average, half of that over a sum
    that grows, and a relative error of A enters X with a factor of up to two in each of five steps."""
    G = make(2, m, n, dtype, seed=7)
    X, want = H.newton_schulz(G), reference(G)
    for k in range(2):
        assert rel(X[k], want[k]) < TOL[dtype] + 10 * (9000 / 48) * 2 ** -25, (k, rel(X[k], want[k]))
