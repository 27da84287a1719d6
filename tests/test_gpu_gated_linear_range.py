"""The gated linear recurrence on states far larger than what follows them: they are forgotten as fast as their gates say."""
import pytest
import torch

from elman_b200 import hasty_pytorch_lib as H
from tests.test_gpu_gated_linear import STATE_TOL, reference

pytestmark = pytest.mark.gpu

WIDTHS = [128, 62, 61, 20]      # the four ways rows are read: TMA, copies on 4 and on 2 bytes (bfloat16), registers


def inputs(T, B, d, gate, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    return dict(f=torch.full((T, B, d), gate, device="cuda"), c=rnd(T, B, d), z=torch.full((T, B, d), 1.0, device="cuda"),
                h0=rnd(B, d), dy=rnd(T, B, d), dh=rnd(B, d))


def worst_slice(got, want, slices):
    got, want = got.double().cpu(), want.double()
    return max(float((got[s] - want[s]).norm() / want[s].norm()) for s in slices)


# The gate forgets 0.88 of the state in a step (f = -2): 1e6 is 1e-9 after 16 steps, below what the states are rounded to.
# What holds norm-wise over a sequence of ordinary values has to hold for every stretch of 8 steps from there on.
@pytest.mark.parametrize("large", [1e4, 1e6])
@pytest.mark.parametrize("T", [100, 300, 2900])
@pytest.mark.parametrize("d", WIDTHS)
def test_a_large_state_is_forgotten(d, T, large):
    s = inputs(T, 2, d, -2.0)
    s["h0"] *= large
    s["dh"] *= large
    f, c, z, h0, dy, dh = (s[k] for k in ("f", "c", "z", "h0", "dy", "dh"))
    want = reference(f, c, z, h0, None, dy, dh)
    y, h, saved = H.gated_linear_forward(True, f, c, z, h0)
    df, dc, dz, dh0 = H.gated_linear_backward(f, c, z, saved, dy, dh)
    after = [slice(t, t + 8) for t in range(16, T, 8)]
    before = [slice(max(t - 8, 0), t) for t in range(T - 16, 0, -8)]
    both = [slice(t, t + 8) for t in range(16, T - 24, 8)]
    assert worst_slice(y, want[0], after) < STATE_TOL and worst_slice(dz, want[4], after) < STATE_TOL
    assert worst_slice(dc, want[3], before) < STATE_TOL and worst_slice(df, want[2], both) < STATE_TOL
    assert worst_slice(h[None], want[1][None], [slice(0, 1)]) < STATE_TOL
    assert worst_slice(dh0[None], want[5][None], [slice(0, 1)]) < STATE_TOL


@pytest.mark.parametrize("gate", [-2.0, -8.0, -30.0])
@pytest.mark.parametrize("d", WIDTHS)
def test_a_spike_is_forgotten(d, gate):
    T = 700
    s = inputs(T, 2, d, gate, seed=1)
    f, c, z, h0, dy, dh = (s[k] for k in ("f", "c", "z", "h0", "dy", "dh"))
    spikes = (15, 128, 399)      # at the edges that warps and tiles hand states over
    for t in spikes:
        c[t] *= 1e6
        dy[t] *= 1e6
    want = reference(f, c, z, h0, None, dy, dh)
    y, h, saved = H.gated_linear_forward(True, f, c, z, h0)
    df, dc, dz, dh0 = H.gated_linear_backward(f, c, z, saved, dy, dh)
    clear = [slice(t, t + 8) for t in range(0, T, 8) if all(t >= x + 16 or t + 8 <= x for x in spikes)]
    clear_back = [slice(t, t + 8) for t in range(0, T, 8) if all(t + 8 <= x - 16 or t > x for x in spikes)]
    assert worst_slice(y, want[0], clear) < STATE_TOL and worst_slice(dz, want[4], clear) < STATE_TOL
    assert worst_slice(dc, want[3], clear_back) < STATE_TOL


@pytest.mark.parametrize("d", WIDTHS)
def test_one_long_call_is_many_short_ones_after_a_large_state(d):
    T = 160
    s = inputs(T, 1, d, -2.0, seed=2)
    h0 = 1e6 * s["h0"]
    y, h, _ = H.gated_linear_forward(False, s["f"], s["c"], s["z"], h0)
    parts = []
    for t in range(0, T, 8):
        at = slice(t, t + 8)
        part, h0, _ = H.gated_linear_forward(False, s["f"][at], s["c"][at], s["z"][at], h0)
        parts.append(part)
    assert worst_slice(y, torch.cat(parts).cpu(), [slice(t, t + 8) for t in range(16, T, 8)]) < 2 * STATE_TOL
    assert worst_slice(h[None], h0[None].cpu(), [slice(0, 1)]) < 2 * STATE_TOL
