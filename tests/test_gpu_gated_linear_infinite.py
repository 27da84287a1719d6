"""The gated linear recurrence on states that are not finite."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests.test_gpu_gated_linear import reference
from tests.test_gpu_gated_linear_range import WIDTHS, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [3, 9, 100, 129, 300, 1290])
@pytest.mark.parametrize("d", WIDTHS)
def test_an_infinite_last_state_is_infinite(d, T, dtype):
    """The steps past the sequence's end, up to a tile's or a warp's, add nothing to it."""
    s = inputs(T, 2, d, 0.0, seed=3)
    f, c, z, dy = (s[k].to(dtype) for k in ("f", "c", "z", "dy"))
    c[-1, 0, ::3] = float("inf")
    y, h, saved = H.gated_linear_forward(True, f, c, z, s["h0"])
    _, want = reference(f, c, z, s["h0"], None)
    assert torch.equal(torch.isinf(h).cpu(), torch.isinf(want)) and not torch.isnan(h).any()
    assert (h[0, ::3] > 0).all() and torch.isfinite(h[1]).all() and torch.isinf(y[-1, 0, ::3]).all()
    c[-1] = 0
    dh = s["dh"].clone()
    dh[1, ::3] = float("-inf")
    y, h, saved = H.gated_linear_forward(True, f, c, z, s["h0"])
    df, dc, dz, dh0 = H.gated_linear_backward(f, c, z, saved, dy, dh)
    assert (dc[-1, 1, ::3] == float("-inf")).all() and torch.isfinite(dc[:, 0]).all() and torch.isfinite(dh0[0]).all()
    assert _lib.device_status()[0] == 0
