"""States that are NaN with every bit set, which is what the scan's workspace starts from, are NaN like any other."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests.test_gpu_gated_linear import make

pytestmark = pytest.mark.gpu


def marked(state, every, bits):
    state = state.clone()
    state.view(torch.int32)[:, ::every] = bits
    return state


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 62, 61, 20])
@pytest.mark.parametrize("T", [3, 9, 64, 300, 2900])
def test_all_ones(T, d, dtype):
    """The same bits out as with the ordinary NaN, and the channels without one are not touched."""
    s = make(T, 2, d, dtype, seed=T)
    runs = []
    for bits in (0x7FC00000, -1):
        h0, dh = marked(s["h0"], 3, bits), marked(s["dh"], 5, bits)
        y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], h0)
        assert torch.isnan(h[:, ::3]).all() and torch.isfinite(h[:, 1::3]).all() and torch.isnan(y[:, :, ::3]).all()
        clean = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])[2]
        df, dc, dz, dh0 = H.gated_linear_backward(s["f"], s["c"], s["z"], clean, s["dy"], dh)
        assert torch.isnan(dh0[:, ::5]).all() and torch.isfinite(dh0[:, 1::5]).all()
        assert torch.isnan(dc[..., ::5]).all() and torch.isfinite(dc[..., 1::5]).all()
        runs.append([torch.nan_to_num(t, nan=7.0) for t in (y, h, df, dc, dz, dh0)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert _lib.device_status()[0] == 0
