"""Gradients that would be written over what the backward pass still reads are refused."""
import pytest
import torch

from elman_b200 import hasty_pytorch_lib as H

pytestmark = pytest.mark.gpu


def test_out_in_the_storage_of_dh_last_or_reset():
    x = torch.randn(70, 2, 8, device="cuda")
    y, h, saved = H.gated_linear_forward(True, x, x, x)
    room = torch.zeros(70 * 2 * 8, device="cuda")
    out = lambda: (room.view(70, 2, 8), torch.empty_like(x), torch.empty_like(x))  # noqa: E731
    with pytest.raises(RuntimeError, match="share storage"):
        H.gated_linear_backward(x, x, x, saved, x, room[:16].view(2, 8), out=out())
    with pytest.raises(RuntimeError, match="share storage"):
        H.gated_linear_backward(x, x, x, saved, x, None, room.view(torch.bool)[:140].view(70, 2), out=out())
    df, dc, dz, dh0 = H.gated_linear_backward(x, x, x, saved, x, out=out())
    assert df.data_ptr() == room.data_ptr() and torch.equal(df, H.gated_linear_backward(x, x, x, saved, x)[0])
