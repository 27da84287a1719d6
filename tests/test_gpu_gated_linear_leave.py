"""One warp of a block gives up its wait for a stage while the others see it land (option "test_leave_warp"): the block ends, the
status word says so, and the same call is right again afterwards."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests._gpu_cases import option
from tests.test_gpu_operator_failure import KID_GATED_LINEAR, _expect_timeout

pytestmark = pytest.mark.gpu


def test_the_option_is_known():
    assert _lib.get_option("test_leave_warp") == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 62, 61])
@pytest.mark.parametrize("T,B,tile", [(40, 1, 0), (40, 1, 1), (4200, 1, 0), (4200, 1, 1), (3000, 16, 0), (3000, 16, 1), (3000, 16, 2)])
def test_every_warp_may_leave_alone(T, B, tile, d, dtype):
    """Scanning warps (the first, one between, the last) and linking ones; a block's first tile, a later one, and the end."""
    g = torch.Generator(device="cuda").manual_seed(1)
    f, c, z, dy = (torch.randn(T, B, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    _lib.device_status(clear=True)
    y, h, saved = H.gated_linear_forward(True, f, c, z)
    want = H.gated_linear_backward(f, c, z, saved, dy)
    for warp in (0, 3, 6, 7, 8):
        with option("spin_limit", 3000), option("test_leave_warp", 32 * tile + warp):
            if warp < 8 or d == 128 or dtype == torch.bfloat16:     # (seven scanning warps and one that links, or two)
                H.gated_linear_forward(True, f, c, z)
                _expect_timeout(KID_GATED_LINEAR)
            H.gated_linear_backward(f, c, z, saved, dy)
            _expect_timeout(KID_GATED_LINEAR)
    again = H.gated_linear_forward(True, f, c, z)
    assert all(torch.equal(a, b) for a, b in zip(again, (y, h, saved)))
    assert all(torch.equal(a, b) for a, b in zip(H.gated_linear_backward(f, c, z, saved, dy), want))
    assert _lib.device_status()[0] == 0
