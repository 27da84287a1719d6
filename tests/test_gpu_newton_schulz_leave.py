"""One of the warps that finish tiles gives up its wait for the next one while the others see it, or the end of the list (option
"test_leave_warp"): the launch returns, the status word says so, and the same call is right again afterwards."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests._gpu_cases import option
from tests.test_gpu_operator_failure import KID_NEWTON_SCHULZ, _expect_timeout

pytestmark = pytest.mark.gpu


# a single block with three products (the fourth wait is the list's end), several blocks, pairs, float32
@pytest.mark.parametrize("count,m,n,steps,dtype,tiles", [
    (1, 64, 64, 1, torch.bfloat16, (0, 1, 2, 3)), (1, 64, 60, 1, torch.float32, (0, 2, 3)), (2, 200, 300, 2, torch.bfloat16, (0, 2)),
    (18, 1280, 1280, 1, torch.bfloat16, (0, 5))])
def test_every_finishing_warp_may_leave_alone(count, m, n, steps, dtype, tiles):
    G = torch.randn(count, m, n, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    _lib.device_status(clear=True)
    want = H.newton_schulz(G, steps)
    for tile in tiles:
        for warp in (4, 7, 11):
            with option("spin_limit", 5000), option("test_leave_warp", 32 * tile + warp):
                H.newton_schulz(G, steps)
                _expect_timeout(KID_NEWTON_SCHULZ)
    assert torch.equal(H.newton_schulz(G, steps), want)
    assert _lib.device_status()[0] == 0
