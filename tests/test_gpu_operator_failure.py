"""The give-up paths of the gated linear recurrence and of the Newton-Schulz products: option "test_stall_step" withholds
one tile's share (the recurrence: that tile publishes nothing; the products: block 0 arms a stage and loads nothing), the
waits for it run out, the launch returns, the status word names the kernel, and the same call is right again afterwards."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H
from tests._gpu_cases import option

pytestmark = pytest.mark.gpu

KID_GATED_LINEAR, KID_NEWTON_SCHULZ = 9, 10


def _expect_timeout(kernel_id):
    torch.cuda.synchronize()
    code, detail = _lib.device_status()
    assert code == 3 and (detail >> 24) & 0xFF == kernel_id, (code, detail)
    x = torch.zeros(1, 1, 2, device="cuda")
    with pytest.raises(_lib.ElmanB200Error, match="bounded"):
        H.gated_linear_forward(False, x, x, x)
    _lib.device_status(clear=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 62, 61, 20])
@pytest.mark.parametrize("tile", [0, 9, 15])      # a pair, or a group's state
def test_recurrence_gives_up_when_a_tile_withholds_its_share_and_recovers(tile, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    f, c, z, dy = (torch.randn(4200, 1, d, generator=g, device="cuda").to(dtype) for _ in range(4))
    _lib.device_status(clear=True)
    y, h, saved = H.gated_linear_forward(True, f, c, z)
    want = H.gated_linear_backward(f, c, z, saved, dy)
    with option("spin_limit", 3000), option("test_stall_step", tile):
        H.gated_linear_forward(True, f, c, z)
        _expect_timeout(KID_GATED_LINEAR)
        H.gated_linear_backward(f, c, z, saved, dy)
        _expect_timeout(KID_GATED_LINEAR)
    again = H.gated_linear_forward(True, f, c, z)
    assert all(torch.equal(a, b) for a, b in zip(again, (y, h, saved)))
    assert all(torch.equal(a, b) for a, b in zip(H.gated_linear_backward(f, c, z, saved, dy), want))
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("count,m,n,dtype", [(1, 200, 300, torch.bfloat16), (4, 1280, 1280, torch.bfloat16), (2, 300, 200, torch.float32)])
def test_products_give_up_when_a_stage_never_lands_and_recover(count, m, n, dtype):
    G = torch.randn(count, m, n, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    _lib.device_status(clear=True)
    want = H.newton_schulz(G)
    with option("spin_limit", 5000), option("test_stall_step", 3):
        H.newton_schulz(G)
        _expect_timeout(KID_NEWTON_SCHULZ)
    assert torch.equal(H.newton_schulz(G), want)
    assert _lib.device_status()[0] == 0
