"""Calls of the serving operators at the edges of what they take."""
import pytest
import torch

from tests.test_gpu_moe import make, router_of, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_into_a_view_at_an_odd_offset(dtype):
    """The kernel stores four values at once; a contiguous out of any address gets the same bits."""
    import qwantize_b200 as q
    up, down, t = make(4, 64, 32, "nvfp4", 1)
    ex = q.FP4Experts(up, down, tensor_scales=(t, t))
    r, x = router_of(4, 64, torch.bfloat16, 2), tokens(3, 64, dtype, 3)
    want = q.fp4_moe(x, r, ex, 2)
    for off in (1, 2, 3, 4):
        buf = torch.full((off + x.numel() + 5,), 7.0, dtype=dtype, device=DEV)
        out = buf[off: off + x.numel()].view(x.shape)
        assert q.fp4_moe(x, r, ex, 2, out=out) is out
        assert torch.equal(out, want) and bool((buf[:off] == 7).all()) and bool((buf[off + x.numel():] == 7).all())
        got, ids, _ = q.fp4_moe(x, r, ex, 2, return_routing=True, out=out)
        assert got is out and ids.shape == (3, 2)
