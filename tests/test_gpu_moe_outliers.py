"""Activations of experts whose rows differ widely in size."""
import pytest
import torch

from tests.test_gpu_linear import BLOCK
from tests.test_gpu_moe import check, router_of, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("up_bits", [0, 6, 12])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_large_gate_row_and_another_large_up_row(up_bits, dtype):
    """The scale of an activation row comes from a bound.  A gate row and the up row
    of another output that are 2^12 times the rest each make one activation 2^12
    times the rest, not 2^24: nothing may be scaled by the product of both.  The
    down rows weigh those two outputs as little as they are large, so that the
    result is made up of the others."""
    import qwantize_b200 as q
    E, H, I, bits = 2, 256, 96, 12
    g = torch.Generator().manual_seed(60 + up_bits)
    up = torch.randn(E, 2 * I, H, generator=g) / H**0.5
    down = torch.randn(E, H, I, generator=g) / I**0.5
    up[:, 3] *= 2.0**bits              # gate row of output 3
    up[:, I + 64] *= 2.0**up_bits      # up row of output 64
    # one block of 32 columns for each of the two: their scales do not touch the rest
    down[:, :, 0:32] *= 2.0 ** -(bits + 4)
    down[:, :, 64:96] *= 2.0 ** -(up_bits + 4)
    pack = lambda w: q.mxfp4_quantize_packed(w.to(DEV, torch.bfloat16).reshape(*w.shape[:-1], -1, BLOCK["mxfp4"]))  # noqa: E731
    check(tokens(3, H, dtype, 61), router_of(E, H, torch.float32, 62), pack(up), pack(down), "mxfp4", 1.0, 2)


@pytest.mark.parametrize("shift", [-90, 80])
def test_weights_far_from_one(shift):
    """MXFP4 scales reach any power of two: weights whose squares leave fp32's range,
    and tokens that bring the products back."""
    H, I = 64, 96
    g = torch.Generator().manual_seed(70)
    pack = lambda w: q.mxfp4_quantize_packed(w.to(DEV, torch.bfloat16).reshape(*w.shape[:-1], -1, BLOCK["mxfp4"]))  # noqa: E731
    import qwantize_b200 as q
    up, down = pack(torch.randn(2, 2 * I, H, generator=g) / H**0.5), pack(torch.randn(2, H, I, generator=g) / I**0.5)
    far = (up[0].int() + shift).to(torch.uint8)
    x = tokens(3, H, torch.bfloat16, 71) * 2.0**-shift
    check(x, torch.zeros(2, H, device=DEV), (far, up[1]), down, "mxfp4", 1.0, 2)
