"""Strides that the key / value operators pass to their kernels, on host tensors."""
import pytest
import torch

from qwantize_b200 import kv_cache

CPU = torch.device("cpu")


def rows(x):
    y, s0, s1 = kv_cache._rows16(x, "x", x.shape[1:], CPU)
    # what qz_kv_append and qz_kv_attention ask for
    assert s0 % 8 == 0 and s1 % 8 == 0 and y.data_ptr() % 16 == 0
    again = torch.as_strided(y, x.shape, (s0, s1, 1)) if x.numel() else y
    assert torch.equal(again, x)
    return y


@pytest.mark.parametrize("n", [0, 1, 2, 3])
@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("width,first", [(68, 0), (68, 4), (65, 0), (65, 1), (72, 8), (64, 0)])
def test_tokens_and_heads_cut_from_wider_rows(n, heads, width, first):
    """A dimension of one element keeps whatever stride it was cut with, also through
    contiguous(): it is no reason to refuse the call."""
    buf = torch.arange(4 * heads * width, dtype=torch.float32).to(torch.bfloat16).reshape(4, heads, width)
    rows(buf[:n, :, first: first + 64] if first + 64 <= width else buf[:n, :, width - 64:])
    rows(buf.transpose(0, 1).contiguous().transpose(0, 1)[:n, :, :64])


def test_what_is_aligned_is_not_copied():
    buf = torch.zeros(4, 12, 64, dtype=torch.float16)
    for x in (buf, buf[:, 2:10], buf[1:2, 3:4], buf[::2]):
        assert rows(x).data_ptr() == x.data_ptr()


@pytest.mark.parametrize("value,kept", [(2**31 - 1, 2**31 - 1), (2**31, 2**31 - 1), (2**32, 2**31 - 1), (2**63 - 1, 2**31 - 1), (-1, -1), (-(2**31) - 1, -(2**31)),
                                        (-(2**40), -(2**31)), (7, 7)])
def test_indices_of_64_bits_do_not_wrap(value, kept):
    """A length that stands for "all", or a page that no cache has, stays what it is."""
    t = kv_cache._index(torch.tensor([value, 3]), "lengths", CPU, 1)
    assert t.dtype == torch.int32 and t.tolist() == [kept, 3]
