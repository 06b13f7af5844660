"""Arguments of the serving operators that no kernel may see: refused on the host
before any device call."""
import pytest

from qwantize_b200 import _lib


def moe(**kw):
    """qz_moe with made-up addresses that pass every check but the one under test
    (and at last, that of the workspace's size)."""
    ok = dict(x=256, dt=1, ldx=64, T=2, H=64, I=32, E=4, top=2, renorm=1, r=256, rd=0, fmt=0, uc=256, us=256, un=256, ut=1.0, dc=256, ds=256,
              dt2=1.0, out=256, ids=None, w=None, ws=256, n=0, st=None)
    return _lib.load().qz_moe(*{**ok, **kw}.values())


def refused(status, word):
    assert status == _lib.QZ_ERR_INVALID
    assert word in _lib.load().qz_last_error(), _lib.load().qz_last_error()


@pytest.mark.parametrize("off", [2, 4, 6, 10])
def test_moe_out_off_the_8_bytes_that_are_stored_at_once(off):
    refused(moe(), b"workspace of 0 bytes")
    refused(moe(out=256 + 8), b"workspace of 0 bytes")
    refused(moe(out=256 + off), b"aligned")


def test_moe_norms_off_the_8_bytes_that_are_loaded_at_once():
    refused(moe(un=256 + 4), b"aligned")


def test_a_cache_in_host_memory_is_refused():
    import qwantize_b200 as q
    with pytest.raises(AssertionError, match="CUDA device"):
        q.KVCache8(4, 2, 64, device="cpu")
