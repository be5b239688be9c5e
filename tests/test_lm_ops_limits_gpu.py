"""What the entry points of the token table, the token log probabilities and the gated scan refuse before anything is launched.
Every call here lacks a pointer that it needs, so none of them could run."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
NEAR = 2 ** 31 - 1 - 65535  # the first size that 32-bit loops could step past


@pytest.fixture()
def refused(cuda_dev):
    from mamba_rs_b200 import ffi
    h = ffi.default_handle(0)

    def call(name, *args):
        rc = getattr(ffi.lib(), "mamba_b200_" + name)(h.ptr, None, *args)
        assert rc < 0
        return ffi.lib().mamba_b200_last_error(h.ptr).decode()
    return call


def test_sizes_beyond_32_bit_loops(refused):
    from mamba_rs_b200 import ffi
    for big in (NEAR, 2 ** 31 - 1):
        assert "too many" in refused("embedding_fwd", 0, None, big, None, 0, None, big, 1, big, 1, 1.0)
        assert "too many" in refused("embedding_bwd", 0, None, 1, None, None, 0, big, 1, 1, 1.0, None, 0)
        assert "too many" in refused("embedding_bwd", 0, None, 1, None, None, 0, 1, 1, big, 1.0, None, 0)
        assert "too many" in refused("token_logprobs", 0, None, big, None, 1.0, None, None, None, 0, None, None, 1, big)
        assert "too many" in refused("token_logprobs_bwd", 0, None, big, None, 1.0, None, None, None, None, None, big, 1, big)
        for B, T, D in ((1, big, 1), (1, 1, big), (1, 100, big)):
            a = ffi.GatedScanArgs(dtype=0, B=B, T=T, D=D, ld_x=D, ld_f=D, ld_y=D, ld_dy=D, ld_dx=D, ld_df=D)
            assert "too many" in refused("gated_scan_fwd", C.byref(a))
            assert "too many" in refused("gated_scan_bwd", C.byref(a))
            assert ffi.lib().mamba_b200_gated_scan_workspace_bytes(B, T, D) == 0
    # one less is a size like any other: what is missing is a pointer
    ok = NEAR - 1
    assert "null" in refused("embedding_fwd", 0, None, ok, None, 0, None, ok, 1, ok, 1, 1.0)
    assert "null" in refused("embedding_bwd", 0, None, 1, None, None, 0, ok, 1, ok, 1.0, None, 0)
    assert "null" in refused("token_logprobs", 0, None, ok, None, 1.0, None, None, None, 0, None, None, 1, ok)
    assert "null" in refused("token_logprobs_bwd", 0, None, ok, None, 1.0, None, None, None, None, None, ok, 1, ok)
    a = ffi.GatedScanArgs(dtype=0, B=1, T=ok, D=ok, ld_x=ok, ld_f=ok, ld_y=ok, ld_dy=ok, ld_dx=ok, ld_df=ok)
    assert "null" in refused("gated_scan_fwd", C.byref(a)) and "null" in refused("gated_scan_bwd", C.byref(a))
