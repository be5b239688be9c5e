"""What the entry points of the token table, the token log probabilities and the gated scan refuse before anything is launched.
The calls of the C entries here lack a pointer that they need, so none of them could run."""
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


def test_pointers_between_elements(refused):
    """Each pointer alone, the others null."""
    from mamba_rs_b200 import ffi
    for dtype, odd in ((ffi.F32, 2), (ffi.BF16, 1)):
        store, words = C.c_void_p(4096 + odd), C.c_void_p(4096 + 2)
        for i, at in ((0, store), (1, words), (2, store)):
            p = [at if k == i else None for k in range(3)]
            assert "misaligned" in refused("embedding_fwd", dtype, p[0], 8, p[1], dtype, p[2], 8, 1, 8, 8, 1.0)
            assert "misaligned" in refused("embedding_bwd", dtype, p[0], 8, p[1], words if i == 2 else None, 0, 1, 8, 8, 1.0, None, 0)
        # an f32 result of a 16-bit table
        assert "misaligned" in refused("embedding_fwd", dtype, None, 8, None, ffi.F32, words, 8, 1, 8, 8, 1.0)
        for i in range(7):
            p = [(store if k == 0 else words) if k == i else None for k in range(7)]
            assert "misaligned" in refused("token_logprobs", dtype, p[0], 8, p[1], 1.0, p[2], p[3], p[4], 1, p[5], p[6], 1, 8)
            p = [(store if k in (0, 6) else words) if k == i else None for k in range(7)]
            assert "misaligned" in refused("token_logprobs_bwd", dtype, p[0], 8, p[1], 1.0, *p[2:6], p[6], 8, 1, 8)
        sizes = dict(dtype=dtype, B=1, T=3, D=8, ld_x=8, ld_f=8, ld_z=8, ld_y=8, ld_dy=8, ld_dx=8, ld_df=8, ld_dz=8)
        for names, at, fwd, bwd in ((("x", "f", "z"), store, True, True), (("y",), store, True, False), (("dy", "d_x", "d_f", "d_z"), store, False, True),
                                    (("h0", "h_last"), words, True, False), (("d_last", "d_h0"), words, False, True), (("chunk_states",), words, True, True)):
            for name in names:
                a = ffi.GatedScanArgs(**sizes, **{name: at})
                if fwd:
                    assert "misaligned" in refused("gated_scan_fwd", C.byref(a)), name
                if bwd:
                    assert "misaligned" in refused("gated_scan_bwd", C.byref(a)), name


def test_a_workspace_that_is_less_memory_than_it_has_elements(cuda_dev):
    """An expanded or strided tensor's elements are not its memory."""
    import torch

    import mamba_rs_b200 as mb
    ids, d = torch.zeros(600, dtype=torch.int32, device=cuda_dev), torch.ones(600, 8, device=cuda_dev)
    need = mb.embedding_bwd_workspace_bytes(600, 8, 5)
    assert need > 0
    one = torch.zeros(1, dtype=torch.uint8, device=cuda_dev)
    for ws in (one.expand(need), torch.zeros(2 * need, dtype=torch.uint8, device=cuda_dev)[::2]):
        with pytest.raises(ValueError, match="contiguous"):
            mb.embedding_bwd(ids, d, 5, workspace=ws)
    x = torch.zeros(1, 1300, 40, device=cuda_dev)
    with pytest.raises(ValueError, match="contiguous"):
        mb.gated_scan_fwd(x, x, workspace=one.expand(mb.gated_scan_workspace_bytes(1, 1300, 40)))
