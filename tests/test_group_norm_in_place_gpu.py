"""Group norm's results in the place of its inputs: with the same row strides, and refused with others before anything is launched."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,S", [(3, 1), (1, 2), (4, 5)])
def test_other_strides_are_refused(cuda_dev, N, S):
    """(The C entries lack the workspace that samples need, or a pointer; no call could run.)"""
    from mamba_rs_b200 import ffi
    h = ffi.default_handle(0)
    at = lambda i: C.c_void_p(4096 * (i + 1))  # noqa: E731

    def refused(name, **kw):
        a = ffi.GroupNormArgs(**{**dict(dtype=0, N=N, S=S, C=8, G=1, eps=1e-5, **{n: 8 for n in ("ld_x", "ld_z", "ld_y", "ld_dy", "ld_dx", "ld_dz")}), **kw})
        rc = getattr(ffi.lib(), "mamba_b200_" + name)(h.ptr, None, C.byref(a))
        assert rc < 0
        return ffi.lib().mamba_b200_last_error(h.ptr).decode()

    fwd = dict(x=at(0), z=at(1), y=at(2))
    for n in ("x", "z"):
        assert "other strides" in refused("group_norm_fwd", **{**fwd, "y": fwd[n], "ld_y": 16})
        assert "other strides" in refused("group_norm_fwd", **{**fwd, "y": fwd[n], "ld_" + n: 24})
    bwd = dict(x=at(0), z=at(1), dy=at(2), stats=at(3), d_x=at(4), d_z=at(5))
    for out, ld in (("d_x", "ld_dx"), ("d_z", "ld_dz")):
        for n in ("x", "z", "dy"):
            assert "other strides" in refused("group_norm_bwd", **{**bwd, out: bwd[n], ld: 16}), (out, n)


def test_views_with_other_strides_are_refused(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    base = torch.randn(64, 32, device=cuda_dev)
    x, wide = base[:32, :16], base.view(32, 64)[:, :16]  # the same first element, rows 32 and 64 apart
    w, b = torch.ones(16, device=cuda_dev), torch.zeros(16, device=cuda_dev)
    before = base.clone()
    z = torch.randn(32, 16, device=cuda_dev)
    y, stats = mb.group_norm_fwd(z, w, b, 4)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.group_norm_fwd(x, w, b, 4, y=wide)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.group_norm_fwd(z, w, b, 4, z=x, y=wide)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.group_norm_bwd(z, x, stats, w, b, 4, d_x=wide)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.group_norm_bwd(x, z, stats, w, b, 4, d_x=wide)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.group_norm_bwd(z, y, stats, w, b, 4, z=x, d_z=wide)
    assert torch.equal(base, before)


@pytest.mark.parametrize("N,S", [(100, 1), (6, 40), (2, 4000)])
def test_the_same_strides_are_taken(cuda_dev, N, S):
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(N)
    both = torch.randn(N, S, 128, device=cuda_dev, generator=g)
    dy = torch.randn(N, S, 64, device=cuda_dev, generator=g)
    w, b = (torch.randn(64, device=cuda_dev, generator=g) for _ in range(2))
    x, z = both[..., :64], both[..., 64:]
    y, stats = mb.group_norm_fwd(x, w, b, 4, z=z)
    want = mb.group_norm_bwd(dy, x, stats, w, b, 4, z=z)
    for i in (0, 1):
        copy = both.clone()
        v = (copy[..., :64], copy[..., 64:])
        assert torch.equal(mb.group_norm_fwd(v[0], w, b, 4, z=v[1], y=v[i])[0], y)
        assert torch.equal(copy[..., 64 * (1 - i):64 * (2 - i)], both[..., 64 * (1 - i):64 * (2 - i)])
    copy = both.clone()
    got = mb.group_norm_bwd(dy, copy[..., :64], stats, w, b, 4, z=copy[..., 64:], d_x=copy[..., :64], d_z=copy[..., 64:])
    for n in ("d_x", "d_z", "d_weight", "d_bias"):
        assert torch.equal(got[n], want[n]), n
