"""Rotation by position against 64 bits.

Tolerances.  The angle is a product of a position and an f32 frequency in 64 bits, rounded to 32 after whole turns are gone: off by at
most 2^-25 of half a turn, 2^-23 rad; sine and cosine are off by 2^-23 of theirs at most beside that, the three products and the sum by
2^-24 each: |error| <= 2^-21 scale (|a| + |b|) and half a step of the result.  Columns that are handed on are the same bits."""
import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]


def close(got, x, want, n, scale, dt):
    from retention_ref import HALF, TINY
    size = x.double().abs()
    if n:
        bound = 2.0 ** -21 * scale * 2 * size[..., :2 * n].amax(-1, keepdim=True) + HALF[dt] * 1.01 * want.abs()[..., :2 * n] + TINY[dt]
        assert ((got.double() - want).abs()[..., :2 * n] <= bound).all()
    assert (got[..., 2 * n:] == x[..., 2 * n:]).all()


SHAPES = [(1, 1, 1, 1, 2, 2), (2, 1, 8, 2, 64, 64), (3, 17, 4, 4, 128, 64), (1, 130, 2, 1, 80, 80), (2, 33, 3, 3, 37, 22), (1, 5, 40, 1, 256, 256),
          (2, 300, 4, 2, 96, 48), (1, 7, 2, 2, 64, 0), (1, 9, 1, 1, 1024, 1000), (4, 11, 5, 1, 192, 86)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,Hk,D,R", SHAPES)
def test_rotation(cuda_dev, dt, interleaved, B, T, H, Hk, D, R):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import DT, rotary
    g = torch.Generator(cuda_dev).manual_seed(R + D)
    proj = torch.randn(B, T, (H + Hk) * D, device=cuda_dev, generator=g).to(DT[dt])
    q, k = proj[..., :H * D].unflatten(-1, (H, D)), proj[..., H * D:].unflatten(-1, (Hk, D))
    freq = mb.rotary_frequencies(R, device=cuda_dev)[0] if R else torch.empty(0, device=cuda_dev)
    for positions in (torch.arange(T, device=cuda_dev, dtype=torch.int32), torch.randint(-5000000, 5000000, (B, T), device=cuda_dev, generator=g).int()):
        for f, inverse in ((mb.rotary_fwd, False), (mb.rotary_bwd, True)):
            got = f(q, k, positions, freq, interleaved=interleaved, scale=1.25)
            for x, y in zip((q, k), got):
                close(y, x, rotary(x, positions, freq, interleaved, 1.25, inverse), R // 2, 1.25, dt)
            # q alone; in place; into columns of a larger tensor; other starts and strides than 16 bytes
            assert torch.equal(f(q, None, positions, freq, interleaved=interleaved, scale=1.25)[0], got[0])
            a, b = q.clone(), k.clone()
            r = f(a, b, positions, freq, interleaved=interleaved, scale=1.25, q_out=a, k_out=b)
            assert r[0] is a and torch.equal(a, got[0]) and torch.equal(b, got[1])
            big = torch.full((B, T, (H + Hk) * D + 3), 7.0, device=cuda_dev, dtype=q.dtype)
            qo, ko = big[..., 1:1 + H * D].unflatten(-1, (H, D)), big[..., 1 + H * D:1 + (H + Hk) * D].unflatten(-1, (Hk, D))
            f(q, k, positions, freq, interleaved=interleaved, scale=1.25, q_out=qo, k_out=ko)
            assert torch.equal(qo, got[0]) and torch.equal(ko, got[1]) and (big[..., 0] == 7).all() and (big[..., -2:] == 7).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_is_the_rotation_back(cuda_dev, interleaved):
    """<rotate(x), y> = <x, rotate_bwd(y)>, and rotating back with scale 1 gives x: sums of 64 x 8 x 40 products in 64 bits of values that are
    off by 2^-21 of theirs."""
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(1)
    x, y = (torch.randn(2, 40, 4, 64, device=cuda_dev, generator=g) for _ in range(2))
    pos = torch.randint(0, 100000, (2, 40), device=cuda_dev, generator=g).int()
    freq, scale = mb.rotary_frequencies(48, scaling="yarn", factor=8.0, trained=4096, device=cuda_dev)
    kw = dict(interleaved=interleaved, scale=scale)
    a = mb.rotary_fwd(x, None, pos, freq, **kw)[0].double() * y.double()
    b = mb.rotary_bwd(y, None, pos, freq, **kw)[0].double() * x.double()
    assert abs(float(a.sum() - b.sum())) <= 2.0 ** -20 * float(a.abs().sum())
    back = mb.rotary_bwd(mb.rotary_fwd(x, None, pos, freq, interleaved=interleaved)[0], None, pos, freq, interleaved=interleaved)[0]
    assert float((back - x).abs().max()) <= 2.0 ** -19 * float(x.abs().max())


def test_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    q = torch.randn(2, 3, 4, 16, device=cuda_dev)
    pos, freq = torch.arange(3, device=cuda_dev, dtype=torch.int32), torch.ones(8, device=cuda_dev)
    assert mb.rotary_fwd(q[:, :0], None, pos[:0], freq)[0].shape == (2, 0, 4, 16) and mb.rotary_fwd(q[:0], q[:0], pos, freq)[1].shape == (0, 3, 4, 16)
    for call in (lambda: mb.rotary_fwd(q, None, pos.long(), freq), lambda: mb.rotary_fwd(q, None, pos[:2], freq),
                 lambda: mb.rotary_fwd(q, None, pos, torch.ones(9, device=cuda_dev)), lambda: mb.rotary_fwd(q, None, pos, freq.double()),
                 lambda: mb.rotary_fwd(q, q.half(), pos, freq), lambda: mb.rotary_fwd(q.double(), None, pos, freq),
                 lambda: mb.rotary_fwd(q, None, pos, freq, q_out=q[..., :8])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: mb.rotary_fwd(q[0], None, pos, freq), lambda: mb.rotary_fwd(q.transpose(2, 3), None, pos, freq[:2]),
                 lambda: mb.rotary_fwd(q, None, pos, freq, q_out=q[:, :, :1].expand(2, 3, 4, 16))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mb.rotary_fwd(q, None, pos.cpu(), freq)
    with pytest.raises(RuntimeError, match="scale"):
        mb.rotary_fwd(q, None, pos, freq, scale=float("nan"))
    flat = torch.randn(2 * 3 * 4 * 16, device=cuda_dev)
    with pytest.raises(RuntimeError, match="other strides"):
        mb.rotary_fwd(flat.view(2, 3, 4, 16), None, pos, freq, q_out=flat.view(2, 4, 3, 16).transpose(1, 2))
