"""Group norm with channels last, activation and gate, forward and backward, against 64 bits.

Tolerances.  n values of a group are summed in 32 bits pairwise or in runs: the mean is off by at most 2^-24 (8 + log2 n + n / 256) of
the largest magnitude, a run of one thread being a 256th of a group at the longest; e below is that.  rstd is taken around the mean, so
its relative error is 2 e and an error of the mean as a part of the deviation, which counts twice: with r = max |x| rstd, xh is off by
at most e r + 4 e |xh| and v by that times |w|.  Activation and gate are off by 2^-18 of theirs in 16 bits (approximate exponential
and reciprocal) and 2^-21 in f32, slopes are at most 1.13.  Results add half a step."""
import math

import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]


def sizes(S, per):
    n = S * per
    return 2.0 ** -24 * (8 + math.log2(n) + n / 256)


def inputs(dev, dt, N, S, C, gate, seed=0, pad=0):
    import torch

    from retention_ref import DT
    g = torch.Generator(dev).manual_seed(seed + N + 13 * S + C)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    rows = lambda t: torch.empty(N, S, C + pad, device=dev, dtype=DT[dt])[..., pad:].copy_(t)  # noqa: E731
    x = rows(rn(N, S, C) * (0.3 + torch.rand(C, device=dev, generator=g)) + 2.0 * rn(C))
    return x, rows(rn(N, S, C)) if gate else None, 1.0 + 0.3 * rn(C), 0.3 * rn(C), rows(rn(N, S, C))


SHAPES = [(1, 1, 1, 1), (3, 1, 8, 1), (5, 1, 64, 8), (70, 1, 2048, 32), (33, 1, 96, 4), (9, 1, 120, 5), (4, 1, 1024, 1), (2, 1, 2048, 1), (3, 1, 36, 12),
          (7, 1, 77, 7), (2, 1, 9000, 2), (1500, 1, 64, 4), (2, 2, 64, 32), (3, 50, 768, 32), (1, 777, 24, 3), (2, 130, 33, 11), (1, 3000, 8, 1),
          (20, 3, 40, 5), (2, 40, 6000, 2), (1, 2, 1300, 1), (300, 2, 16, 2)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("activation,gate", [(None, False), ("silu", False), ("gelu", True), (None, True)])
@pytest.mark.parametrize("N,S,C,G", SHAPES)
def test_forward_and_backward(cuda_dev, dt, activation, gate, N, S, C, G):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import HALF, TINY, fro, group_norm
    pad = 0 if C % 8 == 0 and (N + S) % 2 else 3
    x, z, w, b, dy = inputs(cuda_dev, dt, N, S, C, gate, pad=pad)
    eps, per, u = 1e-3, C // G, HALF[dt]
    leaves = [t.double().requires_grad_() for t in (x, w, b)] + ([z.double().requires_grad_()] if gate else [])
    want, mean, rstd = group_norm(leaves[0], leaves[1], leaves[2], G, eps, activation, leaves[3] if gate else None)
    grads = torch.autograd.grad(want, leaves, dy.double())
    want, mean, rstd = want.detach(), mean.detach(), rstd.detach()
    e = sizes(S, per)
    y, stats = mb.group_norm_fwd(x, w, b, G, eps=eps, activation=activation, z=z)
    big = x.double().abs().view(N, S, G, per).amax((1, 3))
    assert ((stats[0].double() - mean).abs() <= e * big).all()
    r = big * rstd  # (a deviation is off by an error of the mean too)
    assert ((stats[1].double() - rstd).abs() <= (2 * e * (1 + r * e) + 4 * e + e * r) * rstd).all()
    spread = lambda t: t[:, None, :, None].expand(N, S, G, per).reshape(N, S, C)  # noqa: E731
    xh = (x.double() - spread(mean)) * spread(rstd)
    f = 2.0 ** -18 if dt != "f32" else 2.0 ** -21
    sz = 1.0 if z is None else (z.double() * torch.sigmoid(z.double())).abs()
    v_err = (e * spread(r) * 2 + 8 * e * xh.abs()) * w.abs().double() + 2.0 ** -23 * (xh * w + b).abs()
    bound = 1.13 * v_err * sz + (u * 1.01 + f) * want.abs() + (f * sz if activation else 0.0) + TINY[dt] + (1e-30 if gate else 0.0)
    assert ((y.double() - want).abs() <= bound).all(), float(((y.double() - want).abs() / bound).max())
    # backward, from stats rounded to 32 bits: through the same xh
    got = mb.group_norm_bwd(dy, x, stats, w, b, G, activation=activation, z=z)
    n = N * S
    # errors of a gradient's parts are those of v (slopes change by at most 1.13 of it, gates by 1.1) and of the sums over a group; their norm
    # stays within a few e of the whole, d_weight and d_bias are sums over rows in 32 bits
    soft = 16 * (e * (1 + float(r.max())) + f)
    if per * S > 1:
        assert fro(got["d_x"], grads[0]) <= 1.2 * u + soft * (1 + float((dy.double().norm() * w.double().abs().max() * rstd.max()) / grads[0].norm()))
    assert fro(got["d_bias"], grads[2]) <= (soft + 2.0 ** -24 * n) * float(dy.double().abs().sum((0, 1)).norm() * 1.3 / grads[2].norm())
    size = (dy.double().abs() * xh.abs()).sum((0, 1)).norm() * 1.3
    assert fro(got["d_weight"], grads[1]) <= (soft + 2.0 ** -24 * n) * float(size / grads[1].norm().clamp(min=1e-30)) + (1.0 if per * S == 1 else 0.0)
    if gate:
        assert fro(got["d_z"], grads[3]) <= 1.2 * u + soft * 4
    # given results are added to (weights) or overwritten; the same bits again
    dw, db = torch.full_like(w, 2.0), torch.full_like(b, -1.0)
    d_x = dy.clone()
    again = mb.group_norm_bwd(dy, x, stats, w, b, G, activation=activation, z=z, d_x=d_x, d_weight=dw, d_bias=db)
    assert torch.equal(d_x, got["d_x"]) and torch.equal(dw, 2.0 + got["d_weight"]) and torch.equal(db, -1.0 + got["d_bias"])
    d_x.copy_(dy)
    zz = None if z is None else z.clone()
    mb.group_norm_bwd(d_x, x, stats, w, b, G, activation=activation, z=zz, d_x=d_x, d_z=zz)  # in the inputs' place
    assert torch.equal(d_x, got["d_x"]) and (z is None or torch.equal(zz, got["d_z"]))
    y2, s2 = mb.group_norm_fwd(x, w, b, G, eps=eps, activation=activation, z=z)
    assert torch.equal(y2, y) and torch.equal(s2, stats) and again["d_x"].shape == x.shape


def test_rows_as_a_matrix_without_weights(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    x = torch.randn(37, 128, device=cuda_dev)
    y, stats = mb.group_norm_fwd(x, None, None, 4)
    w, s3 = mb.group_norm_fwd(x[:, None], torch.ones(128, device=cuda_dev), torch.zeros(128, device=cuda_dev), 4)
    assert y.shape == (37, 128) and torch.equal(y, w[:, 0]) and torch.equal(stats, s3)
    g = mb.group_norm_bwd(x, x, stats, None, None, 4)
    assert torch.equal(g["d_x"], mb.group_norm_bwd(x[:, None], x[:, None], stats, torch.ones(128, device=cuda_dev), None, 4)["d_x"][:, 0])


def test_values_far_from_zero(cuda_dev):
    """A mean of 4096 deviations: around the mean the variance keeps its digits (in f32; E[x^2] - E[x]^2 would have lost them all)."""
    import torch

    import mamba_rs_b200 as mb
    gen = torch.Generator(cuda_dev).manual_seed(2)
    for N, S, C, G in ((6, 1, 512, 4), (2, 300, 64, 2)):
        x = torch.randn(N, S, C, device=cuda_dev, generator=gen) + 4096.0
        _, stats = mb.group_norm_fwd(x, None, None, G, eps=0.0)
        g = x.double().view(N, S, G, C // G)
        rstd = g.var((1, 3), correction=0).rsqrt()
        # each x is a number of its own: deviations are exact differences of f32 numbers to an error of the mean of 4096 2^-24 (8 + log2 n), which
        # counts squared, and to 2^-24 of themselves
        assert ((stats[1].double() / rstd - 1).abs() <= 2.0 ** -17).all()


def test_gradients_against_differences(cuda_dev):
    """Central differences in f32: steps of 2^-8 leave 2^-16 of a third derivative of order one, roundings 2^-22 / 2^-8 of the sum's terms."""
    import torch

    import mamba_rs_b200 as mb
    for S, act in ((1, "silu"), (9, "gelu")):
        x, z, w, b, dy = inputs(cuda_dev, "f32", 4, S, 24, True, seed=3)
        x = x - x.mean((0, 1))
        _, stats = mb.group_norm_fwd(x, w, b, 3, activation=act, z=z)
        g = mb.group_norm_bwd(dy, x, stats, w, b, 3, activation=act, z=z)
        gen = torch.Generator(cuda_dev).manual_seed(7)
        base = [x, w, b, z]
        for i, name in enumerate(("d_x", "d_weight", "d_bias", "d_z")):
            way = torch.randn(base[i].shape, device=cuda_dev, generator=gen)
            way /= way.norm()
            ends = []
            for h in (2.0 ** -8, -2.0 ** -8):
                args = list(base)
                args[i] = base[i] + h * way
                y, _ = mb.group_norm_fwd(args[0], args[1], args[2], 3, activation=act, z=args[3])
                ends.append(float((y.double() * dy.double()).sum()))
            want = float((g[name].double() * way.double()).sum())
            size = float(g[name].double().norm()) + float(dy.double().norm())
            assert abs((ends[0] - ends[1]) * 2.0 ** 7 - want) <= 2.0 ** -9 * size, (S, name)


def test_nothing_to_do_and_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    x = torch.randn(3, 4, 12, device=cuda_dev)
    w, b = torch.ones(12, device=cuda_dev), torch.zeros(12, device=cuda_dev)
    for e in (x[:0], x[:, :0]):
        y, stats = mb.group_norm_fwd(e, w, b, 3)
        assert y.shape == e.shape
        g = mb.group_norm_bwd(y, e, stats, w, b, 3)
        assert not g["d_weight"].any() and not g["d_bias"].any()
    _, stats = mb.group_norm_fwd(x, w, b, 3)
    for call in (lambda: mb.group_norm_fwd(x, w, b, 5), lambda: mb.group_norm_fwd(x, w, b, 0), lambda: mb.group_norm_fwd(x[0, 0], w, b, 3),
                 lambda: mb.group_norm_fwd(x, w, b, 3, activation="tanh"), lambda: mb.group_norm_fwd(x.transpose(0, 1), w, b, 3),
                 lambda: mb.group_norm_fwd(x.transpose(1, 2), w[:4], b[:4], 2), lambda: mb.group_norm_fwd(x, w, b, 3, y=x[:, :1].expand(3, 4, 12)),
                 lambda: mb.group_norm_bwd(x, x, stats, w, b, 3, d_weight=w.clone())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: mb.group_norm_fwd(x, w[:11], b, 3), lambda: mb.group_norm_fwd(x, w.half(), b, 3), lambda: mb.group_norm_fwd(x.double(), w, b, 3),
                 lambda: mb.group_norm_fwd(x, w, b, 3, z=x.half()), lambda: mb.group_norm_bwd(x, x, stats[:, :2], w, b, 3),
                 lambda: mb.group_norm_bwd(x, x, stats, w, b, 3, d_weight=w.double(), d_bias=b.double())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mb.group_norm_fwd(x.cpu(), w, b, 3)
    for eps in (-1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="eps"):
            mb.group_norm_fwd(x, w, b, 3, eps=eps)
    with pytest.raises(RuntimeError, match="workspace"):
        mb.group_norm_bwd(x, x, stats, w, b, 3, workspace=torch.empty(256, dtype=torch.uint8, device=cuda_dev))
