"""The gated linear recurrence, forward, backward and step, against the recurrence in 64 bits, step by step.

Tolerances.  u = sigmoid(-f) has a relative error e_u of at most 2^-21 (2 + |f|).  A state is a mean of earlier inputs whose
weights are products of u and (1 - u): an error e_u in each u moves it by at most 2 e_u times the largest |x| or |h0|
(weights near a change of u are shifted to the neighbours); every step's own rounding, 2^-24 of the magnitudes, lasts for
1 / u steps.  With W = the largest of |x|, |h0|, and n = the longest memory (at most T) an error of a state is below
(2 e_u + 3 n 2^-24) W; joining spans of steps rounds each join once more, counted by the 3.  The backward's g is a sum whose
terms are weighted the same way, so its bound has W = the largest sum of |dy SiLU(z)| over a memory.  16-bit results add half an ulp."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DT = ["f32", "bf16", "f16"]
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _inputs(B, T, D, dt, dev, gate=True, seed=0, pad=0, slow=True):
    """x, f, z as columns of one projection (pad: columns more between them), with h0."""
    import torch
    g = torch.Generator(dev).manual_seed(seed + B * T + D)
    w = 3 if gate else 2
    proj = torch.randn(B, T, w * (D + pad) + pad, device=dev, generator=g)
    at = [pad + i * (D + pad) for i in range(w)]
    if slow:  # memories of 2 to 500 steps
        rate = torch.exp(torch.rand(D, device=dev, generator=g) * math.log(250.0)) / 500
        proj[..., at[1]:at[1] + D] += torch.log1p(-rate) - torch.log(rate)
    proj = proj.to(_dt(dt))
    x, f, z = [proj[..., a:a + D] for a in at] + [None] * (3 - w)
    return x, f, z, torch.randn(B, D, device=dev, generator=g)


def _plain(x, f, z, h0):
    """h of every step, and y."""
    import torch
    x, f = x.double(), f.double()
    u = 1.0 / (1.0 + torch.exp(f))
    h, hs = h0.double(), torch.empty_like(x)
    for t in range(x.shape[1]):
        h = (1.0 - u[:, t]) * h + u[:, t] * x[:, t]
        hs[:, t] = h
    y = hs if z is None else hs * z.double() * torch.sigmoid(z.double())
    return hs, y, h


def _state_tol(x, f, h0):
    import torch
    e_u = 2.0 ** -21 * (2 + float(f.double().abs().max())) if f.numel() else 0.0
    u = torch.sigmoid(-f.double())
    n = min(x.shape[1], 1.0 / max(float(u.mean(1).min()), 1e-9)) if f.numel() else 0
    W = max(float(x.double().abs().max()) if x.numel() else 0.0, float(h0.abs().max()))
    return (2 * e_u + 3 * max(n, 1) * 2.0 ** -24) * W


SHAPES = [(1, 1, 1), (2, 1, 5), (1, 2, 33), (3, 63, 64), (2, 64, 40), (2, 65, 7), (1, 200, 768), (4, 129, 96), (2, 1000, 31), (1, 2500, 64),
          (1, 5003, 24), (33, 17, 130), (16, 300, 520)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_forward(cuda_dev, dt, gate, B, T, D):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, gate)
    for start in (h0, None):
        hs, y, last = _plain(x, f, z, torch.zeros_like(h0) if start is None else start)
        tol = _state_tol(x, f, h0)
        h_last, cs = torch.empty_like(h0), torch.full(mb.gated_scan_states(B, T, D), 9.0, device=cuda_dev)
        got = mb.gated_scan_fwd(x, f, z, h0=start, h_last=h_last, chunk_states=cs)
        gz = 1.0 if z is None else (z.double() * torch.sigmoid(z.double())).abs()
        assert ((got.double() - y).abs() <= tol * (gz + 0.0) + (HALF[dt] * 1.01 + 2.0 ** -20) * y.abs() + TINY[dt]).all()
        assert ((h_last.double() - last).abs() <= tol).all()
        want = torch.cat([(torch.zeros_like(h0) if start is None else start)[:, None].double(), hs[:, 63:-1:64]], 1)
        assert ((cs.double() - want).abs() <= tol).all()
        # the same bits again, without what is optional
        assert torch.equal(got, mb.gated_scan_fwd(x, f, z, h0=start))
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_backward(cuda_dev, dt, gate, B, T, D):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, gate, seed=1)
    g_ = torch.Generator(cuda_dev).manual_seed(T)
    dy, d_last = torch.randn(B, T, D, device=cuda_dev, generator=g_).to(_dt(dt)), torch.randn(B, D, device=cuda_dev, generator=g_)
    cs = torch.empty(mb.gated_scan_states(B, T, D), device=cuda_dev)
    mb.gated_scan_fwd(x, f, z, h0=h0, chunk_states=cs)
    hs, _, _ = _plain(x, f, z, h0)
    u = torch.sigmoid(-f.double())
    before = torch.cat([h0[:, None].double(), hs[:, :-1]], 1)
    e = dy.double()
    want = {}
    if gate:
        zd = z.double()
        q = torch.sigmoid(zd)
        want["d_z"] = e * hs * (q + zd * q * (1 - q))
        e = e * zd * q
    for last in (d_last, None):
        g, mag = (torch.zeros_like(h0).double() if last is None else last.double()), None
        m = g.abs()
        dx, df, bx, bf = (torch.empty_like(e) for _ in range(4))
        st = _state_tol(x, f, h0)
        e_u = 2.0 ** -21 * (2 + float(f.double().abs().max()))
        for t in range(T - 1, -1, -1):
            g, m = g + e[:, t], m + e[:, t].abs()  # m: the same sum of magnitudes, which bounds what an error can weigh
            span = before[:, t] - x[:, t].double()
            dx[:, t], df[:, t] = g * u[:, t], g * span * u[:, t] * (1 - u[:, t])
            n = min(T, 1000.0)
            rel = 3 * e_u * (1 + 2 * math.log(1 + T)) + 3 * n * 2.0 ** -24 + 2.0 ** -19
            bx[:, t] = rel * m * u[:, t]
            bf[:, t] = (rel * m * span.abs() + m * (st + 2.0 ** -23 * (before[:, t].abs() + x[:, t].double().abs()))) * u[:, t]
            g, m = g * (1 - u[:, t]), m * (1 - u[:, t])
        want.update(d_x=dx, d_f=df, d_h0=g)
        tol = dict(d_x=bx, d_f=bf, d_h0=rel * m + 1e-30)
        if gate:
            tol["d_z"] = dy.double().abs() * (st * 1.2 + 2.0 ** -19 * hs.abs())
        got = mb.gated_scan_bwd(x, f, dy, cs, z, d_last=last)
        assert set(got) == set(want)
        for k, v in got.items():
            half = (HALF[dt] if k != "d_h0" else 2.0 ** -24) * 1.01
            assert ((v.double() - want[k]).abs() <= tol[k] + half * want[k].abs() + TINY[dt]).all(), k
        again = mb.gated_scan_bwd(x, f, dy, cs, z, d_last=last)
        assert all(torch.equal(got[k], again[k]) for k in got)
    mb.ffi.default_handle(0).check_status()


def test_gradients_agree_with_differences(cuda_dev):
    """Central differences of a loss of y and the last state, of the 64-bit recurrence around the f32 inputs."""
    import torch

    import mamba_rs_b200 as mb
    B, T, D = 2, 70, 3
    x, f, z, h0 = _inputs(B, T, D, "f32", cuda_dev, seed=3)
    g = torch.Generator(cuda_dev).manual_seed(4)
    wy, wl = torch.randn(B, T, D, device=cuda_dev, generator=g), torch.randn(B, D, device=cuda_dev, generator=g)
    cs = torch.empty(mb.gated_scan_states(B, T, D), device=cuda_dev)
    mb.gated_scan_fwd(x, f, z, h0=h0, chunk_states=cs)
    got = mb.gated_scan_bwd(x, f, wy, cs, z, d_last=wl)

    def loss(x, f, z, h0):
        _, y, last = _plain(x, f, z, h0)
        return float((y * wy).sum() + (last * wl).sum())
    eps = 1e-5
    for k, name in enumerate(("d_x", "d_f", "d_z", "d_h0")):
        for at in ([(0, 0, 0), (1, 33, 2), (0, 64, 1), (1, 69, 0)] if name != "d_h0" else [(0, 0), (1, 2)]):
            sides = []
            for s in (eps, -eps):
                v = [x.double(), f.double(), z.double(), h0.double()]
                v[k] = v[k].clone()
                v[k][at] += s
                sides.append(loss(*v))
            # differences: eps^2 times third derivatives of order one, 64-bit rounding of the loss over eps; the kernel: 1e-5
            assert abs((sides[0] - sides[1]) / (2 * eps) - float(got[name][at])) <= 2e-5, (name, at)


@pytest.mark.parametrize("dt", DT)
def test_windows_and_steps_carry_the_state_on(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    B, T, D = 3, 150, 72
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, seed=5)
    hs, y, last = _plain(x, f, z, h0)
    tol = 2 * _state_tol(x, f, h0)
    h, parts, at = h0.clone(), [], 0
    for n in (1, 64, 0, 70):
        parts.append(mb.gated_scan_fwd(x[:, at:at + n].contiguous(), f[:, at:at + n].contiguous(), z[:, at:at + n].contiguous(), h0=h, h_last=h))
        at += n
    for t in range(at, T):
        parts.append(mb.gated_scan_step(x[:, t], f[:, t], h, z[:, t])[:, None])
    got = torch.cat(parts, 1)
    gz = (z.double() * torch.sigmoid(z.double())).abs()
    assert ((got.double() - y).abs() <= tol * gz + (HALF[dt] * 1.01 + 2.0 ** -20) * y.abs() + TINY[dt]).all()
    assert ((h.double() - last).abs() <= tol).all()
    keep = h.clone()
    out = torch.empty_like(h)
    mb.gated_scan_step(x[:, 0], f[:, 0], h, h_last=out)  # (not in place, no gate)
    assert torch.equal(h, keep) and not torch.equal(out, h)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,D,pad", [(2, 130, 64, 8), (2, 130, 64, 1), (1, 700, 33, 3), (3, 90, 41, 0)])
def test_columns_of_a_projection(cuda_dev, dt, B, T, D, pad):
    """Odd strides and starts, outputs between other columns."""
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, seed=6, pad=pad)
    cs, cs2 = (torch.empty(mb.gated_scan_states(B, T, D), device=cuda_dev) for _ in range(2))
    room = torch.full((B, T, D + 2 * pad + 1), 5.0, device=cuda_dev, dtype=_dt(dt))
    y = room[..., pad:pad + D]
    mb.gated_scan_fwd(x, f, z, h0=h0, y=y, chunk_states=cs)
    c = [t.contiguous() for t in (x, f, z)]
    want = mb.gated_scan_fwd(*c, h0=h0, chunk_states=cs2)
    step = 2.0 ** -7 if dt == "bf16" else 1e-4  # (an ulp or two of the results, which are below 8 or so in both layouts)
    assert ((y.float() - want.float()).abs() <= step * (1e-3 + want.float().abs())).all() and (cs - cs2).abs().max() <= 1e-4
    assert (room[..., :pad] == 5).all() and (room[..., pad + D:] == 5).all()
    dproj = torch.full((B, T, 3 * (D + pad) + pad), 5.0, device=cuda_dev, dtype=_dt(dt))
    outs = dict(zip(("d_x", "d_f", "d_z"), (dproj[..., pad + i * (D + pad):][..., :D] for i in range(3))))
    dy = want
    mb.gated_scan_bwd(x, f, dy, cs2, z, **outs)
    ref = mb.gated_scan_bwd(c[0], c[1], dy, cs2, c[2])
    for k, v in outs.items():
        assert ((v.float() - ref[k].float()).abs() <= step * (1e-3 + ref[k].float().abs())).all(), k
    if pad:
        for i in range(4):
            assert (dproj[..., i * (D + pad):][..., :pad] == 5).all()


def test_gates_at_their_ends(cuda_dev):
    """A gate that is shut or open for good, and values that are no numbers, stay in their channel."""
    import torch

    import mamba_rs_b200 as mb
    B, T, D = 1, 200, 40
    x, f, z, h0 = _inputs(B, T, D, "f32", cuda_dev, gate=False, seed=7)
    f = f.clone()
    f[..., 0], f[..., 1], f[..., 2], f[..., 3] = 200.0, -200.0, math.inf, -math.inf
    x = x.clone()
    x[0, 50, 4] = math.nan
    x[0, 60, 5] = math.inf
    h_last = torch.empty_like(h0)
    y = mb.gated_scan_fwd(x, f, h0=h0, h_last=h_last)
    assert (y[..., 0] == h0[:, 0]).all() and (y[..., 2] == h0[:, 2]).all()      # kept
    assert ((y[..., 1] - x[..., 1]).abs() <= 1e-6 * (1 + x[..., 1].abs())).all()  # replaced at every step
    assert ((y[..., 3] - x[..., 3]).abs() <= 1e-6 * (1 + x[..., 3].abs())).all()
    assert torch.isfinite(y[0, :50, 4]).all() and torch.isnan(y[0, 50:, 4]).all()
    assert torch.isfinite(y[0, :60, 5]).all() and not torch.isfinite(y[0, 60:, 5]).any()
    assert torch.isfinite(y[..., 6:]).all()


def test_empty_windows_and_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(2, 6, 8, "f32", cuda_dev)
    c = [t.contiguous() for t in (x, f, z)]
    none = [t[:, :0] for t in c]
    last = torch.empty_like(h0)
    assert mb.gated_scan_fwd(*none, h0=h0, h_last=last).shape == (2, 0, 8) and torch.equal(last, h0)
    g = mb.gated_scan_bwd(none[0], none[1], none[0], torch.empty(2, 0, 8, device=cuda_dev), none[2], d_last=h0)
    assert torch.equal(g["d_h0"], h0)
    assert mb.gated_scan_fwd(c[0][:0], c[1][:0]).shape == (0, 6, 8)
    cs = torch.empty(mb.gated_scan_states(2, 6, 8), device=cuda_dev)
    for bad in (lambda: mb.gated_scan_fwd(c[0], c[1].half()), lambda: mb.gated_scan_fwd(c[0], c[1][:, :5]), lambda: mb.gated_scan_fwd(c[0].double(), c[1].double()),
                lambda: mb.gated_scan_fwd(c[0], c[1], h0=h0.half()), lambda: mb.gated_scan_fwd(c[0], c[1], h0=h0[:1]),
                lambda: mb.gated_scan_fwd(c[0], c[1], chunk_states=cs[:1]), lambda: mb.gated_scan_bwd(c[0], c[1], c[2][:1], cs)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: mb.gated_scan_fwd(c[0].transpose(1, 2).contiguous().transpose(1, 2), c[1]),
                lambda: mb.gated_scan_fwd(torch.cat([c[0], c[0]], 1)[:, :6], c[1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="row stride"):
        mb.gated_scan_fwd(c[0], c[1][:1, :1].expand(2, 6, 8))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mb.gated_scan_fwd(c[0].cpu(), c[1])


def test_step_refusals_and_strides(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(3, 1, 9, "bf16", cuda_dev, pad=2)
    x, f, z = x[:, 0], f[:, 0], z[:, 0]
    out = torch.empty_like(h0)
    want = mb.gated_scan_step(x.contiguous(), f.contiguous(), h0, z.contiguous(), h_last=out)
    assert torch.equal(mb.gated_scan_step(x, f, h0, z, h_last=out), want)
    for bad in (lambda: mb.gated_scan_step(x, f[:2], h0), lambda: mb.gated_scan_step(x, f.float(), h0), lambda: mb.gated_scan_step(x, f, h0.half()),
                lambda: mb.gated_scan_step(x, f, h0, h_last=h0[:2])):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(ValueError):
        mb.gated_scan_step(x, torch.zeros(9, 3, device=cuda_dev, dtype=x.dtype).t(), h0)
    with pytest.raises(RuntimeError, match="row stride"):
        mb.gated_scan_step(x, f[:1].expand(3, 9), h0)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,T,D", [(1, 1300, 40), (1, 700, 130), (2, 5000, 33)])
def test_any_workspace_gives_the_same_up_to_rounding(cuda_dev, dt, B, T, D):
    """None, too little for every segment, and more than enough."""
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, seed=9)
    hs, y, last = _plain(x, f, z, h0)
    tol, gz = _state_tol(x, f, h0), (z.double() * torch.sigmoid(z.double())).abs()
    need = mb.gated_scan_workspace_bytes(B, T, D)
    for size in (0, 8 * B * D, 8 * B * D * 3, need, need + 4096):
        h = h0.clone()
        got = mb.gated_scan_fwd(x, f, z, h0=h, h_last=h, workspace=torch.full((size,), 255, dtype=torch.uint8, device=cuda_dev))
        assert ((got.double() - y).abs() <= tol * gz + (HALF[dt] * 1.01 + 2.0 ** -20) * y.abs() + TINY[dt]).all()
        assert ((h.double() - last).abs() <= tol).all()
