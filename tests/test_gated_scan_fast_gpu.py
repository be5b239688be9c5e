"""The gated linear recurrence where channels forget fast: strongly negative forget gates, large states that are gone a few steps
later.  Against the recurrence in 64 bits with both u = sigmoid(-f) and p = sigmoid(f) from their own exponentials.

Tolerances, step by step with eps = 2^-24.  s, the smaller of u and p, has a relative error of at most e = 2^-21 (2 + |f|): its
exponential's argument is rounded twice at |f|, and the exponential, a sum, a reciprocal and a product follow.  The larger one is
1 - s: relative error e s / (1 - s), and a rounding.  With H the same recurrence of magnitudes, H' = p H + u |x|, an error F of a state
obeys F' = p (F + H (d_p + 4 eps)) + u |x| (d_u + 4 eps) + 2 eps H'; the roundings counted for a step cover the joins of spans, whose
products and sums have no more of them than the steps that they stand for.  The gradient g obeys the same law from the end, with
dy SiLU(z) in the place of u x (relative error 2^-19), and d_f = g (h - x) u p has the relative errors of s twice, the error of g, and
that of h - x.  16-bit results add half an ulp."""
import math

import pytest

pytestmark = pytest.mark.gpu
DT = ["f32", "bf16", "f16"]
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}
EPS = 2.0 ** -24
SHAPES = [(1, 1, 9), (2, 3, 33), (2, 8, 40), (2, 20, 64), (2, 130, 64), (3, 90, 41), (1, 1300, 40), (2, 700, 33)]


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _inputs(B, T, D, dt, dev, lo, hi, gate, large, seed=0):
    """Gates between lo and hi, some channels at the ends; a state of `large`."""
    import torch
    g = torch.Generator(dev).manual_seed(seed + T * D + B)
    x, z = (torch.randn(B, T, D, device=dev, generator=g).to(_dt(dt)) for _ in range(2))
    f = lo + (hi - lo) * torch.rand(B, T, D, device=dev, generator=g)
    f[..., 0], f[..., 1], f[..., 2], f[..., 3], f[..., 4], f[..., 5] = 200.0, -200.0, math.inf, -math.inf, -4.0, -17.0
    f[..., 6], f[..., 7] = 4.0, -12.0
    h0 = large * torch.randn(B, D, device=dev, generator=g)
    return x, f.to(_dt(dt)), z if gate else None, h0


def _gates(f):
    """u, p and the bounds of their relative errors."""
    import torch
    f = f.double()
    u, p = 1.0 / (1.0 + torch.exp(f)), 1.0 / (1.0 + torch.exp(-f))
    e = 2.0 ** -21 * (2 + f.abs().clamp(max=200.0))
    s = torch.minimum(u, p)
    large = e * s / (1 - s)
    slow = u < p
    return u, p, torch.where(slow, e, large), torch.where(slow, large, e)


def _states(x, f, h0):
    """The state before every step and behind the last, and bounds of their errors: [B, T + 1, D] each."""
    import torch
    u, p, du, dp = _gates(f)
    x = x.double()
    h, H, F = h0.double(), h0.double().abs(), torch.zeros_like(h0).double()
    hs, Fs = [h], [F]
    for t in range(x.shape[1]):
        ux = u[:, t] * x[:, t].abs()
        F = p[:, t] * (F + H * (dp[:, t] + 4 * EPS)) + ux * (du[:, t] + 4 * EPS)
        h, H = p[:, t] * h + u[:, t] * x[:, t], p[:, t] * H + ux
        F = F + 2 * EPS * H
        hs.append(h)
        Fs.append(F)
    return torch.stack(hs, 1), torch.stack(Fs, 1)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("lo,hi,large", [(-24.0, 2.0, 1000.0), (-5.0, 0.0, 1e6), (-2.0, 3.0, 1000.0)])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_a_large_state_is_forgotten(cuda_dev, dt, gate, lo, hi, large, B, T, D):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, lo, hi, gate, large)
    hs, F = _states(x, f, h0)
    h_last, cs = torch.empty_like(h0), torch.empty(mb.gated_scan_states(B, T, D), device=cuda_dev)
    y = mb.gated_scan_fwd(x, f, z, h0=h0, h_last=h_last, chunk_states=cs)
    assert ((h_last.double() - hs[:, -1]).abs() <= F[:, -1] + EPS * hs[:, -1].abs() + 1e-37).all()
    assert ((cs.double() - hs[:, :T:64]).abs() <= F[:, :T:64] + EPS * hs[:, :T:64].abs()).all()
    silu = 1.0 if z is None else z.double() * torch.sigmoid(z.double())
    want, size = hs[:, 1:] * silu, silu.abs() if gate else 1.0
    fits = want.abs() < 6e4 if dt == "f16" else torch.ones_like(want, dtype=torch.bool)
    bad = (y.double() - want).abs() > F[:, 1:] * size + (HALF[dt] * 1.01 + 2.0 ** -20) * want.abs() + TINY[dt]
    assert not (bad & fits).any()
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DT)
def test_a_large_state_is_forgotten_step_by_step(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h = _inputs(3, 12, 40, dt, cuda_dev, -24.0, 2.0, True, 1000.0)
    hs, F = _states(x, f, h)
    for t in range(12):
        y = mb.gated_scan_step(x[:, t], f[:, t], h, z[:, t])
        assert ((h.double() - hs[:, t + 1]).abs() <= F[:, t + 1] + EPS * hs[:, t + 1].abs() + 1e-37).all()
        zt = z[:, t].double()
        want, size = hs[:, t + 1] * zt * torch.sigmoid(zt), (zt * torch.sigmoid(zt)).abs()
        assert ((y.double() - want).abs() <= F[:, t + 1] * size + (HALF[dt] * 1.01 + 2.0 ** -20) * want.abs() + TINY[dt]).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("lo,hi,large", [(-24.0, 2.0, 1.0), (-20.0, -8.0, 1.0), (-5.0, 0.0, 1.0), (-3.0, 3.0, 100.0)])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_gradients_of_fast_channels(cuda_dev, dt, gate, lo, hi, large, B, T, D):
    """d_f has the factor 1 - u, which is far below 1's last place where a gate is strongly negative."""
    import torch

    import mamba_rs_b200 as mb
    x, f, z, h0 = _inputs(B, T, D, dt, cuda_dev, lo, hi, gate, large, seed=1)
    g_ = torch.Generator(cuda_dev).manual_seed(T)
    dy, d_last = torch.randn(B, T, D, device=cuda_dev, generator=g_).to(_dt(dt)), large * torch.randn(B, D, device=cuda_dev, generator=g_)
    cs = torch.empty(mb.gated_scan_states(B, T, D), device=cuda_dev)
    mb.gated_scan_fwd(x, f, z, h0=h0, chunk_states=cs)
    hs, F = _states(x, f, h0)
    u, p, du, dp = _gates(f)
    e, want, tol = dy.double(), {}, {}
    if gate:
        q = torch.sigmoid(z.double())
        want["d_z"] = e * hs[:, 1:] * (q + z.double() * q * (1 - q))
        tol["d_z"] = e.abs() * (1.2 * F[:, 1:] + 2.0 ** -19 * hs[:, 1:].abs())
        e = e * z.double() * q
    g = d_last.double()
    m, E = g.abs(), torch.zeros_like(g)
    dx, df, bx, bf = (torch.empty_like(e) for _ in range(4))
    for t in range(T - 1, -1, -1):
        g, m = g + e[:, t], m + e[:, t].abs()
        E = E + 2.0 ** -19 * e[:, t].abs() + 2 * EPS * m
        span, up = hs[:, t] - x[:, t].double(), u[:, t] * p[:, t]
        dx[:, t], df[:, t] = g * u[:, t], g * span * up
        bx[:, t] = u[:, t] * (E + m * (du[:, t] + 4 * EPS))
        bf[:, t] = up * (span.abs() * (E + m * (du[:, t] + dp[:, t] + 6 * EPS)) + m * (F[:, t] + EPS * (hs[:, t].abs() + x[:, t].double().abs())))
        E = p[:, t] * (E + m * (dp[:, t] + 4 * EPS))
        g, m = p[:, t] * g, p[:, t] * m
    want.update(d_x=dx, d_f=df, d_h0=g)
    tol.update(d_x=bx, d_f=bf, d_h0=E + EPS * g.abs())
    got = mb.gated_scan_bwd(x, f, dy, cs, z, d_last=d_last)
    assert set(got) == set(want)
    for k, v in got.items():
        half = (HALF[dt] if k != "d_h0" else EPS) * 1.01
        tiny = TINY[dt] if k != "d_h0" else 1e-37
        assert ((v.double() - want[k]).abs() <= tol[k] + half * want[k].abs() + tiny).all(), k
    mb.ffi.default_handle(0).check_status()


def test_channels_that_forget_slowly_do_not_drift(cuda_dev):
    """Memories of 3000 to a million steps: each step keeps 1 - u, which rounded the same way at every step would move the state by
    2^-25 a step.  Rounded once in 16 steps (three roundings) the bound is 3 T / 16 eps; u's own relative error moves it by 2 e."""
    import torch

    import mamba_rs_b200 as mb
    T, D = 20000, 96
    g = torch.Generator(cuda_dev).manual_seed(2)
    f = (8.0 + 6.0 * torch.rand(D, device=cuda_dev, generator=g)).expand(1, T, D).contiguous()
    x, h0 = torch.ones(1, T, D, device=cuda_dev), 1.0 + torch.rand(1, D, device=cuda_dev, generator=g)
    u, p, _, _ = _gates(f[0, 0])
    want = 1.0 + (h0.double() - 1.0) * p ** torch.arange(1, T + 1, device=cuda_dev, dtype=torch.float64)[:, None]
    tol = 2.0 * (3 * T / 16 * EPS + 2 * 2.0 ** -21 * 16)  # (states of up to 2)
    for size in (0, mb.gated_scan_workspace_bytes(1, T, D)):
        h_last = torch.empty_like(h0)
        y = mb.gated_scan_fwd(x, f, h0=h0, h_last=h_last, workspace=torch.empty(size, dtype=torch.uint8, device=cuda_dev))
        assert ((y[0].double() - want).abs() <= tol).all() and ((h_last[0].double() - want[-1]).abs() <= tol).all()
    h = h0.clone()
    for t in range(4000):
        mb.gated_scan_step(x[:, t], f[:, t], h)
    # (each step rounds the state once, to the nearest, and its change of at most 2^-11 once more)
    assert ((h[0].double() - want[3999]).abs() <= 2.0 * (4000 * EPS * 0.5 + 2 * 2.0 ** -21 * 16)).all()
