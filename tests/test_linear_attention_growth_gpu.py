"""Linear attention with decays above 0: a state that grows as the formula says.

Tolerances are those of test_linear_attention_gpu.py, and l^n on top: in 32 bits its exponent n log2 l passes three roundings of 2^-24 (log2 e, the
product with it, the product with n <= 127), which move l^n by 3 2^-24 n |log l| of itself, and with growth the oldest tokens, whose n is
largest, weigh most."""
import math

import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]
LIMIT = {"f32": 1e38, "bf16": 1e38, "f16": 65504.0}


def compare(got, want, mags, dt, n, decay):
    """Element by element and in the norm, where the formula's value is in the type by more than it may be off (an error that the bound
    allows may take a value that close to the largest number to infinity)."""
    import torch
    from retention_ref import HALF, TINY
    l = 3 * 2.0 ** -24 * 127 * decay
    u = HALF[dt] if dt != "f32" else 0.0
    bound = (2 * u + l + (n + 16) * 2.0 ** -24) * mags + (u + 2.0 ** -24) * want.abs() * 1.01 + TINY[dt]
    inside = want.abs() + bound < LIMIT[dt]
    assert torch.isfinite(got[inside]).all()
    err = (got.double() - want).abs()
    assert (err[inside] <= bound[inside]).all(), float((err / bound)[inside].max())
    # the norm, of rows whose terms' magnitudes leave room for all of them (a choice by the results themselves would take small ones beside the
    # errors of large ones; where most of a result is below the type's smallest number, its norm says nothing)
    tol = 2 * u + l + 2.0 ** -24 * 2 * (16 + math.sqrt(n))
    rows = mags.amax(-1) < LIMIT[dt] / 2
    assert float(err[rows].norm()) <= tol * float(want[rows].norm()) + TINY[dt] * math.sqrt(err.numel())
    return float(inside.double().mean())


def compare_state(got, want, mags, T, decay):
    l = 3 * 2.0 ** -24 * 127 * decay
    err = (got.double() - want).abs()
    bound = ((T + 16) * 2.0 ** -24 + 2.0 ** -22 + l) * mags
    assert (err <= bound).all(), float((err / bound).max())
    assert float(err.norm()) <= (2.0 ** -24 * 2 * (16 + math.sqrt(T)) + l) * float(want.norm())


@pytest.mark.parametrize("decay", [0.02, 0.087, 0.1, 0.2, 0.5])
@pytest.mark.parametrize("T,K,V", [(128, 64, 64), (140, 128, 64), (300, 40, 72)])
@pytest.mark.parametrize("dt", DTS)
def test_growth(cuda_dev, dt, T, K, V, decay):
    """Forward and backward, with the scale that keeps the last results in the type and with one that keeps the first."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import inputs
    B, H = 1, 2
    T = min(T, int(80 / decay))
    q, k, v, do, _, state, d_last = inputs(cuda_dev, dt, B, T, H, K, V, seed=11)
    g = torch.full((H,), decay, device=cuda_dev)
    for scale in (K ** -0.5, K ** -0.5 * math.exp(-decay * T)):
        args, mag = (q, k, v), [t.abs() for t in (q, k, v)]
        want, last = attention(*args, g, scale, state)
        mags, last_mags = attention(*mag, g, scale, state.abs())
        s = torch.empty_like(state)
        o = mb.linear_attention_fwd(*args, g, scale=scale, state=state, state_out=s)
        compare(o, want, mags, dt, K + T, decay)
        compare_state(s, last, last_mags, T, decay)
        compare(mb.linear_attention_fwd(*args, g, scale=scale, state=state), want, mags, dt, K + T, decay)
        wants = attention_grads(*args, do, g, scale, state, d_last * scale)
        gmags = attention_grads(*mag, do.abs(), g, scale, state.abs(), d_last.abs() * scale)
        got = mb.linear_attention_bwd(*args, do, g, scale=scale, state=state, d_state_out=d_last * scale)
        for name, w, m in zip(("d_q", "d_k", "d_v"), wants, gmags):
            compare(got[name], w, m, dt, K + V + T, decay)
        compare_state(got["d_state"], wants[3], gmags[3], T, decay)
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("decay", [0.1, 0.5])
@pytest.mark.parametrize("dt", DTS)
def test_growth_behind_nothing(cuda_dev, dt, decay):
    """Rows of zeros (a padded start) weigh most and add nothing: what follows keeps its digits."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import inputs
    T, K, V, H = 150, 64, 64, 2
    q, k, v, do, _, _, _ = inputs(cuda_dev, dt, 1, T, H, K, V, seed=12)
    k[:, :110] = 0
    do[:, 40:] = 0
    g = torch.full((H,), decay, device=cuda_dev)
    scale = K ** -0.5 * math.exp(-decay * 40)
    want, last = attention(q, k, v, g, scale)
    mags, last_mags = attention(q.abs(), k.abs(), v.abs(), g, scale)
    s = torch.empty_like(last, dtype=torch.float32)
    o = mb.linear_attention_fwd(q, k, v, g, scale=scale, state_out=s)
    assert compare(o, want, mags, dt, K + T, decay) == 1.0
    compare_state(s, last, last_mags, T, decay)
    wants = attention_grads(q, k, v, do, g, scale)
    gmags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), g, scale)
    d_state = torch.empty_like(s)
    got = mb.linear_attention_bwd(q, k, v, do, g, scale=scale, d_state=d_state)
    for name, w, m in zip(("d_q", "d_k", "d_v"), wants, gmags):
        assert compare(got[name], w, m, dt, K + V + T, decay) == 1.0
    compare_state(d_state, wants[3], gmags[3], T, decay)


@pytest.mark.parametrize("dt", DTS)
def test_growth_over_a_text_in_segments(cuda_dev, dt):
    """A long text of few heads, which the kernels cut; growing and decaying heads beside each other, odd widths among them."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import inputs
    T, H = 1501, 3
    for K, V in ((64, 64), (40, 72)):
        q, k, v, do, _, state, d_last = inputs(cuda_dev, dt, 1, T, H, K, V, 3, 1, 3, seed=13)
        g = torch.tensor([0.05, -0.02, 0.001], device=cuda_dev)
        scale = K ** -0.5 * math.exp(-0.05 * T)
        want, last = attention(q, k, v, g, scale, state)
        mags, last_mags = attention(q.abs(), k.abs(), v.abs(), g, scale, state.abs())
        s = torch.empty_like(state)
        o = mb.linear_attention_fwd(q, k, v, g, scale=scale, state=state, state_out=s)
        wants = attention_grads(q, k, v, do, g, scale, state, d_last * scale)
        gmags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), g, scale, state.abs(), d_last.abs() * scale)
        got = mb.linear_attention_bwd(q, k, v, do, g, scale=scale, state=state, d_state_out=d_last * scale)
        for h in range(H):
            compare(o[:, :, h], want[:, :, h], mags[:, :, h], dt, K + T, 0.05)
            compare_state(s[:, h], last[:, h], last_mags[:, h], T, 0.05)
            compare_state(got["d_state"][:, h], wants[3][:, h], gmags[3][:, h], T, 0.05)
        for name, w, m in zip(("d_q", "d_k", "d_v"), wants, gmags):
            compare(got[name], w, m, dt, K + V + T + H, 0.05)
    mb.ffi.default_handle(0).check_status()
