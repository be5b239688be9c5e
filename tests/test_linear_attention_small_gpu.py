"""Linear attention of small values: 16-bit gradients without a loss scale, small keys and values, small products.

Tolerances are those of test_linear_attention_gpu.py: states are sums in 32 bits of products kept to 2^-22 whatever the type and size."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("heads", [(4, 4, 4), (4, 2, 2)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_small_gradients_and_values(cuda_dev, dt, heads, size):
    """Gradients of o, then values, of that size, with a scale below 1 (which f16 keeps on the tensor cores)."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import close, inputs, state_close
    T, H, K, V = 300, 4, 128, 64
    q, k, v, do, decay, state, d_last = inputs(cuda_dev, dt, 1, T, H, K, V, *heads, seed=21)
    scale = K ** -0.5
    small = (do.float() * size).to(do.dtype)
    for s0, d_s in ((state, d_last * size * scale), (state, None)):
        wants = attention_grads(q, k, v, small, decay, scale, s0, d_s)
        mags = attention_grads(q.abs(), k.abs(), v.abs(), small.abs(), decay, scale, s0.abs(), None if d_s is None else d_s.abs())
        got = mb.linear_attention_bwd(q, k, v, small, decay, scale=scale, state=s0, d_state_out=d_s)
        for name, w, m in zip(("d_q", "d_k", "d_v"), wants, mags):
            err, tiny = (got[name].double() - w).abs(), 2.0 ** -25 if dt == "f16" else 0.0
            u = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dt]
            assert (err <= (2 * u + (K + V + T + H + 16) * 2.0 ** -24) * m + (u + 2.0 ** -24) * 1.01 * w.abs() + tiny).all(), name
        state_close(got["d_state"], wants[3], mags[3], T)
    low = (v.float() * size).to(v.dtype)
    for s0 in (state * size, None):
        want, last = attention(q, k, low, decay, scale, s0)
        mags, last_mags = attention(q.abs(), k.abs(), low.abs(), decay, scale, None if s0 is None else s0.abs())
        s = torch.empty_like(state)
        o = mb.linear_attention_fwd(q, k, low, decay, scale=scale, state=s0, state_out=s)
        if size > 1e-4 or dt != "f16":  # (else o itself is among the numbers that f16 has few digits for)
            close(o, want, mags, dt, K + T, 0.0 if dt == "f32" else 2.0)
        state_close(s, last, last_mags, T)


@pytest.mark.parametrize("scale", [2.0 ** -20, 2.0 ** -60])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_a_small_scale(cuda_dev, dt, scale):
    """d_state is 32 bits: a scale that takes it far below what 16 bits can hold costs it no digits."""
    import mamba_rs_b200 as mb
    from retention_ref import attention_grads
    from test_linear_attention_gpu import inputs, state_close
    T, H, K, V = 290, 3, 64, 64
    q, k, v, do, decay, state, d_last = inputs(cuda_dev, dt, 1, T, H, K, V, seed=22)
    d_s = d_last * scale
    want = attention_grads(q, k, v, do, decay, scale, state, d_s)[3]
    mags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, scale, state.abs(), d_s.abs())[3]
    state_close(mb.linear_attention_bwd(q, k, v, do, decay, scale=scale, state=state, d_state_out=d_s)["d_state"], want, mags, T)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_state_gradients_of_decays_of_every_speed(cuda_dev, dt):
    import math

    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention_grads
    from test_linear_attention_gpu import inputs, state_close
    decay = torch.tensor([0.0, -1e-6, -0.04, -0.05, -0.3149, -1.5, -30.0, -math.inf, 1e-3], device=cuda_dev)
    H, T, K, V = decay.numel(), 300, 64, 64
    q, k, v, do, _, state, d_last = inputs(cuda_dev, dt, 1, T, H, K, V, seed=23)
    want = attention_grads(q, k, v, do, decay, K ** -0.5, state, d_last)[3]
    mags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, K ** -0.5, state.abs(), d_last.abs())[3]
    state_close(mb.linear_attention_bwd(q, k, v, do, decay, state=state, d_state_out=d_last)["d_state"], want, mags, T)
