"""Products of scores and values that are small for 32 bits, at decays on both sides of every change of ways in the tensor cores' kernel: bf16
values have the range of f32, so nothing of them may be lost on the way that the formula's own products hold.

Scores of 64 columns and the values beside them are some 2^-120, 2^6 above the smallest normal number of f32; a chunk's fastest folded weight is
2^-8 and leaves a product 21 of 24 bits below it, which is 2^-13 of the two roundings of 2^-8 that the tolerances of test_linear_attention_gpu.py count."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("decay", [-0.01, -0.03, -0.0436, -0.0437, -0.1, -0.2, -0.3, -0.3149, -0.3150, -0.5])
def test_small_products(cuda_dev, decay):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import close, inputs, state_close
    T, H, K, V = 290, 2, 64, 64
    q, k, v, do, _, state, d_last = inputs(cuda_dev, "f32", 1, T, H, K, V, seed=31)
    q, k, v, do = ((t * 2.0 ** -41).bfloat16() for t in (q, k, v, do))
    decays = torch.full((H,), decay, device=cuda_dev)
    scale, state, d_last = 2.0 ** 80, state * 2.0 ** -82, d_last * 2.0 ** -2
    for s0, d_s in ((state, d_last), (None, None)):
        want, last = attention(q, k, v, decays, scale, s0)
        mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decays, scale, None if s0 is None else s0.abs())
        for out in (None, torch.empty_like(state)):
            o = mb.linear_attention_fwd(q, k, v, decays, scale=scale, state=s0, state_out=out)
            close(o, want, mags, "bf16", K + T, 2.0)
            if out is not None:
                state_close(out, last, last_mags, T)
        got = mb.linear_attention_bwd(q, k, v, do, decays, scale=scale, state=s0, d_state_out=d_s)
        wants = attention_grads(q, k, v, do, decays, scale, s0, d_s)
        gmags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decays, scale, None if s0 is None else s0.abs(), None if d_s is None else d_s.abs())
        for name, w, m in zip(("d_q", "d_k", "d_v"), wants, gmags):
            close(got[name], w, m, "bf16", K + V + T, 2.0)
