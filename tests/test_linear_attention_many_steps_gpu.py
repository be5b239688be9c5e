"""A text taken token by token, thousands of them: the state of slow decays against the recurrence in 64 bits and against the whole text at once.

Tolerance: a step rounds twice, each by at most 2^-24 of the state (of what is in it and comes to it), with signs that random values make
random, and older roundings decay with the state: 2^-24 sqrt(2 T) at most.  Twice that, and as much for the whole text."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry", ["step", "fwd"])
@pytest.mark.parametrize("dt,V", [("f32", 8), ("bf16", 8), ("f16", 7)])
def test_many_steps(cuda_dev, dt, V, entry):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import DT, attention, fro
    T, B, K = 6000, 1, 16
    decay = torch.tensor([math.log1p(-2.0 ** -n) for n in (5, 10, 11, 12, 13)] + [-1e-4, -1e-6, 0.0, 1e-4, -0.6, -0.7, -3.0, -math.inf],
                         device=cuda_dev, dtype=torch.float64).float()
    H = decay.numel()
    g = torch.Generator(cuda_dev).manual_seed(41)
    # (values with a mean, so that states of slow decays are large beside what a token adds)
    q, k, v = ((torch.randn(B, T, H, w, device=cuda_dev, generator=g) + 0.5).to(DT[dt]) for w in (K, K, V))
    start = 100 * torch.randn(B, H, K, V, device=cuda_dev, generator=g)
    scale = K ** -0.5
    _, want = attention(q, k, v, decay, scale, start)
    s = start.clone()
    for t in range(T):
        if entry == "step":
            mb.linear_attention_step(q[:, t], k[:, t], v[:, t], decay, s)
        else:
            mb.linear_attention_fwd(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], decay, state=s, state_out=s)
    whole = torch.empty_like(s)
    mb.linear_attention_fwd(q, k, v, decay, state=start, state_out=whole)
    tol = 2 * 2.0 ** -24 * math.sqrt(2 * T)
    for h in range(H):
        assert fro(s[:, h], want[:, h]) <= tol, (float(decay[h]), fro(s[:, h], want[:, h]) / tol)
        assert fro(s[:, h], whole[:, h].double()) <= 2 * tol, float(decay[h])
