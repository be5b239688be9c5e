"""Values at the edge of the types in linear attention: infinities and NaN, which may change no row before their own (nor, in the gradients of
k and v, behind it), other heads and sequences; large and small 16-bit values; slow and fast decays side by side.

The tolerances are those of the plain comparison (test_linear_attention_gpu.py), element by element."""
import math

import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]
# T, K, V, heads of v; decays
CASES = [(300, 128, 64, 2, "slow"), (300, 64, 128, 1, "slow"), (300, 128, 64, 2, "fast"), (129, 40, 24, 2, "fast"), (31, 16, 8, 1, "slow"),
         (5000, 64, 64, 1, "slow")]


def make(dev, dt, T, K, V, Hv, decays, B=2, H=2):
    import torch

    from retention_ref import DT
    g = torch.Generator(dev).manual_seed(T + K)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    decay = {"slow": -0.01, "fast": -0.8}[decays] * (1 + torch.arange(H, device=dev, dtype=torch.float32))
    return rn(B, T, H, K).to(DT[dt]), rn(B, T, H, K).to(DT[dt]), rn(B, T, Hv, V).to(DT[dt]), rn(B, T, H, V).to(DT[dt]), decay, rn(B, H, K, V)


def run(ops, q, k, v, decay, state, scale=None):
    import torch
    last = torch.empty_like(state)
    return ops.linear_attention_fwd(q, k, v, decay, scale=scale, state=state, state_out=last), last


def gradients(ops, q, k, v, do, decay, state, d_last=None, scale=None):
    d = ops.linear_attention_bwd(q, k, v, do, decay, scale=scale, state=state, d_state_out=d_last)
    return d["d_q"], d["d_k"], d["d_v"]


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_values_that_are_not_finite_go_forwards_alone(cuda_dev, dt, case, bad):
    import torch

    from mamba_rs_b200 import ops
    T, K, V, Hv, decays = case
    q, k, v, _, decay, state = make(cuda_dev, dt, T, K, V, Hv, decays)
    o, last = run(ops, q, k, v, decay, state)
    at, col = T // 2 - 1, V // 3
    for place in ("q", "k", "v", "state"):
        q2, k2, v2, s2 = (t.clone() for t in (q, k, v, state))
        {"q": q2[1, at, 1], "k": k2[1, at, 1], "v": v2[1, at, -1], "state": s2[1, 1].T}[place][col % K if place in "qk" else col] = bad
        o2, last2 = run(ops, q2, k2, v2, decay, s2)
        hit = torch.zeros_like(o, dtype=torch.bool)
        heads = slice(0, 2) if place == "v" and Hv == 1 else slice(1, 2)
        cols = slice(col, col + 1) if place in ("v", "state") else slice(None)
        rows = {"q": slice(at, at + 1), "state": slice(0, None)}.get(place, slice(at, None))
        hit[1, rows, heads, cols] = True
        # f32's general kernel and the tensor cores' sum other rows in the same order whatever is beside them; f16's copy of a state is scaled
        # by the largest magnitude that is finite, so it is compared to half a step of the sums it is part of
        if dt == "f16":
            assert torch.isfinite(o2[~hit]).all()
            assert ((o2 - o).float()[~hit].abs() <= 2.0 ** -9 * o.float().abs().max()).all()
        else:
            assert torch.equal(o2[~hit], o[~hit]), place
        if place == "q":
            assert not torch.isfinite(o2[hit]).any() and torch.equal(last2, last)
            continue
        # (a weight that has gone to 0 on the way makes NaN of an infinity, and nothing of it stays finite)
        near = hit.clone()
        near[:, at + 20:] = False
        assert not torch.isfinite(o2[near]).any(), place
        clean = torch.ones_like(last, dtype=torch.bool)
        if place == "k":
            clean[1, 1, col % K] = False
        else:
            clean[1, heads, :, cols] = False
        assert torch.isfinite(last2[clean]).all()
        assert torch.equal(last2[clean], last[clean])
        assert not torch.isfinite(last2[~clean]).any()


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients_of_rows_that_do_not_meet_them(cuda_dev, dt, case, bad):
    """A gradient that is not finite at one step leaves the later steps of d_k and d_v, and d_q of other steps, as they were."""
    import torch

    from mamba_rs_b200 import ops
    T, K, V, Hv, decays = case
    q, k, v, do, decay, state = make(cuda_dev, dt, T, K, V, Hv, decays)
    want = gradients(ops, q, k, v, do, decay, state)
    at = T // 2 + 1
    do2 = do.clone()
    do2[1, at, 1, V // 2] = bad
    got = gradients(ops, q, k, v, do2, decay, state)
    for i, (g, w) in enumerate(zip(got, want)):
        hit = torch.zeros_like(w, dtype=torch.bool)
        last = slice(-1, None)
        if i == 0:
            hit[1, at, last] = True
        elif i == 1:
            hit[1, :at + 1, last] = True
        else:
            hit[1, :at + 1, last, V // 2] = True
        assert torch.isfinite(g[~hit]).all(), i
        if dt == "f16":
            assert ((g - w).float()[~hit].abs() <= 2.0 ** -9 * w.float().abs().max()).all()
        else:
            assert torch.equal(g[~hit], w[~hit]), i
        near = hit.clone()
        near[:, :max(at - 20, 0)] = False
        assert not torch.isfinite(g[near]).any(), i


@pytest.mark.parametrize("dt", DTS)
def test_padding_of_any_content(cuda_dev, dt):
    """Rows behind a sequence's end may hold anything: its own rows are those of the sequence alone."""
    import torch

    from mamba_rs_b200 import ops
    q, k, v, _, decay, _ = make(cuda_dev, dt, 400, 128, 64, 2, "slow")
    for n in (1, 37, 130, 256, 391):
        q2, k2, v2 = (t.clone() for t in (q, k, v))
        for t in (q2, k2, v2):
            t[:, n:] = math.nan
        o = ops.linear_attention_fwd(q, k, v, decay)
        o2 = ops.linear_attention_fwd(q2, k2, v2, decay)
        if dt == "f16":  # (rows' and tiles' scales are powers of two from the rows of the same chunk: digits, not values)
            assert ((o2 - o).float()[:, :n].abs() <= 2.0 ** -9 * o.float().abs().max()).all()
        else:
            assert torch.equal(o2[:, :n], o[:, :n]), n


@pytest.mark.parametrize("dt,size", [("f16", 2.0 ** 7), ("f16", 2.0 ** -7), ("f16", 2.0 ** -12), ("bf16", 2.0 ** 40), ("bf16", 2.0 ** -40),
                                     ("f32", 2.0 ** 40), ("f32", 2.0 ** -30)])
@pytest.mark.parametrize("heads", [(4, 4, 4), (2, 1, 4)])
def test_large_and_small_values(cuda_dev, dt, size, heads):
    """Scores of K size^2 and states beside them: f16 keeps their digits by powers of two; a scale brings the result back into the type."""
    import torch

    from retention_ref import DT, attention, attention_grads
    from test_linear_attention_gpu import close, inputs, state_close

    from mamba_rs_b200 import ops
    B, T, H, K, V = 1, 290, 4, 64, 64
    q, k, v, do, decay, state, d_last = inputs(cuda_dev, "f32", B, T, H, K, V, *heads)
    q, k, v, do = ((t * size).to(DT[dt]) for t in (q, k, v, do))
    scale = 2.0 ** round(-2 * math.log2(size)) / 32
    state = state * size ** 2
    args = (q, k, v, decay)
    want, last = attention(*args, scale, state)
    mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, scale, state.abs())
    o, s = run(ops, *args, state, scale)
    assert torch.isfinite(o).all()
    close(o, want, mags, dt, K + T, extra=2.0)
    state_close(s, last, last_mags, T)
    d_last = d_last * size ** 2 * scale
    grads = gradients(ops, q, k, v, do, decay, state, d_last, scale)
    wants = attention_grads(*args[:3], do, decay, scale, state, d_last)
    gmags = attention_grads(*(t.abs() for t in args[:3]), do.abs(), decay, scale, state.abs(), d_last.abs())
    for g, w, m, n in zip(grads, wants[:3], gmags[:3], (V, V, K)):
        close(g, w, m, dt, n + T + H, extra=2.0)


@pytest.mark.parametrize("dt", DTS)
def test_decays_of_every_speed_side_by_side(cuda_dev, dt):
    """From none to total, on both sides of where the tensor cores' kernel changes its way (-40 / 127), and a little growth."""
    import torch

    from retention_ref import attention, attention_grads
    from test_linear_attention_gpu import close, inputs, state_close

    from mamba_rs_b200 import ops
    decay = torch.tensor([0.0, -1e-6, -0.3149, -0.3150, -1.5, -30.0, -math.inf, 1e-3], device=cuda_dev)
    H, B, T, K, V = decay.numel(), 1, 300, 64, 64
    q, k, v, do, _, state, d_last = inputs(cuda_dev, dt, B, T, H, K, V)
    o, s = run(ops, q, k, v, decay, state)
    want, last = attention(q, k, v, decay, K ** -0.5, state)
    mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, K ** -0.5, state.abs())
    close(o, want, mags, dt, K + T, extra=2.0)
    state_close(s, last, last_mags, T)
    grads = gradients(ops, q, k, v, do, decay, state, d_last)
    wants = attention_grads(q, k, v, do, decay, K ** -0.5, state, d_last)
    gmags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, K ** -0.5, state.abs(), d_last.abs())
    for g, w, m in zip(grads, wants[:3], gmags[:3]):
        close(g, w, m, dt, 64 + T, extra=2.0)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("T,K,V,H", [(20000, 64, 64, 3), (6000, 128, 64, 40), (6000, 40, 72, 40)])
def test_states_of_long_texts_keep_their_digits(cuda_dev, dt, T, K, V, H):
    """A state that hardly decays is a sum of thousands of tokens.  The tensor cores' sums of a chunk's 24 partial products are cut off, not
    rounded: up to 24 2^-23 of a chunk's sum, always towards zero, so up to as much of the state; its terms are kept to 2^-22; the chunks'
    roundings, T / 128 of 2^-24 with random signs (f32: T / 32), come on top.  Nothing may grow with T faster."""
    import torch
    from retention_ref import DT, fro

    from mamba_rs_b200 import ops
    g = torch.Generator(cuda_dev).manual_seed(T + K)
    rn = lambda *s: torch.randn(*s, device=cuda_dev, generator=g)  # noqa: E731
    # (values with a mean, so that the state grows)
    q, k = ((rn(1, T, H, K) + 0.5).to(DT[dt]) for _ in range(2))
    v, do = ((rn(1, T, H, V) + 0.5).to(DT[dt]) for _ in range(2))
    decay = -1e-4 * torch.arange(H, device=cuda_dev, dtype=torch.float32) / H
    state, d_last = 10 * rn(1, H, K, V), 10 * rn(1, H, K, V)
    tol = 24 * 2.0 ** -23 + 2.0 ** -22 + 4 * 2.0 ** -24 * math.sqrt(T / 32)
    t = torch.arange(T, device=cuda_dev, dtype=torch.float64)[:, None]
    whole = torch.exp(decay.double() * T)[None, :, None, None]
    w = torch.exp(decay.double() * (T - 1 - t))
    want = torch.stack([(k[0, :, h].double() * w[:, h, None]).T @ v[0, :, h].double() for h in range(H)])[None] + whole * state.double()
    _, last = run(ops, q, k, v, decay, state)
    assert fro(last, want) <= tol, fro(last, want) / tol
    scale = K ** -0.5
    w = torch.exp(decay.double() * (t + 1)) * scale
    want = torch.stack([(q[0, :, h].double() * w[:, h, None]).T @ do[0, :, h].double() for h in range(H)])[None] + whole * d_last.double()
    got = ops.linear_attention_bwd(q, k, v, do, decay, state=state, d_state_out=d_last)["d_state"]
    assert fro(got, want) <= tol, fro(got, want) / tol
