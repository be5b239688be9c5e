"""Linear attention with a decay for each head, forward, backward and step, against the recurrence in 64 bits, token by token.

Tolerances.  o is a sum of terms l^{t-s} q_a k_a v; A is the sum of their magnitudes (the reference run on magnitudes).  In 32 bits every
term passes at most K + T + 16 roundings of 2^-24 (products of a dot product, sums over tokens, powers of l to 2 ulp and an exponent's
rounding, which moves l^n by |n log l| l^n 2^-24 <= 2^-25), so |error| <= (K + T + 16) 2^-24 A.  16-bit kernels round the scores
and the copy of the state that is read, each by at most half a step: 2 HALF A more.  The result's own rounding adds HALF |o|.  Those
bounds hold for every element; errors of that many terms have random signs, so the norm of all of them is far smaller: half a step is
1 / sqrt(3) of itself in the mean square, three such roundings (scores, state copy, result) make HALF of the result's norm, and 2^-24
sqrt(K + T) times a few in 32 bits.  Twice that is asked for.  States are sums in 32 bits of products kept to 2^-22 whatever the type.
The backward's results are the same sums of other operands; gradients of shared heads are sums of up to H / Hx of them in 32 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]


def norm_tol(dt, n):
    """For the norm of a result's errors; n: terms of a sum."""
    from retention_ref import HALF
    return 2 * (HALF[dt] if dt != "f32" else 0.0) + 2.0 ** -24 * 2 * (16 + math.sqrt(n))


def close(got, want, mags, dt, n, extra=0.0):
    from retention_ref import HALF, TINY, fro
    u = HALF[dt]
    bound = (extra * u + (n + 16) * 2.0 ** -24) * mags + u * want.abs() * 1.01 + TINY[dt]
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert fro(got, want) <= norm_tol(dt, n), (fro(got, want), norm_tol(dt, n))


def state_close(got, want, mags, T):
    from retention_ref import fro
    assert ((got.double() - want).abs() <= ((T + 16) * 2.0 ** -24 + 2.0 ** -22) * mags + 1e-37).all()
    assert fro(got, want) <= 2.0 ** -24 * 2 * (16 + math.sqrt(T))


def inputs(dev, dt, B, T, H, K, V, Hq=None, Hk=None, Hv=None, seed=0, decays="mixed", pad=0):
    """q, k, v as columns of one projection (pad: columns between them), do, decay, states."""
    import torch

    from retention_ref import DT
    g = torch.Generator(dev).manual_seed(seed + 7 * T + K)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    widths = [(Hq or H, K), (Hk or H, K), (Hv or H, V)]
    proj = rn(B, T, sum(h * w + pad for h, w in widths)).to(DT[dt])
    q, at = [], 0
    for h, w in widths:
        q.append(proj[..., at:at + h * w].unflatten(-1, (h, w)))
        at += h * w + pad
    q, k, v = q
    decay = {"mixed": -torch.exp2(-9.0 * torch.rand(H, device=dev, generator=g)), "none": torch.zeros(H, device=dev),
             "fast": -20.0 * torch.rand(H, device=dev, generator=g)}[decays]
    return q, k, v, rn(B, T, H, V).to(DT[dt]), decay, rn(B, H, K, V), rn(B, H, K, V)


# B, T, H, K, V and, where heads are shared, Hq, Hk, Hv
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 3, 24, 40), (1, 2, 2, 64, 64), (2, 31, 2, 16, 8), (1, 33, 3, 5, 7), (2, 127, 2, 128, 64), (1, 128, 2, 64, 128),
          (2, 129, 4, 40, 56, 2, 2, 4), (1, 300, 4, 128, 128, 4, 1, 1), (1, 257, 2, 160, 96), (1, 130, 1, 256, 33), (3, 200, 6, 72, 64, 3, 2, 6),
          (1, 1500, 2, 64, 64), (1, 2100, 1, 31, 17), (2, 640, 8, 128, 64, 1, 1, 8)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(cuda_dev, dt, shape):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention
    q, k, v, _, decay, s0, _ = inputs(cuda_dev, dt, *shape)
    T, K = q.shape[1], q.shape[3]
    scale = K ** -0.5
    for state in (None, s0):
        want, last = attention(q, k, v, decay, scale, state)
        mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, scale, None if state is None else state.abs())
        out = torch.empty_like(s0)
        o = mb.linear_attention_fwd(q, k, v, decay, state=state, state_out=out)
        close(o, want, mags, dt, K + T, 0.0 if dt == "f32" else 2.0)
        state_close(out, last, last_mags, T)
        close(mb.linear_attention_fwd(q, k, v, decay, state=state), want, mags, dt, K + T, 0.0 if dt == "f32" else 2.0)
    # the same bits again, and in place
    s = s0.clone()
    assert torch.equal(mb.linear_attention_fwd(q, k, v, decay, state=s, state_out=s), o) and torch.equal(s, out)
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(cuda_dev, dt, shape):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention_grads
    q, k, v, do, decay, s0, d_last = inputs(cuda_dev, dt, *shape, seed=1)
    T, K, V = q.shape[1], q.shape[3], v.shape[3]
    scale, n = K ** -0.5, K + V + T + decay.shape[0]
    for state, d_s in ((None, None), (s0, d_last), (None, d_last)):
        want = attention_grads(q, k, v, do, decay, scale, state, d_s)
        mags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, scale, None if state is None else state.abs(),
                               None if d_s is None else d_s.abs())
        got = mb.linear_attention_bwd(q, k, v, do, decay, state=state, d_state_out=d_s)
        for name, w, m in zip(("d_q", "d_k", "d_v"), want, mags):
            close(got[name], w, m, dt, n, 0.0 if dt == "f32" else 2.0)
        assert ("d_state" in got) == (state is not None)
        if state is not None:
            state_close(got["d_state"], want[3], mags[3], T)
    # columns of one projection's gradient, the same bits; a state's gradient without a state
    widths = [t.shape[2] * t.shape[3] for t in (q, k, v)]
    d = torch.full((q.shape[0], T, sum(widths) + 3), 7.0, device=cuda_dev, dtype=q.dtype)
    parts = [d[..., sum(widths[:i]):sum(widths[:i + 1])].unflatten(-1, t.shape[2:]) for i, t in enumerate((q, k, v))]
    d_s0 = torch.empty_like(s0)
    again = mb.linear_attention_bwd(q, k, v, do, decay, d_state_out=d_last, d_q=parts[0], d_k=parts[1], d_v=parts[2], d_state=d_s0)
    # (a state that is handed on is kept in more terms, which d_v is made of too: the same results asked for, the same bits)
    got.update(mb.linear_attention_bwd(q, k, v, do, decay, d_state_out=d_last, d_state=torch.empty_like(s0)))
    for name, w, m in zip(("d_q", "d_k", "d_v"), want, mags):
        close(got[name], w, m, dt, n, 0.0 if dt == "f32" else 2.0)
        assert torch.equal(again[name], got[name]), name
    assert (d[..., -3:] == 7.0).all() and again["d_state"] is d_s0
    state_close(d_s0, want[3], mags[3], T)
    mb.ffi.default_handle(0).check_status()


def test_gradients_against_differences(cuda_dev):
    """Central differences of a weighted sum of o and of the state that leaves, in f32.  A step of 2^-4 leaves no error of the formula (it
    is linear in each of q, k, v and the state), the sums' roundings are below 2^-19 of them."""
    import torch

    import mamba_rs_b200 as mb
    q, k, v, do, decay, s0, d_last = inputs(cuda_dev, "f32", 2, 140, 4, 24, 16, 2, 4, 2, seed=3)
    g = mb.linear_attention_bwd(q, k, v, do, decay, state=s0, d_state_out=d_last)

    def value(q, k, v, s):
        last = torch.empty_like(s0)
        o = mb.linear_attention_fwd(q, k, v, decay, state=s, state_out=last)
        return float((o.double() * do.double()).sum() + (last.double() * d_last.double()).sum())

    gen = torch.Generator(cuda_dev).manual_seed(5)
    for i, name in enumerate(("d_q", "d_k", "d_v", "d_state")):
        args = [q, k, v, s0]
        way = torch.randn(args[i].shape, device=cuda_dev, generator=gen)
        ends = []
        for h in (2.0 ** -4, -2.0 ** -4):
            args[i] = (q, k, v, s0)[i] + h * way
            ends.append(value(*args))
        want = float((g[name].double() * way.double()).sum())
        size = float(g[name].double().norm() * way.double().norm())
        assert abs((ends[0] - ends[1]) * 8 - want) <= 2.0 ** -12 * size, name


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,K,V,heads", [(1, 1, 1, 1, (1, 1, 1)), (3, 4, 64, 64, (4, 4, 4)), (2, 6, 128, 64, (3, 2, 6)), (5, 2, 31, 17, (2, 2, 1)),
                                           (2, 3, 256, 256, (3, 3, 3)), (70, 4, 40, 56, (4, 1, 1)), (1, 2, 200, 4, (2, 2, 2))])
def test_step(cuda_dev, dt, B, H, K, V, heads):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention
    q, k, v, _, decay, s0, _ = inputs(cuda_dev, dt, B, 3, H, K, V, *heads, seed=2, pad=3)
    for t in range(3):
        want, last = attention(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], decay, 0.3, s0)
        mags, last_mags = attention(q[:, t:t + 1].abs(), k[:, t:t + 1].abs(), v[:, t:t + 1].abs(), decay, 0.3, s0.abs())
        out = torch.empty_like(s0)
        o = mb.linear_attention_step(q[:, t], k[:, t], v[:, t], decay, s0, scale=0.3, state_out=out)
        close(o, want[:, 0], mags[:, 0], dt, K + 1)
        state_close(out, last, last_mags, 1)
        # in place, and as a text of one token
        s = s0.clone()
        assert torch.equal(mb.linear_attention_step(q[:, t], k[:, t], v[:, t], decay, s, scale=0.3), o) and torch.equal(s, out)
        assert torch.equal(mb.linear_attention_fwd(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], decay, scale=0.3, state=s0)[:, 0], o)
        s0 = out


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("decays", ["none", "fast"])
def test_decays(cuda_dev, dt, decays):
    """No decay at all, and decays that leave nothing of a token a few steps later."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    q, k, v, do, decay, s0, d_last = inputs(cuda_dev, dt, 2, 700, 3, 64, 64, decays=decays)
    if decays == "fast":
        decay[0] = -math.inf  # (the reference's exp gives 0, which forgets everything before the token itself)
    for call in range(2):
        want, last = attention(q, k, v, decay, 0.125, s0)
        mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, 0.125, s0.abs())
        out = torch.empty_like(s0)
        close(mb.linear_attention_fwd(q, k, v, decay, state=s0, state_out=out), want, mags, dt, 64 + 700, 0.0 if dt == "f32" else 2.0)
        state_close(out, last, last_mags, 700)
    want = attention_grads(q, k, v, do, decay, 0.125, s0, d_last)
    mags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, 0.125, s0.abs(), d_last.abs())
    got = mb.linear_attention_bwd(q, k, v, do, decay, state=s0, d_state_out=d_last)
    for name, w, m in zip(("d_q", "d_k", "d_v"), want, mags):
        close(got[name], w, m, dt, 128 + 700, 0.0 if dt == "f32" else 2.0)
    state_close(got["d_state"], want[3], mags[3], 700)


@pytest.mark.parametrize("dt", DTS)
def test_pieces_of_a_text(cuda_dev, dt):
    """A text in pieces, its state handed on, some of them of one token or none."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention
    q, k, v, _, decay, s0, _ = inputs(cuda_dev, dt, 2, 520, 2, 64, 64, seed=4)
    want, last = attention(q, k, v, decay, 0.125, s0)
    mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, 0.125, s0.abs())
    s, parts, at = s0.clone(), [], 0
    for n in (1, 0, 130, 2, 1, 386):
        parts.append(mb.linear_attention_fwd(q[:, at:at + n], k[:, at:at + n], v[:, at:at + n], decay, state=s, state_out=s))
        at += n
    close(torch.cat(parts, 1), want, mags, dt, 64 + 520, 0.0 if dt == "f32" else 2.0)
    state_close(s, last, last_mags, 520)


def test_nothing_to_do(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    q, k, v, do, decay, s0, d_last = inputs(cuda_dev, "bf16", 2, 5, 3, 8, 16)
    e = lambda t: t[:, :0]  # noqa: E731
    out = torch.full_like(s0, 3.0)
    assert mb.linear_attention_fwd(e(q), e(k), e(v), decay, state=s0, state_out=out).shape == (2, 0, 3, 16) and torch.equal(out, s0)
    mb.linear_attention_fwd(e(q), e(k), e(v), decay, state_out=out)
    assert not out.any()
    g = mb.linear_attention_bwd(e(q), e(k), e(v), e(do), decay, state=s0, d_state_out=d_last)
    assert torch.equal(g["d_state"], d_last) and g["d_q"].shape == (2, 0, 3, 8)
    assert not mb.linear_attention_bwd(e(q), e(k), e(v), e(do), decay, state=s0)["d_state"].any()
    assert mb.linear_attention_fwd(q[:0], k[:0], v[:0], decay).shape == (0, 5, 3, 16)
    mb.linear_attention_bwd(q[:0], k[:0], v[:0], do[:0], decay)


@pytest.mark.parametrize("dt", DTS)
def test_layouts(cuda_dev, dt):
    """Heads before tokens, odd starts, batches apart, results inside a larger tensor whose rest stays."""
    import torch

    import mamba_rs_b200 as mb
    q, k, v, do, decay, s0, _ = inputs(cuda_dev, dt, 2, 200, 4, 64, 64, seed=6)
    want = mb.linear_attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), decay, state=s0)

    def moved(t, how):
        B, T, H, W = t.shape
        if how == "heads first":
            return torch.empty(B, H, T, W, device=cuda_dev, dtype=t.dtype).transpose(1, 2).copy_(t)
        if how == "odd":
            return torch.empty(B * T * H * W + 1, device=cuda_dev, dtype=t.dtype)[1:].view(t.shape).copy_(t)
        return torch.empty(B, T + 3, H + 1, W + 8, device=cuda_dev, dtype=t.dtype)[:, 3:, 1:, 8:].copy_(t)

    from retention_ref import attention
    ref, _ = attention(q, k, v, decay, 0.125, s0)
    mags, _ = attention(q.abs(), k.abs(), v.abs(), decay, 0.125, s0.abs())
    for how in ("heads first", "odd", "inside"):
        o = torch.full((2, 203, 5, 72), 7.0, device=cuda_dev, dtype=q.dtype)
        view = o[:, 3:, 1:, 8:]
        got = mb.linear_attention_fwd(moved(q, how), moved(k, how), moved(v, how), decay, state=s0, o=view)
        close(got, ref, mags, dt, 264, 0.0 if dt == "f32" else 2.0)
        if how != "odd":
            assert torch.equal(got, want)
        assert (o[:, :3] == 7).all() and (o[:, :, :1] == 7).all() and (o[..., :8] == 7).all()


def test_few_heads_of_a_long_text_with_and_without_scratch(cuda_dev):
    """Segments side by side, and one after another where no scratch is lent."""
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import attention, attention_grads
    for dt in DTS:
        q, k, v, do, decay, s0, d_last = inputs(cuda_dev, dt, 1, 2300, 2, 64, 64, seed=8)
        need = mb.linear_attention_workspace_bytes(1, 2300, 2, 64, 64)
        assert need > 0
        want, last = attention(q, k, v, decay, 0.125, s0)
        mags, last_mags = attention(q.abs(), k.abs(), v.abs(), decay, 0.125, s0.abs())
        for ws in (None, torch.empty(need, dtype=torch.uint8, device=cuda_dev), torch.empty(0, dtype=torch.uint8, device=cuda_dev)):
            out = s0.clone()
            o = mb.linear_attention_fwd(q, k, v, decay, state=out, state_out=out, workspace=ws)
            close(o, want, mags, dt, 64 + 2300, 0.0 if dt == "f32" else 2.0)
            state_close(out, last, last_mags, 2300)
        want = attention_grads(q, k, v, do, decay, 0.125, s0, d_last)
        mags = attention_grads(q.abs(), k.abs(), v.abs(), do.abs(), decay, 0.125, s0.abs(), d_last.abs())
        for ws in (None, torch.empty(0, dtype=torch.uint8, device=cuda_dev)):
            g = mb.linear_attention_bwd(q, k, v, do, decay, state=s0, d_state_out=d_last, workspace=ws)
            for name, w, m in zip(("d_q", "d_k", "d_v"), want, mags):
                close(g[name], w, m, dt, 128 + 2300, 0.0 if dt == "f32" else 2.0)
            state_close(g["d_state"], want[3], mags[3], 2300)


def test_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    q, k, v, do, decay, s0, d_last = inputs(cuda_dev, "bf16", 2, 6, 4, 8, 16)
    fwd, bwd, step = mb.linear_attention_fwd, mb.linear_attention_bwd, mb.linear_attention_step
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fwd(q, k.cpu(), v, decay)
    for call in (lambda: fwd(q, k[..., :4], v, decay), lambda: fwd(q, k.half(), v, decay), lambda: fwd(q, k, v, decay.double()),
                 lambda: fwd(q, k, v, decay, state=s0[:1]), lambda: fwd(q, k, v, decay, state=s0.half()), lambda: fwd(q, k[:, :3], v, decay),
                 lambda: fwd(q.double(), k.double(), v.double(), decay), lambda: fwd(q, k, v, decay, o=torch.empty_like(q)),
                 lambda: bwd(q, k, v, do[..., :8], decay), lambda: bwd(q, k, v, do, decay, d_state_out=d_last.transpose(2, 3)),
                 lambda: step(q[:, 0], k[:, 0], v[:, 0], decay, s0[:1]), lambda: step(q[:, 0], k[:1, 0], v[:, 0], decay, s0)):
        with pytest.raises(TypeError):
            call()
    wide = torch.zeros(2, 6, 1, 264, device=cuda_dev, dtype=torch.bfloat16)
    for call in (lambda: fwd(q[:, :, :3], k, v, decay), lambda: fwd(q, k, v, decay[:3]), lambda: fwd(q.transpose(2, 3), k.transpose(2, 3), v, decay),
                 lambda: fwd(wide, wide, v, decay), lambda: fwd(q, k, wide, decay), lambda: fwd(q[0], k[0], v[0], decay),
                 lambda: fwd(q, k, v, decay, o=do[:, :, :1].expand(2, 6, 4, 16)),
                 lambda: fwd(q, k, v, decay, workspace=torch.empty(1, dtype=torch.uint8, device=cuda_dev).expand(9))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="scale"):
        fwd(q, k, v, decay, scale=math.inf)
    with pytest.raises(RuntimeError, match="same memory"):
        bwd(q, k, v, do, decay, state=s0, d_state_out=d_last, d_state=d_last)
    with pytest.raises(RuntimeError, match="shared heads need a workspace"):
        bwd(q[:, :, :2], k, v, do, decay, workspace=torch.empty(256, dtype=torch.uint8, device=cuda_dev))
    mb.ffi.default_handle(0).check_status()
