"""Linear attention, rotation and group norm of very many sequences, heads, samples or groups: results do not depend on what else a call
holds, so each is compared, bit for bit, with calls on parts of it that are of an ordinary size."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("N,S,C,G", [(1500000, 1, 64, 4), (300000, 2, 16, 2), (70000, 1, 8, 8), (100003, 5, 24, 3), (40000, 3, 33, 11)])
def test_norms_of_many_samples(cuda_dev, dt, N, S, C, G):
    import torch
    from retention_ref import DT, fro

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(N)
    x, z, dy = (torch.randn(N, S, C, device=cuda_dev, generator=g).to(DT[dt]) for _ in range(3))
    w, b = torch.randn(2, C, device=cuda_dev, generator=g)
    y, stats = mb.group_norm_fwd(x, w, b, G, activation="silu", z=z)
    d = mb.group_norm_bwd(dy, x, stats, w, b, G, activation="silu", z=z)
    part = 1000
    sums = torch.zeros(2, C, dtype=torch.float64, device=cuda_dev)
    for at in (0, N // 2, N - part):
        p = slice(at, at + part)
        yp, sp = mb.group_norm_fwd(x[p], w, b, G, activation="silu", z=z[p])
        # (a part may be cut into other blocks, whose sums join in another order: a few roundings, and half a step of the result)
        assert fro(yp, y[p].double()) <= (2.0 ** -8 if dt == "bf16" else 2.0 ** -20)
        dp = mb.group_norm_bwd(dy[p], x[p], sp, w, b, G, activation="silu", z=z[p])
        for n in ("d_x", "d_z"):
            assert fro(dp[n], d[n][p].double()) <= (2.0 ** -8 if dt == "bf16" else 2.0 ** -20), n
    for at in range(0, N, 20000):
        p = slice(at, min(at + 20000, N))
        dp = mb.group_norm_bwd(dy[p], x[p], stats[:, p].contiguous(), w, b, G, activation="silu", z=z[p])
        sums += torch.stack((dp["d_weight"], dp["d_bias"])).double()
    # sums of N S products in 32 bits, joined from blocks: 2^-24 sqrt(N S) of their size in the mean, 2^-24 times the depth of the joining beside it
    size = (dy.double().abs().sum((0, 1)) * 8 + 1) * 2.0 ** -20
    assert (torch.stack((d["d_weight"], d["d_bias"])).double() - sums).abs().le(size).all()
    mb.ffi.default_handle(0).check_status()


def test_norms_of_many_groups(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    x = torch.randn(3, 1, 400000, device=cuda_dev)
    y, stats = mb.group_norm_fwd(x, None, None, 100000)
    want, s2 = mb.group_norm_fwd(x.view(300000, 1, 4), None, None, 1)
    assert torch.equal(y.view(300000, 1, 4), want) and torch.equal(stats.flatten(1), s2.flatten(1))
    d = mb.group_norm_bwd(y, x, stats, None, None, 100000)["d_x"]
    assert torch.allclose(d.view(300000, 1, 4), mb.group_norm_bwd(want, x.view(300000, 1, 4), s2, None, None, 1)["d_x"], rtol=2.0 ** -18, atol=2.0 ** -18)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_many_sequences_and_heads(cuda_dev, dt):
    import torch
    from retention_ref import DT

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(3)
    for B, T, H in ((50000, 3, 20), (1, 3, 100000), (100000, 1, 2)):
        q, k, v, do = (torch.randn(B, T, H, 8, device=cuda_dev, generator=g).to(DT[dt]) for _ in range(4))
        decay = -torch.rand(H, device=cuda_dev, generator=g)
        s = torch.randn(B, H, 8, 8, device=cuda_dev, generator=g)
        last = torch.empty_like(s)
        o = mb.linear_attention_fwd(q, k, v, decay, state=s, state_out=last)
        d = mb.linear_attention_bwd(q, k, v, do, decay, state=s)
        for at in (0, B // 2, B - 1):
            p = slice(at, at + 1)
            l1 = torch.empty_like(s[p])
            assert torch.equal(mb.linear_attention_fwd(q[p], k[p], v[p], decay, state=s[p].contiguous(), state_out=l1), o[p]) and torch.equal(l1, last[p])
            d1 = mb.linear_attention_bwd(q[p], k[p], v[p], do[p], decay, state=s[p].contiguous())
            for n in d:
                assert torch.equal(d1[n], d[n][p]), n
        f = mb.rotary_frequencies(8, device=cuda_dev)[0]
        positions = torch.arange(T, device=cuda_dev, dtype=torch.int32)
        if H <= 65536:
            a, b = mb.rotary_fwd(q, k, positions, f)
            for at in (0, B - 1):
                p = slice(at, at + 1)
                a1, b1 = mb.rotary_fwd(q[p], k[p], positions, f)
                assert torch.equal(a1, a[p]) and torch.equal(b1, b[p])
        else:
            with pytest.raises(RuntimeError, match="heads"):
                mb.rotary_fwd(q, k, positions, f)
    mb.ffi.default_handle(0).check_status()
