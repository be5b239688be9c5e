"""Token log probabilities where a row is hard on the arithmetic: very large and very low logits, tiny temperatures, one token
that is all but certain, rows that are mostly no numbers.  All against the definition in 64 bits.

Tolerances.  As beside the ordinary rows: with E = 2^-21 (2 + log V) + 2^-24 (V / 256 + 16), log S is off by E, the entropy by
E (2 + log V), a log probability by E and 2^-22 of its value.  For a token that is all but certain the bound is closer, since the
others carry little weight: its exponent is rounded at no more than 8 or 9 in base 2 (2^-21), two exponentials (2^-22 each) scale it
and a handful of roundings (2^-24 each) follow, below 2^-19 in all; the entropy's second sum is 8 or 9 times the first before the two
are subtracted, which adds roundings of 2^-21 each, below 2^-18, and the rest have exponents of up to 100, whose relative error of 2^-17
weighs as much as they do in the entropy."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DT = ["f32", "bf16", "f16"]
# short rows, rows over a cluster's CTAs, rows one after another
SIZES = [(5, 777), (3, 5003), (700, 5003), (3, 50280), (600, 50277)]


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _plain(l, t, temp):
    """log S, entropy, log probabilities of all tokens (beyond f32's range: infinite) and of the targets."""
    import torch
    l = l.double() / float(np.float32(temp))
    d = l - l.amax(1)[:, None]
    e = torch.exp(d)
    log_s = torch.log1p((e.sum(1) - 1.0).clamp(min=0.0))
    logp = d - log_s[:, None]
    H = log_s - (e * torch.where(e > 0, d, 0.0)).sum(1) / e.sum(1)
    logp = torch.where(logp < -float(torch.finfo(torch.float32).max), -math.inf, logp)
    return log_s, H, logp, logp.gather(1, t.long()[:, None])[:, 0]


def _close(got, want, tol):
    import torch
    got, fin = got.double(), torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    tol = tol.expand_as(want)[fin] if hasattr(tol, "expand_as") else tol
    assert ((got - want).abs()[fin] <= tol).all(), (got - want)[fin].abs().max()


def _check(l, t, temp, top=5):
    import torch

    import mamba_rs_b200 as mb
    V = l.shape[1]
    log_s, H, logp, lp = _plain(l, t, temp)
    e, big = 2.0 ** -21 * (2 + math.log(V)) + 2.0 ** -24 * (V / 256 + 16), 2.0 ** -22
    r = mb.token_logprobs(l, t, top=top, temperature=temp)
    assert torch.equal(r["lse"][0], l.float().amax(1))
    _close(r["lse"][1], log_s, e)
    _close(r["entropy"], H, e * (2 + math.log(V)))
    _close(r["logprob"], lp, e + big * lp.abs())
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(r["top_ids"].long(), order)
    want = logp.gather(1, order)
    _close(r["top_logprobs"], want, e + big * want.abs())
    plain = mb.token_logprobs(l, t, temperature=temp)  # (without alternatives: another kernel)
    for k, tol in (("lse", e), ("entropy", e * (2 + math.log(V)))):
        assert ((plain[k] - r[k]).abs() <= 2 * tol).all()
    mb.ffi.default_handle(0).check_status()
    return r


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("high", [1e6, 1e9, 1e10, 1e30, "max"])
def test_tokens_that_are_forced(cuda_dev, dt, rows, V, high):
    """A very large logit in one place, in some, in the whole row."""
    import torch
    g = torch.Generator(cuda_dev).manual_seed(V + rows)
    l = torch.randn(rows, V, device=cuda_dev, generator=g) * 3
    high = torch.finfo(_dt(dt)).max if high == "max" else min(high, torch.finfo(_dt(dt)).max)
    at = torch.randint(0, V, (rows, 4), device=cuda_dev, generator=g)
    l.scatter_(1, at[:, :1], high)
    l[1::3] = l[1::3].scatter(1, at[1::3], high)
    l[2::3] = high
    t = torch.randint(0, V, (rows,), device=cuda_dev, dtype=torch.int32, generator=g)
    t[::2] = at[::2, 0].int()
    for temp in (1.0, 0.7):
        _check(l.to(_dt(dt)), t, temp)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e10, -1e20, -1e30])
def test_masks_of_large_negative_values(cuda_dev, dt, rows, V, low):
    """All but a few neighbouring tokens at one low value; whole rows of it."""
    import torch
    g = torch.Generator(cuda_dev).manual_seed(V + rows)
    low = max(low, torch.finfo(_dt(dt)).min)
    l = torch.full((rows, V), low, device=cuda_dev)
    for r in range(rows):
        if r % 3 != 1:
            at = (977 * r + 31) % (V - 9)
            l[r, at:at + 9] = torch.randn(9, device=cuda_dev, generator=g) * 3
    t = torch.arange(rows, device=cuda_dev, dtype=torch.int32) * 977 + 33
    t = (t % (V - 9)).int()
    for temp in (1.0, 0.7):
        _check(l.to(_dt(dt)), t, temp)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("temp", [1e-4, 1e-6, 1e-8, 1e-12, 1e-30])
def test_tiny_temperatures(cuda_dev, dt, rows, V, temp):
    import torch
    g = torch.Generator(cuda_dev).manual_seed(V + rows)
    l = (torch.randn(rows, V, device=cuda_dev, generator=g) * 3).to(_dt(dt))
    l[1::3] -= 40.0
    t = torch.randint(0, V, (rows,), device=cuda_dev, dtype=torch.int32, generator=g)
    t[::2] = l.float().argmax(1)[::2].int()
    _check(l, t, temp)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,V", SIZES)
@pytest.mark.parametrize("gap", [10, 12, 15, 20, 25, 30, 40])
def test_one_token_that_is_all_but_certain(cuda_dev, dt, rows, V, gap):
    """One logit stands above the rest, in the row's later half; no probability is above 1 and no entropy below 0."""
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(V + rows + gap)
    l = torch.randn(rows, V, device=cuda_dev, generator=g) * 2
    at = torch.randint(V // 2, V, (rows, 1), device=cuda_dev, generator=g)
    l.scatter_(1, at, l.amax(1, keepdim=True) + gap)
    l = l.to(_dt(dt))
    t = at[:, 0].int()
    log_s, H, logp, lp = _plain(l, t, 1.0)
    for top in (0, 3):
        r = mb.token_logprobs(l, t, top=top)
        assert (r["logprob"] <= 0).all() and (r["entropy"] >= 0).all() and (r["lse"][1] >= 0).all()
        _close(r["lse"][1], log_s, 2.0 ** -19 * (1 + log_s))
        _close(r["logprob"], lp, 2.0 ** -19 * (1 + lp.abs()))
        _close(r["entropy"], H, 2.0 ** -18 + 2.0 ** -17 * H)
        if top:
            assert (r["top_logprobs"] <= 0).all() and torch.equal(r["top_ids"][:, 0], t)


@pytest.mark.parametrize("dt", DT)
def test_alternatives_of_rows_that_are_mostly_no_numbers(cuda_dev, dt):
    """NaN ranks as minus infinity among the alternatives wherever it lies, in rows that start between 16-byte places too."""
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(11)
    for V, ld, off in ((1024, 1025, 1), (1024, 1031, 3), (512, 513, 1), (2048, 2049, 5), (4096, 4097, 1), (6000, 6001, 1)):
        rows = 64
        store = torch.full((rows * ld + off,), math.nan, device=cuda_dev, dtype=_dt(dt))
        l = store[off:].view(rows, ld)[:, :V]
        for r in range(rows):
            n = 1 + r % 12
            where = torch.randperm(V, device=cuda_dev, generator=g)[:n]
            l[r, where] = torch.randn(n, device=cuda_dev, generator=g).to(_dt(dt))
        ranked = torch.where(torch.isnan(l), -math.inf, l.float())
        for top in (1, 5, 8, 20, 32):
            order = torch.sort(ranked, dim=1, descending=True, stable=True)[1][:, :top]
            assert torch.equal(mb.token_logprobs(l, top=top)["top_ids"].long(), order), (V, top)


def test_temperatures_whose_reciprocal_leaves_the_range_are_refused(cuda_dev):
    """log2(e) / temperature has to be a number of 32 bits."""
    import torch

    import mamba_rs_b200 as mb
    l, t = torch.zeros(2, 40, device=cuda_dev), torch.zeros(2, dtype=torch.int32, device=cuda_dev)
    v, v2 = torch.zeros(2, device=cuda_dev), torch.zeros(2, 2, device=cuda_dev)
    for temp in (4e-39, 3.5e-39, 1e-44):
        with pytest.raises(RuntimeError, match="temperature"):
            mb.token_logprobs(l, t, temperature=temp)
        with pytest.raises(RuntimeError, match="temperature"):
            mb.token_logprobs_bwd(l, t, v2, v, v, temperature=temp)
    r = mb.token_logprobs(l, t, temperature=5e-39)
    assert (r["lse"][1] - math.log(40)).abs().max() <= 2.0 ** -19
