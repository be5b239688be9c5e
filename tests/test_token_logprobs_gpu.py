"""Log probabilities of given tokens, entropy, alternatives, and the gradient of the logits, in 64 bits beside them.

Tolerances.  With d = (l - max) / temperature, log S the log of the sum of exp d, an exponential of the device has a relative error of at most 2^-22 and its
argument one of 2^-22 |d| (two roundings and the product with log2 e); weighted by p, whose mean |d| is at most
1 + log V, the sum's relative error and with it log S, log p and the entropy are off by E = 2^-21 (2 + log V) and one rounding
of the value itself; the entropy's second sum has the same error relative to 1 + log V.  A sum of V terms in chains of a
thread's length adds at most 2^-24 (V / 256 + 16) more.  The gradient is a product with p, whose log is off by E and 2^-23 of
its value."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DT = ["f32", "bf16", "f16"]
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half an ulp


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _case(rows, V, dt, dev, seed=0, mask=None):
    import torch
    g = torch.Generator(dev).manual_seed(seed + V)
    l = torch.randn(rows, V, device=dev, generator=g) * 3
    if mask == "half":
        l[torch.rand(rows, V, device=dev, generator=g) < 0.5] = -math.inf
        l[1::3] = -math.inf
        l[2::5, : V - 1] = -math.inf  # one token left, if that
    if mask == "lowest":
        l[torch.rand(rows, V, device=dev, generator=g) < 0.5] = torch.finfo(_dt(dt)).min
        l[1::3] = torch.finfo(_dt(dt)).min
    l = l.to(_dt(dt))
    t = torch.randint(0, V, (rows,), device=dev, dtype=torch.int32, generator=g)
    if rows > 3:
        t[3] = -1
        t[rows - 1] = V
    return l, t


def _plain(l, t, temp):
    """log S, entropy, logprob, p, log p in 64 bits; a row with nothing left as the operator defines it, and what lies
    beyond f32's range infinite."""
    import torch
    l = l.double() / float(np.float32(temp))
    V = l.shape[1]
    m = l.amax(1)
    none = torch.isinf(m) & (m < 0)
    d = l - torch.where(none, 0.0, m)[:, None]  # (the type's lowest value takes the sum's logarithm, also of 64 bits)
    log_s = torch.where(none, 0.0, torch.log(torch.exp(d).sum(1)))
    logp = d - log_s[:, None]
    logp = torch.where(logp < -float(torch.finfo(torch.float32).max), -math.inf, logp)
    p = torch.exp(logp)
    H = -(p * torch.where(p == 0, 0.0, logp)).sum(1)
    counted = (t >= 0) & (t < V)
    lp = torch.where(counted, logp.gather(1, t.long().clamp(0, V - 1)[:, None])[:, 0], 0.0)
    return log_s, H, lp, p, logp, counted, none


def _close(got, want, tol):
    import torch
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin])
    assert ((got - want).abs()[fin] <= (tol.expand_as(want)[fin] if hasattr(tol, "expand_as") else tol)).all(), (got - want)[fin].abs().max()


def _tol(V):
    return 2.0 ** -21 * (2 + math.log(V)) + 2.0 ** -24 * (V / 256 + 16)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("mask", [None, "half", "lowest"])
@pytest.mark.parametrize("rows,V", [(1, 1), (5, 2), (9, 31), (4, 257), (3, 1000), (300, 777), (7, 50280), (2, 50277), (700, 5003), (1, 120001)])
def test_values_and_alternatives(cuda_dev, dt, mask, rows, V):
    import torch

    import mamba_rs_b200 as mb
    l, t = _case(rows, V, dt, cuda_dev, mask=mask)
    for top, temp in ((min(20, V), 1.0), (min(32, V), 0.7), (0, 1.0), (1, 2.5)):
        log_s, H, lp, p, logp, counted, none = _plain(l, t, temp)
        r = mb.token_logprobs(l, t, top=top, temperature=temp)
        e = _tol(V)
        big = 2.0 ** -22  # of the value itself: the product with 1 / temperature and the final rounding
        assert torch.equal(r["lse"][0], l.float().amax(1))
        _close(r["lse"][1], log_s, e)
        _close(r["entropy"], H, e * (2 + math.log(V)))
        _close(r["logprob"], lp, e + big * lp.abs())
        assert (r["logprob"][~counted] == 0).all()
        if top:
            order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1][:, :top]
            assert torch.equal(r["top_ids"].long(), order)
            want = logp.gather(1, order)
            _close(r["top_logprobs"], want, e + big * want.abs())
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DT)
def test_alternatives_among_many_equals(cuda_dev, dt):
    """Equal logits, runs of large ones in any place, rising and falling rows: always by value, then by index."""
    import torch

    import mamba_rs_b200 as mb
    V = 20011
    i = torch.arange(V, device=cuda_dev)
    rows = [torch.zeros(V, device=cuda_dev), (i % 3 == 1).float(), i.float() / 16, -i.float() / 16, (i // 4096 == 3).float() * 5,
            (i % 4096 < 300).float() * (5 + (i % 7)), (i % 2048 >= 2000).float() + (i % 5), torch.where(i < 31, 1.0, -math.inf),
            torch.where(i == V - 1, 1.0, -math.inf), (i // 700 % 2).float() * (i % 700)]
    l = torch.stack(rows).to(_dt(dt))
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1]
    for n in (1, len(rows)):  # (few rows, and again as many)
        for top in (1, 2, 20, 32):
            for many in (1, 80):
                got = mb.token_logprobs(l[:n].repeat(many, 1), top=top)["top_ids"]
                assert torch.equal(got.long(), order[:n, :top].repeat(many, 1))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("V", [20011, 50280])
def test_alternatives_where_more_stand_out_than_there_is_room_for(cuda_dev, dt, V):
    """Large logits that gather in a few columns of the row's layout, distinct and in runs of equals, at its start or its end."""
    import torch

    import mamba_rs_b200 as mb
    i = torch.arange(V, device=cuda_dev)
    rows = []
    for span in (2048, 1024):  # (256 threads x 16 bytes, in 16 and 32 bits)
        for few in (24, 160, 400):
            top = i % span < few
            rows += [torch.where(top, 100.0 + i * 0.5, 0.0), torch.where(top, 3.0, 0.0), torch.where(top, 3.0 + (i % 5), -math.inf),
                     torch.where(top & (i > V // 2), 3.0, -1.0), torch.where(top, 2000.0 - (i // 7), -i * 0.01)]
    l = torch.stack(rows).to(_dt(dt))
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1]
    for top in (1, 20, 32):
        for many in (1, 25):
            assert torch.equal(mb.token_logprobs(l.repeat(many, 1), top=top)["top_ids"].long(), order[:, :top].repeat(many, 1))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("V", [637, 4001, 20011, 50280])
def test_alternatives_where_neighbours_are_left_or_many_are_equal(cuda_dev, dt, V, rows):
    """A run of tokens is left and all others are ruled out, or the logits have few distinct values."""
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(V + rows)
    l = torch.randn(8, V, device=cuda_dev, generator=g) * 3
    for i, n in enumerate((5, 100, 300, 600, 1000)):
        at = (137 * i + 1) % V
        l[i, :at] = -math.inf
        l[i, at + n:] = -math.inf
    l[5] = torch.round(l[5])
    l[6] = torch.round(l[6] * 8) / 8
    l[7] = -1.5
    l = l.to(_dt(dt))
    order = torch.sort(l.float(), dim=1, descending=True, stable=True)[1]
    many = (rows + 7) // 8
    for top in (1, 8, 9, 20, 32):
        got = mb.token_logprobs(l.repeat(many, 1)[:rows], top=top)["top_ids"]
        assert torch.equal(got.long(), order[:, :top].repeat(many, 1)[:rows])
        if rows < 8:
            got = mb.token_logprobs(l[8 - rows:], top=top)["top_ids"]
            assert torch.equal(got.long(), order[8 - rows:, :top])


@pytest.mark.parametrize("dt", DT)
def test_what_is_not_a_number_shows(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    V = 3000
    l = torch.randn(6, V, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(4)).to(_dt(dt))
    l[1, 17] = math.nan
    l[2, 2999] = math.inf
    l[3] = math.nan
    l[4, 5] = math.nan
    l[4, 9:] = -math.inf
    t = torch.full((6,), 40, dtype=torch.int32, device=cuda_dev)
    r = mb.token_logprobs(l, t, top=4)
    for k in ("lse", "entropy", "logprob"):
        bad = torch.isnan(r[k].sum(0) if k == "lse" else r[k])
        assert bad.tolist() == [False, True, True, True, True, False], k
    ranked = torch.where(torch.isnan(l), -math.inf, l.float())
    assert torch.equal(r["top_ids"].long(), torch.sort(ranked, dim=1, descending=True, stable=True)[1][:, :4])
    assert torch.isnan(r["top_logprobs"][[1, 2, 3, 4]]).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("mask", [None, "half", "lowest"])
@pytest.mark.parametrize("rows,V", [(1, 1), (9, 31), (4, 257), (300, 777), (5, 50280), (3, 50277)])
def test_gradient(cuda_dev, dt, mask, rows, V):
    import torch

    import mamba_rs_b200 as mb
    l, t = _case(rows, V, dt, cuda_dev, seed=1, mask=mask)
    g = torch.Generator(cuda_dev).manual_seed(9)
    gl, gh = torch.randn(rows, device=cuda_dev, generator=g), torch.randn(rows, device=cuda_dev, generator=g)
    for temp in (1.0, 0.7):
        _, H, lp, p, logp, counted, none = _plain(l, t, temp)
        r = mb.token_logprobs(l, t, temperature=temp)
        hot = torch.zeros_like(p)
        hot[counted, t[counted].long()] = 1.0
        safe = torch.where(p == 0, 0.0, logp)
        parts = (gl[:, None].double() * (hot - p) * (counted & ~none)[:, None], -gh[:, None].double() * p * (safe + H[:, None]))
        e = _tol(V)
        mag = (gl.abs()[:, None] * (hot + p) + gh.abs()[:, None] * p * (safe.abs() + H[:, None] + 4)) / temp
        for dl, dh, want in ((gl, gh, sum(parts)), (gl, None, parts[0]), (None, gh, parts[1])):
            got = mb.token_logprobs_bwd(l, t if dl is not None else None, r["lse"], r["entropy"], dl, dh, temperature=temp)
            tiny = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}[dt]
            tol = (2 * e + 2.0 ** -22 * safe.abs()) * mag + HALF[dt] * 1.01 * (want / temp).abs() + tiny
            assert ((got.double() - want / temp).abs() <= tol).all()
            assert not got[none].any()
        own = l.clone()  # in place of the logits
        assert torch.equal(mb.token_logprobs_bwd(own, t, r["lse"], r["entropy"], gl, gh, temperature=temp, dlogits=own),
                           mb.token_logprobs_bwd(l, t, r["lse"], r["entropy"], gl, gh, temperature=temp))


def test_gradient_agrees_with_differences(cuda_dev):
    """Central differences of sum(a logprob + b entropy), taken of the 64-bit definition around the f32 logits."""
    import torch

    import mamba_rs_b200 as mb
    l, t = _case(4, 40, "f32", cuda_dev, seed=2)
    t[3] = 7
    g = torch.Generator(cuda_dev).manual_seed(3)
    a, b = torch.randn(4, device=cuda_dev, generator=g), torch.randn(4, device=cuda_dev, generator=g)
    r = mb.token_logprobs(l, t, temperature=0.9)
    got = mb.token_logprobs_bwd(l, t, r["lse"], r["entropy"], a, b, temperature=0.9).double()

    def loss(x):
        _, H, lp, *_ = _plain(x, t, 0.9)
        return a.double() * lp + b.double() * H
    eps = 1e-5
    for v in (0, 7, 39):
        up, down = l.double(), l.double()
        up[:, v] += eps
        down[:, v] -= eps
        # third differences: eps^2 times derivatives of order one; then 64-bit rounding over eps
        assert ((loss(up) - loss(down)) / (2 * eps) - got[:, v]).abs().max() <= 1e-5


@pytest.mark.parametrize("dt", DT)
def test_strides_and_offsets(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    for rows, V, ld, off in ((5, 1000, 1008, 0), (6, 999, 1003, 5), (300, 515, 516, 1), (4, 50277, 50277, 3), (7, 64, 1, 0)):
        if ld == 1:
            ld = 2 * V + 1
        store = (torch.randn(rows * ld + off, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(ld)) * 3).to(_dt(dt))
        l = store[off:off + rows * ld].view(rows, ld)[:, :V]
        t = torch.arange(rows, dtype=torch.int32, device=cuda_dev)
        want, got = mb.token_logprobs(l.contiguous(), t, top=5), mb.token_logprobs(l, t, top=5)
        e = 2 * _tol(V)
        assert torch.equal(want["top_ids"], got["top_ids"])
        for k in ("lse", "entropy", "logprob", "top_logprobs"):
            assert ((want[k] - got[k]).abs() <= e * (2 + math.log(V)) + 2.0 ** -22 * want[k].abs()).all()
        room = torch.full((rows, ld + 9), 3.0, device=cuda_dev, dtype=_dt(dt))
        d = room[:, 2:2 + V]
        gl = torch.ones(rows, device=cuda_dev)
        mb.token_logprobs_bwd(l, t, want["lse"], want["entropy"], gl, gl, dlogits=d)
        assert torch.equal(d, mb.token_logprobs_bwd(l.contiguous(), t, want["lse"], want["entropy"], gl, gl))
        assert (room[:, :2] == 3).all() and (room[:, 2 + V:] == 3).all()


def test_the_same_bits_again_and_without_targets(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    for rows, V in ((3, 50277), (400, 3001)):
        l, t = _case(rows, V, "bf16", cuda_dev)
        a, b = (mb.token_logprobs(l, t, top=20) for _ in range(2))
        assert all(torch.equal(a[k], b[k]) for k in a)
        c = mb.token_logprobs(l, top=20)
        assert "logprob" not in c and all(torch.equal(a[k], c[k]) for k in c)


def test_no_rows_and_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    l, t = _case(4, 40, "f32", cuda_dev)
    v = torch.zeros(4, device=cuda_dev)
    assert mb.token_logprobs(l[:0], t[:0], top=3)["top_ids"].shape == (0, 3)
    v2 = torch.zeros(2, 4, device=cuda_dev)
    assert mb.token_logprobs_bwd(l[:0], t[:0], v2[:, :0].contiguous(), v[:0], v[:0]).shape == (0, 40)
    for bad in (lambda: mb.token_logprobs(l.t(), t), lambda: mb.token_logprobs(l, t.long()), lambda: mb.token_logprobs(l, t[:3]),
                lambda: mb.token_logprobs(l.double(), t), lambda: mb.token_logprobs_bwd(l, t, v2.half(), v, v),
                lambda: mb.token_logprobs_bwd(l, t, v, v, v), lambda: mb.token_logprobs_bwd(l, t, v2, v, v, dlogits=l.half())):
        with pytest.raises(TypeError):
            bad()
    for top in (-1, 33, 41):
        with pytest.raises(ValueError):
            mb.token_logprobs(l, t, top=top)
    for temp in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="temperature"):
            mb.token_logprobs(l, t, temperature=temp)
    with pytest.raises(RuntimeError, match="null"):
        mb.token_logprobs_bwd(l, None, v2, v, v)  # a gradient of log probabilities of no tokens
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mb.token_logprobs(l.cpu())


def test_rows_that_are_one_in_memory_are_refused(cuda_dev):
    """An expanded tensor has a row stride of 0: it is no matrix of that many rows for the kernels."""
    import torch

    import mamba_rs_b200 as mb
    l, t = _case(1, 40, "f32", cuda_dev)
    v = torch.zeros(3, device=cuda_dev)
    with pytest.raises(RuntimeError, match="bad dims"):
        mb.token_logprobs(l.expand(3, 40))
    with pytest.raises(RuntimeError, match="bad dims"):
        mb.token_logprobs_bwd(l.expand(3, 40), None, torch.zeros(2, 3, device=cuda_dev), v, None, v)
