"""Token table lookup with scaling and the table's gradient, against plain sums in 64 bits.

Tolerances.  The lookup is one f32 product (exact in 64 bits, rounded once) and one rounding to the output's dtype: bit
for bit.  A gradient element is a sum of n f32 terms in some order, times the scale: its error is at most
(n + 2) 2^-24 times the sum of the terms' magnitudes (every addition rounds by half an ulp of a partial sum)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DT = ["f32", "bf16", "f16"]


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _ids(kind, rows, vocab, rng):
    if kind == "one":
        return np.full(rows, vocab // 2, np.int32)
    if kind == "each":  # every token at most once
        return rng.permutation(max(rows, vocab))[:rows].astype(np.int32) % vocab
    ids = np.minimum((vocab * rng.random(rows) ** 4).astype(np.int32), vocab - 1)  # a few tokens often, most seldom
    if kind == "padded":
        ids[rows // 2:] = 0
        ids[3::7] = -1
        ids[5::11] = vocab
        ids[6::13] = np.iinfo(np.int32).min
    return ids


def _grad64(ids, d, vocab, scale):
    """The sums, the sums of magnitudes, and how many terms each has."""
    ok = (ids >= 0) & (ids < vocab)
    s, mag, n = np.zeros((vocab, d.shape[1])), np.zeros((vocab, d.shape[1])), np.zeros(vocab)
    np.add.at(s, ids[ok], d[ok].astype(np.float64) * scale)
    np.add.at(mag, ids[ok], np.abs(d[ok].astype(np.float64) * scale))
    np.add.at(n, ids[ok], 1)
    return s, mag, n[:, None]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,vocab,dim", [(1, 7, 1), (3, 50, 33), (257, 1000, 768), (64, 50280, 100), (5, 9, 2563), (2050, 300, 8)])
def test_lookup_is_the_scaled_row_bit_for_bit(cuda_dev, dt, rows, vocab, dim):
    import torch

    import mamba_rs_b200 as mb
    rng = np.random.default_rng(rows + dim)
    table = torch.randn(vocab, dim, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(dim)).to(_dt(dt))
    ids = torch.from_numpy(_ids("padded", rows, vocab, rng)).to(cuda_dev)
    ok = ((ids >= 0) & (ids < vocab))[:, None]
    for scale in (1.0, 27.712812921102035):
        want = torch.where(ok, (table.double()[ids.long().clamp(0, vocab - 1)] * np.float32(scale).astype(np.float64)).float(), 0.0)
        assert torch.equal(mb.embedding_fwd(table, ids, scale=scale), want)
        assert torch.equal(mb.embedding_fwd(table, ids, scale=scale, out_dtype=_dt(dt)), want.to(_dt(dt)))


@pytest.mark.parametrize("dt", DT)
def test_lookup_takes_strides_and_offsets(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(1)
    for dim, ld, off in ((64, 64, 1), (64, 72, 8), (96, 97, 0), (31, 40, 3), (768, 769, 2)):
        store = torch.randn(50 * ld + off, device=cuda_dev, generator=g).to(_dt(dt))
        table = store[off:off + 50 * ld].view(50, ld)[:, :dim]
        ids = torch.randint(0, 50, (4, 9), device=cuda_dev, dtype=torch.int32, generator=g)
        room = torch.full((36, ld + 5), 7.0, device=cuda_dev)
        out = room[:, 3:3 + dim]
        mb.embedding_fwd(table, ids, out=out)
        assert torch.equal(out, table[ids.view(-1).long()].float())
        assert (room[:, :3] == 7).all() and (room[:, 3 + dim:] == 7).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("kind", ["zipf", "one", "each", "padded"])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 3, 5), (32, 1000, 128), (33, 40, 77), (700, 500, 33), (3001, 257, 64), (5000, 50280, 24),
                                            (9000, 2000, 260), (40000, 700, 9)])
def test_gradient_is_the_sum_by_token(cuda_dev, dt, kind, rows, vocab, dim):
    import torch

    import mamba_rs_b200 as mb
    rng = np.random.default_rng(rows + vocab + dim)
    ids_h = _ids(kind, rows, vocab, rng)
    d = torch.randn(rows, dim, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(rows)).to(_dt(dt))
    ids = torch.from_numpy(ids_h).to(cuda_dev)
    scale = 1.7
    want, mag, n = _grad64(ids_h, d.float().cpu().numpy(), vocab, float(np.float32(scale)))
    got = mb.embedding_bwd(ids, d, vocab, scale=scale)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= (n + 2) * 2.0 ** -24 * mag).all()
    # the same bits again, and beside what was there
    assert torch.equal(got, mb.embedding_bwd(ids, d, vocab, scale=scale))
    base = torch.randn(vocab, dim, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(5))
    acc = mb.embedding_bwd(ids, d, d_table=base.clone(), scale=scale)
    b = base.double().cpu().numpy()
    assert (np.abs(acc.double().cpu().numpy() - b - want) <= (n + 3) * 2.0 ** -24 * (mag + np.abs(b))).all()
    absent = torch.from_numpy(n[:, 0] == 0).to(cuda_dev)
    assert torch.equal(acc[absent], base[absent]) and not got[absent].any()
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gradient_takes_strides_a_given_workspace_and_dirty_memory(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    rng = np.random.default_rng(3)
    for rows, vocab, dim, ld, off in ((300, 60, 64, 72, 8), (2600, 3000, 31, 33, 1), (6000, 90, 130, 131, 0)):
        store = torch.randn(rows * ld + off, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(2)).to(_dt(dt))
        d = store[off:off + rows * ld].view(rows, ld)[:, :dim]
        ids_h = _ids("padded", rows, vocab, rng)
        want, mag, n = _grad64(ids_h, d.float().cpu().numpy(), vocab, 1.0)
        ws = torch.full((mb.embedding_bwd_workspace_bytes(rows, dim, vocab),), 255, dtype=torch.uint8, device=cuda_dev)
        for _ in range(2):
            got = mb.embedding_bwd(torch.from_numpy(ids_h).to(cuda_dev), d, vocab, workspace=ws)
            assert (np.abs(got.double().cpu().numpy() - want) <= (n + 2) * 2.0 ** -24 * mag).all()


def test_gradient_agrees_with_differences_of_the_lookup(cuda_dev):
    """A loss that is linear in the rows: its change with one entry of the table, in 64 bits, is the entry's gradient."""
    import torch

    import mamba_rs_b200 as mb
    rng = np.random.default_rng(8)
    ids_h = _ids("zipf", 200, 12, rng)
    ids = torch.from_numpy(ids_h).to(cuda_dev)
    w = torch.randn(200, 6, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(8))
    table = torch.randint(-8, 8, (12, 6), device=cuda_dev).float()
    got = mb.embedding_bwd(ids, w, 12, scale=0.5).double()
    loss = lambda t: (mb.embedding_fwd(t, ids, scale=0.5).double() * w.double()).sum()  # noqa: E731
    for v, c in ((0, 0), (1, 5), (11, 3)):
        up, down = table.clone(), table.clone()
        up[v, c] += 1.0    # (whole numbers: the lookups are exact)
        down[v, c] -= 1.0
        n = (ids_h == v).sum()
        mag = float(w[ids == v, c].abs().double().sum()) * 0.5
        assert abs(float((loss(up) - loss(down)) / 2 - got[v, c])) <= (n + 2) * 2.0 ** -24 * mag + 1e-12


def test_no_rows_and_refusals(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    t = torch.ones(5, 8, device=cuda_dev)
    none = torch.empty(0, dtype=torch.int32, device=cuda_dev)
    ids = torch.zeros(4, dtype=torch.int32, device=cuda_dev)
    assert mb.embedding_fwd(t, none).shape == (0, 8)
    assert not mb.embedding_bwd(none, t[:0], 5).any()
    assert torch.equal(mb.embedding_bwd(none, t[:0], d_table=t.clone()), t)
    for bad in (lambda: mb.embedding_fwd(t, ids.long()), lambda: mb.embedding_fwd(t.t(), ids),
                lambda: mb.embedding_fwd(t.double(), ids), lambda: mb.embedding_bwd(ids, t[:4].double(), 5),
                lambda: mb.embedding_bwd(ids, t[:4], d_table=t.half())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: mb.embedding_fwd(t, ids, out=t[:3]), lambda: mb.embedding_bwd(ids, t[:3], 5), lambda: mb.embedding_bwd(ids, t[:4]),
                lambda: mb.embedding_bwd(ids, t[:4], 6, d_table=t)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="embedding_fwd"):
        mb.embedding_fwd(t, ids, out_dtype=torch.float16)  # an f32 table comes out as f32
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        mb.embedding_fwd(t.cpu(), ids)
    if mb.embedding_bwd_workspace_bytes(9000, 8, 5):
        with pytest.raises(RuntimeError, match="workspace"):
            mb.embedding_bwd(torch.zeros(9000, dtype=torch.int32, device=cuda_dev), torch.ones(9000, 8, device=cuda_dev), 5,
                             workspace=torch.empty(0, dtype=torch.uint8, device=cuda_dev))


def test_rows_that_are_one_in_memory_are_refused(cuda_dev):
    """An expanded tensor has a row stride of 0: it is no matrix of that many rows for the kernels."""
    import torch

    import mamba_rs_b200 as mb
    one, ids = torch.ones(1, 8, device=cuda_dev), torch.zeros(4, dtype=torch.int32, device=cuda_dev)
    for bad in (lambda: mb.embedding_fwd(one.expand(5, 8), ids), lambda: mb.embedding_bwd(ids, one.expand(4, 8), 5)):
        with pytest.raises(RuntimeError, match="bad dims"):
            bad()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [4, 129, 520])
@pytest.mark.parametrize("lengths", [(9000,), (1, 1023, 1025, 31, 2048, 33), (700, 5000, 3, 1100, 1100, 64), (40000, 513, 30000)])
def test_tokens_that_reach_over_many_runs(cuda_dev, dt, dim, lengths):
    """Sums of small whole numbers are exact in f32 in any order: rows of one token in thousands, in order and shuffled."""
    import torch

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(dim + len(lengths))
    tokens = torch.tensor([5, 17, 18, 400, 401, 650][: len(lengths)], device=cuda_dev)
    ids = torch.repeat_interleave(tokens, torch.tensor(lengths, device=cuda_dev)).int()
    d = torch.randint(-3, 4, (ids.numel(), dim), device=cuda_dev, generator=g).to({"f32": torch.float32, "bf16": torch.bfloat16}[dt])
    for order in (torch.arange(ids.numel(), device=cuda_dev), torch.randperm(ids.numel(), device=cuda_dev, generator=g)):
        i, x = ids[order].contiguous(), d[order].contiguous()
        want = torch.zeros(700, dim, dtype=torch.float64, device=cuda_dev).index_add_(0, i.long(), x.double())
        assert torch.equal(mb.embedding_bwd(i, x, 700).double(), want)
        start = torch.ones(700, dim, device=cuda_dev)
        assert torch.equal(mb.embedding_bwd(i, x, d_table=start).double(), want + 1)
