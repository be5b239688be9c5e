"""Linear attention, rotation and group norm on rows that lie far apart: offsets of more than 2^31 elements, columns of one wide buffer.  What a
row holds does not depend on where it lies, so the results are those of contiguous tensors, bit for bit."""
import pytest

pytestmark = pytest.mark.gpu
T, WIDE = 33000, 65536  # 33000 x 65536 > 2^31


def test_rows_far_apart(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    for dtype in (torch.bfloat16, torch.float32):
        big = torch.empty(T, WIDE, device=cuda_dev, dtype=dtype)
        g = torch.Generator(cuda_dev).manual_seed(1)
        at = iter(range(0, WIDE, 128))

        def far(t=None, big=big, at=at):
            c = next(at)
            view = big[:, c:c + 128].view(1, T, 2, 64)
            return view if t is None else view.copy_(t)
        q, k, v, do = (torch.randn(1, T, 2, 64, device=cuda_dev, generator=g).to(dtype) for _ in range(4))
        fq, fk, fv, fdo = far(q), far(k), far(v), far(do)
        assert fq.stride(1) == WIDE and (T - 1) * WIDE > 2 ** 31
        decay = torch.tensor([-0.01, -0.5], device=cuda_dev)
        o = mb.linear_attention_fwd(q, k, v, decay)
        assert torch.equal(mb.linear_attention_fwd(fq, fk, fv, decay, o=far()), o)
        want = mb.linear_attention_bwd(q, k, v, do, decay)
        got = mb.linear_attention_bwd(fq, fk, fv, fdo, decay, d_q=far(), d_k=far(), d_v=far())
        for n in want:
            assert torch.equal(got[n], want[n]), n
        freq, positions = mb.rotary_frequencies(64, device=cuda_dev)[0], torch.arange(T, device=cuda_dev, dtype=torch.int32)
        for w, r in zip(mb.rotary_fwd(q, k, positions, freq), mb.rotary_fwd(fq, fk, positions, freq, q_out=far(), k_out=far())):
            assert torch.equal(r, w)
        w = torch.randn(128, device=cuda_dev, generator=g)
        for shape in ((T, 1, 128), (1, T, 128), (T // 3, 3, 128)):
            rows = lambda t: t.as_strided(shape, (t.stride(1) * shape[1], t.stride(1), 1))  # noqa: E731, B023
            y, stats = mb.group_norm_fwd(rows(q), w, w, 4, activation="silu", z=rows(k))
            fy, fstats = mb.group_norm_fwd(rows(fq), w, w, 4, activation="silu", z=rows(fk), y=rows(far()))
            assert torch.equal(fy, y) and torch.equal(fstats, stats)
            want = mb.group_norm_bwd(rows(do), rows(q), stats, w, w, 4, activation="silu", z=rows(k))
            got = mb.group_norm_bwd(rows(fdo), rows(fq), stats, w, w, 4, activation="silu", z=rows(fk), d_x=rows(far()), d_z=rows(far()))
            for n in want:
                assert torch.equal(got[n], want[n]), n
        del big, fq, fk, fv, fdo, got, fy
    mb.ffi.default_handle(0).check_status()
