"""Group norm: a group that holds a NaN says so everywhere, whatever form of the kernels its sizes take."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
# rows; rows between vectors; whole samples in one kernel (as a few and as many rows); samples in two kernels; groups wider than a block
@pytest.mark.parametrize("N,S,C,G", [(300, 1, 256, 4), (300, 1, 66, 6), (6, 3, 256, 8), (6, 200, 256, 8), (2, 4000, 64, 2), (2, 40, 6000, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_groups_results_and_statistics(cuda_dev, dt, N, S, C, G, bad):
    import torch

    import mamba_rs_b200 as mb
    from retention_ref import DT
    g = torch.Generator(cuda_dev).manual_seed(C)
    x = torch.randn(N, S, C, device=cuda_dev, generator=g).to(DT[dt])
    w, b = (torch.randn(C, device=cuda_dev, generator=g) for _ in range(2))
    y0, stats0 = mb.group_norm_fwd(x, w, b, G)
    n, c = N // 2, C - 2
    x[n, S // 2, c] = bad
    y, stats = mb.group_norm_fwd(x, w, b, G)
    group = slice((G - 1) * (C // G), C)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[n, :, group] = True
    assert torch.equal(y[~hit], y0[~hit])
    assert not torch.isfinite(stats[0, n, G - 1]) and torch.isnan(stats[1, n, G - 1])
    assert torch.isnan(y[hit]).all()
    clean = torch.ones_like(stats, dtype=torch.bool)
    clean[:, n, G - 1] = False
    assert torch.equal(stats[clean], stats0[clean])
