"""The operators together: the example's language model against torch autograd in 64 bits, its scores against its steps, and
GpuMambaLM.score against the engine's own logits."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("gated_lm", os.path.join(ROOT, "examples", "gated_lm.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _loss64(lm, ids, bonus):
    """The same model in torch operations in 64 bits, step by step; returns the loss and the gradients."""
    import torch
    p = {k: v.double().clone().requires_grad_() for k, v in lm.p.items()}
    norm = lambda x, w: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w  # noqa: E731
    inp, tgt = ids[:, :-1].long(), ids[:, 1:].long()
    res = p["table"][inp] * lm.scale
    for i in range(lm.layers):
        x, f, z = (norm(res, p[f"norm{i}"]) @ p[f"in{i}"]).split(lm.D, 2)
        h, ys = torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            a = torch.sigmoid(f[:, t])
            h = a * h + (1 - a) * x[:, t]
            ys.append(h * torch.nn.functional.silu(z[:, t]))
        res = res + torch.stack(ys, 1) @ p[f"out{i}"]
    lp = torch.log_softmax(norm(res, p["norm_f"]) @ p["table"].t(), -1)
    loss = -lp.gather(2, tgt[..., None]).mean() - bonus * (-(lp.exp() * lp).sum(-1)).mean()
    loss.backward()
    return loss, {k: v.grad for k, v in p.items()}


def test_gradients_of_the_example_match_autograd(cuda_dev):
    import torch
    lm = _example().GatedLM(vocab=61, d_model=32, d_inner=48, layers=2, dtype=torch.float32, device=cuda_dev)
    ids = torch.randint(0, 61, (2, 151), device=cuda_dev, dtype=torch.int32, generator=torch.Generator(cuda_dev).manual_seed(1))
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        loss = lm.gradients(ids, entropy_bonus=0.1)
        want, grads = _loss64(lm, ids, 0.1)
        assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
        # f32 products and sums over 300 rows: some hundred roundings of 2^-24 a gradient element, of its largest
        for k, g in grads.items():
            assert (lm.g[k].double() - g).abs().max() <= 2e-5 * g.abs().max(), k
        # the same bits again: no sum depends on the order of atomics
        first = lm.grad.clone()
        lm.grad.zero_()
        lm.gradients(ids, entropy_bonus=0.1)
        assert torch.equal(lm.g["table"], first[:61 * 32].view(61, 32))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_the_example_learns_scores_and_generates(cuda_dev, dt):
    import torch
    m = _example()
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[dt]
    lm = m.GatedLM(vocab=40, d_model=64, d_inner=96, layers=2, dtype=dtype, device=cuda_dev, seed=3)
    text = torch.arange(0, 400, device=cuda_dev, dtype=torch.int32) * 7 % 23
    batch = torch.stack([text[i:i + 101] for i in range(0, 64, 8)])
    losses = [float(lm.train_step(batch, entropy_bonus=1e-3)) for _ in range(60)]
    assert losses[-1] < 0.2 * losses[0] and np.isfinite(losses).all()
    prompt = text[None, :30].contiguous()
    ids, lp, alternatives, alt_lp = lm.generate(prompt, 12, top=4)
    assert torch.equal(ids[0], text[30:42])                # it has learned the sequence
    assert torch.equal(alternatives[..., 0], ids) and torch.equal(alt_lp[..., 0], lp)
    assert (alt_lp[..., :-1] >= alt_lp[..., 1:]).all()
    # what the steps said of the tokens they took is what scoring the whole text says of them, but for the rounding of rows that
    # went through products of other shapes
    s = lm.score(torch.cat([prompt, ids], 1), top=4, rows=17)
    assert s["logprob"].shape == (1, 41) and s["top_ids"].shape == (1, 41, 4)
    assert (s["logprob"][:, 29:] - lp).abs().max() <= (1e-4 if dt == "f32" else 0.1)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_engine_scores_are_the_log_softmax_of_its_logits(cuda_dev, dt):
    import torch

    import mamba_rs_b200 as mb
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[dt]
    w = mb.MambaWeights(mb.MambaConfig(d_model=64, n_layers=2), cuda_dev, dtype=dtype, vocab=501).init_random(5)
    w.tail("master")["embedding"].mul_(30.0)
    w.refresh()
    lm = mb.GpuMambaLM(w, 3)
    ids = torch.randint(0, 501, (3, 40), device=cuda_dev, dtype=torch.int32, generator=torch.Generator(cuda_dev).manual_seed(2))
    got = lm.score(ids, top=3, rows=50)
    assert got["logprob"].shape == got["entropy"].shape == (3, 39) and got["top_ids"].shape == (3, 39, 3)
    lm.backbone.reset()
    hidden = lm.backbone.prefill_sequence(mb.embedding_gather(w.tail()["embedding"], ids[:, :-1].contiguous()).view(3, 39, 64))
    lp = torch.log_softmax((hidden.reshape(-1, 64) @ w.tail()["embedding"].t()).double(), 1).view(3, 39, 501)
    want = lp.gather(2, ids[:, 1:, None].long())[..., 0]
    # (products of other row counts may round a logit differently in the storage dtype)
    assert (got["logprob"] - want).abs().max() <= (1e-3 if dt == "f32" else 0.2)
    lm.backbone.reset()
    first = lm.prefill(ids[:, :-1].contiguous()).float()
    lm.backbone.reset()
    again = lm.score(ids, top=3)
    assert torch.equal(again["top_ids"][:, -1, 0].long(), lp[:, -1].argmax(1)) and first.shape == (3, 501)
    # the state is carried: a text in two windows scores as in one
    lm.backbone.reset()
    one = lm.score(ids[:, :20].contiguous())["logprob"]
    two = lm.score(ids[:, 19:].contiguous())["logprob"]
    assert (torch.cat([one, two], 1) - want).abs().max() <= (1e-3 if dt == "f32" else 0.2)
    with pytest.raises(TypeError):
        lm.score(ids.long())
    with pytest.raises(ValueError):
        lm.score(ids[:, :1].contiguous())
