"""The token table, token log probabilities and the gated scan launch asynchronously on the caller's stream, allocate nothing in
the library and keep nothing between calls: a captured sequence of them replays with the eager launches' bits, also on other
inputs, and a side stream's calls do not wait for or disturb the default one's."""
import pytest

pytestmark = pytest.mark.gpu


def _work(mb, torch, s):
    """One call of everything, cut scans, sorted gradients and split rows among them."""
    h = torch.empty_like(s["h0"])
    cs = torch.empty(mb.gated_scan_states(*s["x"].shape), device=h.device)
    out = dict(emb=mb.embedding_fwd(s["table"], s["ids"], scale=3.0), d_table=mb.embedding_bwd(s["ids"], s["d_out"], s["table"].shape[0], scale=3.0),
               few=mb.embedding_bwd(s["ids"][:40], s["d_out"][:40], s["table"].shape[0]),
               y=mb.gated_scan_fwd(s["x"], s["f"], s["z"], h0=s["h0"], h_last=h, chunk_states=cs), h=h, cs=cs)
    out.update(mb.gated_scan_bwd(s["x"], s["f"], out["y"], cs, s["z"], d_last=h))
    out["step"] = mb.gated_scan_step(s["x"][:, 0], s["f"][:, 0], s["h0"], s["z"][:, 0], h_last=torch.empty_like(h))
    for k in ("logits", "short", "many"):
        r = mb.token_logprobs(s[k], s["t"][:s[k].shape[0]], top=7)
        out.update({k + n: v for n, v in r.items()})
        out[k + "d"] = mb.token_logprobs_bwd(s[k], s["t"][:s[k].shape[0]], r["lse"], r["entropy"], r["logprob"], r["entropy"])
    return out


def _inputs(torch, dev, seed):
    g = torch.Generator(dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g).bfloat16()  # noqa: E731
    ids = lambda n, v: torch.randint(0, v, (n,), device=dev, dtype=torch.int32, generator=g)  # noqa: E731
    return dict(table=rn(700, 96), ids=ids(1500, 700), d_out=rn(1500, 96), x=rn(2, 900, 136), f=rn(2, 900, 136), z=rn(2, 900, 136),
                h0=torch.randn(2, 136, device=dev, generator=g), logits=rn(5, 20011) * 3, short=rn(300, 999) * 3, many=rn(700, 9000) * 3, t=ids(700, 999))


def test_captured_calls_replay_with_the_eager_bits(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    s, other = _inputs(torch, cuda_dev, 1), _inputs(torch, cuda_dev, 2)
    eager = [{k: v.clone() for k, v in _work(mb, torch, q).items()} for q in (s, other)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = _work(mb, torch, s)
    for want, inputs in ((eager[0], None), (eager[1], other), (eager[1], None)):
        if inputs is not None:
            for k, v in inputs.items():
                s[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for k, v in want.items():
            assert torch.equal(out[k], v), k
    mb.ffi.default_handle(0).check_status()


def test_calls_on_two_streams_at_once(cuda_dev):
    import torch

    import mamba_rs_b200 as mb
    a, b = _inputs(torch, cuda_dev, 3), _inputs(torch, cuda_dev, 4)
    want = [{k: v.clone() for k, v in _work(mb, torch, q).items()} for q in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i, (st, q) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(st):
                got[i] = _work(mb, torch, q)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        for k, v in w.items():
            assert torch.equal(o[k], v), k
