"""A layer of retention as it is used: queries and keys rotated, linear attention with a decay for each head, every head's output normalised by
itself and gated; forward, backward, prompt and steps; captured, replayed, and on two streams at once.

Each operator is held to the bounds of its own test at what it was given, so those of a run need none of their own.  Where whole runs are compared
(f32), every one of the operators is off by norm_tol of its result's norm and passes on what it is given at no more than four times: the state
that enters keeps every token's output near size one, which bounds what the norm does."""
import pytest

pytestmark = pytest.mark.gpu
DTS = ["f32", "bf16", "f16"]


def make(torch, dev, dt, B=2, T=300, H=4, Hk=2, K=64, V=32, seed=0):
    from retention_ref import DT

    import mamba_rs_b200 as mb
    g = torch.Generator(dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    d = DT[dt]
    return dict(q=rn(B, T, H, K).to(d), k=rn(B, T, Hk, K).to(d), v=rn(B, T, H, V).to(d), z=rn(B, T, H * V).to(d), dy=rn(B, T, H * V).to(d),
                decay=torch.log1p(-torch.exp2(-3.0 - torch.arange(H, device=dev))), w=1.0 + 0.3 * rn(H * V), b=0.3 * rn(H * V),
                state=3.0 * rn(B, H, K, V), positions=torch.arange(T, device=dev, dtype=torch.int32),
                freq=mb.rotary_frequencies(K, device=dev)[0])


def forward(mb, s, state_out=None, at=slice(None)):
    q, k = mb.rotary_fwd(s["q"][:, at], s["k"][:, at], s["positions"][at], s["freq"])
    o = mb.linear_attention_fwd(q, k, s["v"][:, at], s["decay"], state=s["state"], state_out=state_out)
    B, T, H, V = o.shape
    y, stats = mb.group_norm_fwd(o.view(B * T, 1, H * V), s["w"], s["b"], H, z=s["z"][:, at].reshape(B * T, 1, H * V))
    return dict(q=q, k=k, o=o, y=y.view(B, T, H * V), stats=stats)


def backward(mb, s, f):
    B, T, H, V = f["o"].shape
    rows = lambda t: t.reshape(B * T, 1, H * V)  # noqa: E731
    n = mb.group_norm_bwd(rows(s["dy"]), rows(f["o"]), f["stats"], s["w"], s["b"], H, z=rows(s["z"]))
    a = mb.linear_attention_bwd(f["q"], f["k"], s["v"], n["d_x"].view(f["o"].shape), s["decay"], state=s["state"])
    d_q, d_k = mb.rotary_bwd(a["d_q"], a["d_k"], s["positions"], s["freq"])
    return dict(q=d_q, k=d_k, v=a["d_v"], z=n["d_z"], w=n["d_weight"], b=n["d_bias"], state=a["d_state"])


def plain(s):
    """In 64 bits, differentiable: (y, leaves)."""
    import torch

    from retention_ref import group_norm
    x = {n: s[n].double().requires_grad_() for n in ("q", "k", "v", "z", "w", "b", "state")}
    B, T, H, V = s["v"].shape
    angle = (s["positions"].double()[:, None] * s["freq"].double())[None, :, None]

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
    q, k = turn(x["q"]), turn(x["k"]).repeat_interleave(H // x["k"].shape[2], 2)
    lam, S, o = torch.exp(s["decay"].double())[None, :, None, None], x["state"], []
    for t in range(T):
        S = lam * S + k[:, t, :, :, None] * x["v"][:, t, :, None, :]
        o.append(torch.einsum("bhk,bhkv->bhv", q[:, t], S) * q.shape[3] ** -0.5)
    y, _, _ = group_norm(torch.stack(o, 1).reshape(B * T, 1, H * V), x["w"], x["b"], H, 1e-5, None, x["z"].reshape(B * T, 1, H * V))
    return y.view(B, T, H * V), x, S


def test_a_layer_against_64_bits(cuda_dev):
    import torch
    from retention_ref import fro
    from test_linear_attention_gpu import norm_tol

    import mamba_rs_b200 as mb
    s = make(torch, cuda_dev, "f32")
    last = torch.empty_like(s["state"])
    f = forward(mb, s, last)
    y, leaves, S = plain(s)
    tol = 4 * 3 * norm_tol("f32", 64 + 300)
    assert fro(f["y"], y.detach()) <= tol and fro(last, S.detach()) <= tol
    want = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
    got = backward(mb, s, f)
    for (name, _), w in zip(leaves.items(), want):
        assert fro(got[name].view(w.shape), w) <= 2 * tol, name
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("prompt", [1, 40, 257])
def test_a_prompt_and_steps(cuda_dev, dt, prompt):
    """A prompt in one call and the tokens after it one by one, or in one more call, against all of it at once."""
    import torch
    from retention_ref import attention
    from test_linear_attention_gpu import close, state_close

    import mamba_rs_b200 as mb
    s = make(torch, cuda_dev, dt, seed=prompt)
    whole_last, state = torch.empty_like(s["state"]), s["state"].clone()
    whole = forward(mb, s, whole_last)
    head = forward(mb, s, state, slice(0, prompt))
    for n in ("q", "k"):
        assert torch.equal(head[n], whole[n][:, :prompt])
    want, last = attention(whole["q"], whole["k"], s["v"], s["decay"], 64 ** -0.5, s["state"])
    mags, last_mags = attention(whole["q"].abs(), whole["k"].abs(), s["v"].abs(), s["decay"], 64 ** -0.5, s["state"].abs())
    outs = [head["o"]]
    middle = min(prompt + 9, 300)
    for t in range(prompt, middle):
        q, k = mb.rotary_fwd(s["q"][:, t:t + 1], s["k"][:, t:t + 1], s["positions"][t:t + 1], s["freq"])
        assert torch.equal(q[:, 0], whole["q"][:, t]) and torch.equal(k[:, 0], whole["k"][:, t])
        outs.append(mb.linear_attention_step(q[:, 0], k[:, 0], s["v"][:, t], s["decay"], state)[:, None])
    rest = dict(s, state=state)
    outs.append(forward(mb, rest, state, slice(middle, 300))["o"])
    for o in (whole["o"], torch.cat(outs, 1)):
        close(o, want, mags, dt, 64 + 300, 0.0 if dt == "f32" else 2.0)
    for got in (whole_last, state):
        state_close(got, last, last_mags, 300)
    mb.ffi.default_handle(0).check_status()


def _work(mb, torch, s):
    """One call of everything, cut sequences and shared heads among them, with what a user would keep."""
    f = forward(mb, s, last := torch.empty_like(s["state"]))
    out = {"f" + n: v for n, v in f.items()}
    out.update({"d" + n: v for n, v in backward(mb, s, f).items()}, last=last)
    out["step"] = mb.linear_attention_step(f["q"][:, 0], f["k"][:, 0], s["v"][:, 0], s["decay"], s["state"], state_out=torch.empty_like(last))
    out["part"] = mb.linear_attention_fwd(f["q"][:, :31], f["k"][:, :31], s["v"][:, :31], s["decay"])
    out["wide"], out["wide_stats"] = mb.group_norm_fwd(f["o"].flatten(2), s["w"], s["b"], 8, activation="silu")
    out["slab"], _ = mb.group_norm_fwd(f["o"][:1, :40].flatten(2), s["w"], s["b"], 8, activation="gelu")
    out.update({"n" + n: v for n, v in mb.group_norm_bwd(s["dy"], f["o"].flatten(2), out["wide_stats"], s["w"], s["b"], 8, activation="silu").items()})
    return out


SIZES = [dict(), dict(T=5000, B=1, H=2, Hk=1)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_captured_calls_replay_with_the_eager_bits(cuda_dev, dt, sizes):
    import torch

    import mamba_rs_b200 as mb
    s, other = make(torch, cuda_dev, dt, seed=1, **sizes), make(torch, cuda_dev, dt, seed=2, **sizes)
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


@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_calls_on_two_streams_at_once(cuda_dev, sizes):
    import torch

    import mamba_rs_b200 as mb
    a, b = make(torch, cuda_dev, "bf16", seed=3, **sizes), make(torch, cuda_dev, "bf16", seed=4, **sizes)
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
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DTS)
def test_two_graphs_of_one_pool_and_given_scratch(cuda_dev, dt):
    """Graphs that share a memory pool replay one after the other; a scratch that is given serves call after call of a stream."""
    import torch

    import mamba_rs_b200 as mb
    sizes = SIZES[1]
    s, t = make(torch, cuda_dev, dt, seed=5, **sizes), make(torch, cuda_dev, dt, seed=6, **sizes)
    want = [{k: v.clone() for k, v in _work(mb, torch, q).items()} for q in (s, t)]
    pool = torch.cuda.graph_pool_handle()
    outs, graphs = [], []
    for q in (s, t):
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, pool=pool, stream=side):
            outs.append(_work(mb, torch, q))
        graphs.append(graph)
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        for k, v in want[i].items():
            assert torch.equal(outs[i][k], v), k
    B, T, H, K = s["q"].shape
    n = mb.linear_attention_workspace_bytes(B, T, H, K, s["v"].shape[3], Hk=1, backward=True)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda_dev)
    for i, q in enumerate((s, t, s)):
        ws.fill_(255)  # (NaN in every float: nothing of an earlier call is read)
        f = want[i % 2]
        # (the same results asked for: where a state is handed on it is kept in more terms)
        o = mb.linear_attention_fwd(f["fq"], f["fk"], q["v"], q["decay"], state=q["state"], state_out=torch.empty_like(q["state"]), workspace=ws)
        assert torch.equal(o, f["fo"])
        a = mb.linear_attention_bwd(f["fq"], f["fk"], q["v"], torch.ones_like(o), q["decay"], state=q["state"], workspace=ws)
        b = mb.linear_attention_bwd(f["fq"], f["fk"], q["v"], torch.ones_like(o), q["decay"], state=q["state"])
        for name in a:
            assert torch.equal(a[name], b[name]), name
    mb.ffi.default_handle(0).check_status()


@pytest.mark.parametrize("dt", DTS)
def test_in_the_inputs_place(cuda_dev, dt):
    """What the documentation allows: a norm's rows over its input or gate, a rotation over its input, on every path of the norm."""
    import torch
    from retention_ref import DT

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(9)
    for N, S, C, G in ((50, 1, 256, 4), (3, 1, 9000, 2), (2, 40, 64, 8), (1, 9000, 64, 4), (2, 33, 77, 7)):
        x, z = (torch.randn(N, S, C, device=cuda_dev, generator=g).to(DT[dt]) for _ in range(2))
        w = 1.0 + torch.randn(C, device=cuda_dev, generator=g)
        want, stats = mb.group_norm_fwd(x, w, None, G, activation="silu", z=z)
        a, b = x.clone(), z.clone()
        y, s2 = mb.group_norm_fwd(a, w, None, G, activation="silu", z=z, y=a)
        assert y is a and torch.equal(a, want) and torch.equal(s2, stats)
        mb.group_norm_fwd(x, w, None, G, activation="silu", z=b, y=b)
        assert torch.equal(b, want)
        d = mb.group_norm_bwd(z, x, stats, w, None, G, activation="silu", z=z)
        a = x.clone()
        assert torch.equal(mb.group_norm_bwd(z, a, stats, w, None, G, activation="silu", z=z, d_x=a)["d_x"], d["d_x"])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dt", DTS)
def test_a_norms_bad_values_stay_in_their_group(cuda_dev, dt, bad):
    import torch
    from retention_ref import DT

    import mamba_rs_b200 as mb
    g = torch.Generator(cuda_dev).manual_seed(8)
    for N, S, C, G in ((50, 1, 256, 4), (3, 1, 9000, 2), (2, 40, 64, 8), (1, 9000, 64, 4), (5, 1, 77, 7), (2, 33, 77, 7), (2, 2, 64, 32)):
        x, dy = (torch.randn(N, S, C, device=cuda_dev, generator=g).to(DT[dt]) for _ in range(2))
        want, stats = mb.group_norm_fwd(x, None, None, G)
        d = mb.group_norm_bwd(dy, x, stats, None, None, G)
        x2 = x.clone()
        x2[-1, S // 2, C // 2] = bad
        y, s2 = mb.group_norm_fwd(x2, None, None, G)
        hit = torch.zeros(N, S, G, C // G, dtype=torch.bool, device=cuda_dev)
        hit[-1, :, C // 2 // (C // G)] = True
        hit = hit.view(N, S, C)
        assert torch.equal(y[~hit], want[~hit]) and not torch.isfinite(y[hit]).all()
        d2 = mb.group_norm_bwd(dy, x2, s2, None, None, G)
        assert torch.equal(d2["d_x"][~hit], d["d_x"][~hit])
        clean = ~hit[-1, S // 2]
        assert torch.equal(d2["d_weight"][clean], d["d_weight"][clean]) and torch.equal(d2["d_bias"], d["d_bias"])
