"""What the ends of a language model and its gated recurrence cost: the token table's lookup and gradient, the log
probabilities of given tokens, and the gated linear scan with its gradient and its single step.

Each case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one call of one
operator.  With `own` false the operators are computed in elementary torch operations in 32 bits, with `own` true by this
framework's entry points.  Seven kinds:

  embed_fwd   out[r] = scale * table[ids[r]]                       (an id outside the table: a row of zeros)
  embed_bwd   d_table[v] = scale * sum over r with ids[r] = v of d_out[r]
  logp        of each row of logits / temperature: log sum exp in two parts (largest logit, log of the sum of exponentials
              beside it), log p(target), entropy, the k most likely tokens
  logp_bwd    gradient of the logits from those of log p(target) and of the entropy
  scan        u = sigmoid(-f), h_t = h_{t-1} + u_t (x_t - h_{t-1}), y_t = h_t * SiLU(z_t)
  scan_bwd    gradients of x, f, z and of the state that entered, from those of y and of the state that left
  step        the scan's single step, one token per sequence
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
SAVE = 64  # steps between the states that the scan's forward keeps for its backward


def listed():
    return [
        # decoding: the embedding rows of one token for each of 8 sequences, 130m architecture (d_model 768)
        dict(name="embed_fwd_r8_d768", kind="embed_fwd", rows=8, vocab=50280, dim=768, ids="zipf", scale=27.712812921102035, dtype="bf16"),
        # a pre-training shard of two sequences of 8192 tokens at the 2.8b width
        dict(name="embed_fwd_r16384_d2560", kind="embed_fwd", rows=16384, vocab=50280, dim=2560, ids="zipf", scale=1.0, dtype="bf16"),
        # the table's gradient in a training step of 32 tokens of a small f32 model
        dict(name="embed_bwd_r32_d128_f32", kind="embed_bwd", rows=32, vocab=1000, dim=128, ids="zipf", scale=1.0, dtype="f32"),
        # 16 sequences of 2048 tokens, a third of them padding (one id for all of it, and some ids that do not count)
        dict(name="embed_bwd_r32768_d768", kind="embed_bwd", rows=32768, vocab=50280, dim=768, ids="padded", scale=27.712812921102035, dtype="f32"),
        # serving: the sampled token's log probability and 20 alternatives for 8 sequences
        dict(name="logp_r8_top20", kind="logp", rows=8, vocab=50280, top=20, temperature=1.0, masked="none", dtype="bf16"),
        # scoring: every position of a batch of prompts, with 5 alternatives
        dict(name="logp_r4096_top5", kind="logp", rows=4096, vocab=50280, top=5, temperature=1.0, masked="none", dtype="bf16"),
        # constrained decoding in f32 at an odd vocabulary: half of the tokens are ruled out, in some rows all of them
        dict(name="logp_r1021_v50277_f32", kind="logp", rows=1021, vocab=50277, top=1, temperature=0.7, masked="half", dtype="f32"),
        # a policy-gradient step: gradient of the log probabilities and of the entropy bonus
        dict(name="logp_bwd_r4096", kind="logp_bwd", rows=4096, vocab=50280, temperature=1.0, masked="none", dtype="bf16"),
        # decoding: one token for each of 8 sequences through one layer (d_inner 1536)
        dict(name="step_b8_d1536", kind="step", B=8, T=1, D=1536, z=True, dtype="bf16"),
        # one layer over a training batch
        dict(name="scan_b16_t2048_d1536", kind="scan", B=16, T=2048, D=1536, z=True, dtype="bf16"),
        # one layer over a single long document: few channels, a long axis of odd length
        dict(name="scan_b1_t32749_d768", kind="scan", B=1, T=32749, D=768, z=True, dtype="bf16"),
        # the training batch's backward
        dict(name="scan_bwd_b16_t2048_d1536", kind="scan_bwd", B=16, T=2048, D=1536, z=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the kinds above; sizes beyond the largest listed case's are drawn again."""
    kind = rng.choice(("embed_fwd", "embed_bwd", "logp", "logp_bwd", "step", "scan", "scan_bwd"))
    while True:
        c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
        if kind.startswith("embed"):
            dim = 8 * _log(rng, 8, 320) if rng.random() < 0.8 else _log(rng, 33, 2560) | 1
            c.update(rows=_log(rng, 1, 65536), vocab=_log(rng, 500, 50280), dim=dim, ids=rng.choice(("zipf", "uniform", "padded")),
                     scale=rng.choice((1.0, math.sqrt(dim))))
        elif kind.startswith("logp"):
            V = 8 * _log(rng, 62, 6285) if rng.random() < 0.7 else _log(rng, 500, 50280) | 1
            c.update(rows=_log(rng, 1, 8192), vocab=V, temperature=rng.choice((1.0, 1.0, 0.7, 1.3)), masked=rng.choice(("none", "none", "half")))
            if kind == "logp":
                c.update(top=rng.choice((0, 1, 5, 20, 32)))
        else:
            D = 8 * _log(rng, 8, 640) if rng.random() < 0.8 else _log(rng, 33, 5120) | 1
            c.update(B=_log(rng, 1, 64 if kind == "step" else 16), T=1 if kind == "step" else _log(rng, 2, 65536), D=D, z=rng.random() < 0.75)
        if work(c)["bytes"] <= (4.4e8 if kind in ("logp", "scan") else 7.0e8):
            return c


# ---------------------------------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _spread(vocab):
    """Shares of a vocabulary's tokens in running text, the frequent ones first."""
    p = 1.0 / (torch.arange(vocab, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _ids(c, rows, dev, g):
    V = c["vocab"]
    u = torch.rand(rows, device=dev, generator=g, dtype=torch.float64)
    if c["ids"] == "uniform":
        return (u * V).int().clamp_(0, V - 1)
    ids = torch.searchsorted(_spread(V).cumsum(0).to(dev), u).clamp_(0, V - 1).int()
    if c["ids"] == "padded":  # the last third is padding, and every 97th row does not count
        ids[rows - rows // 3:] = 0
        ids[13::97] = -1
    return ids


def _logits(c, dev, g):
    """Logits of a trained head: a bell with a few tokens that stand out."""
    R, V = c["rows"], c["vocab"]
    l = torch.randn(R, V, device=dev, generator=g).mul_(2.0)
    out = torch.randint(0, V, (R, 8), device=dev, generator=g)
    l.scatter_add_(1, out, 3.0 + 3.0 * torch.rand(R, 8, device=dev, generator=g))
    if c["masked"] == "half":
        l[torch.rand(R, V, device=dev, generator=g) < 0.5] = -math.inf
        l[5::97] = -math.inf
    targets = torch.where(torch.rand(R, device=dev, generator=g) < 0.5, out[:, 0], torch.randint(0, V, (R,), device=dev, generator=g)).int()
    targets[7::61] = -1  # prompt and padding positions
    return l.to(_DT[c["dtype"]]), targets


def _states(u, x, h0):
    """States that enter each block of SAVE steps [B, blocks, D], from f32 gates and inputs."""
    h = _recurrence(1.0 - u, u * x, h0)
    return torch.cat([h0[:, None], h[:, SAVE - 1:-1:SAVE]], 1).contiguous()


def prepare(case, seed):
    c, kind = case, case["kind"]
    dev, dt = _device(), _DT[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    s = dict(kind=kind)
    if kind == "embed_fwd":
        s.update(table=rn(c["vocab"], c["dim"]).mul_(0.02).to(dt), ids=_ids(c, c["rows"], dev, g), scale=c["scale"])
    elif kind == "embed_bwd":
        s.update(d_out=rn(c["rows"], c["dim"]).mul_(1e-3).to(dt), ids=_ids(c, c["rows"], dev, g), vocab=c["vocab"], scale=c["scale"])
    elif kind in ("logp", "logp_bwd"):
        logits, targets = _logits(c, dev, g)
        s.update(logits=logits, targets=targets, temperature=c["temperature"], top=c.get("top", 0))
        if kind == "logp_bwd":  # what the forward left, and the gradients of its results
            l = logits.float()
            m = l.amax(1)
            d = (l - torch.where(torch.isinf(m), 0.0, m)[:, None]) / c["temperature"]
            e = torch.exp(d)
            S = torch.where(torch.isinf(m), 1.0, e.sum(1))
            s["lse"] = torch.stack([m, torch.log(S)])
            s["entropy"] = torch.log(S) - (e * torch.where(e > 0, d, 0.0)).sum(1) / S
            s.update(d_logprob=rn(c["rows"]).div_(c["rows"]), d_entropy=torch.full((c["rows"],), 0.01 / c["rows"], device=dev))
    else:
        B, T, D, w = c["B"], c["T"], c["D"], 3 if c["z"] else 2
        # one projection gives the input, the forget gate and the output gate, side by side
        proj = rn(B, T, w * D)
        rate = torch.exp(torch.rand(D, device=dev, generator=g) * math.log(500.0) + math.log(1e-3))  # 1/rate steps of memory
        proj[..., D:2 * D] += torch.log1p(-rate) - torch.log(rate)
        proj = proj.to(dt)
        view = lambda t: [t[..., i * D:(i + 1) * D] for i in range(w)] + [None] * (3 - w)  # noqa: E731
        s["x"], s["f"], s["z"] = view(proj if kind != "step" else proj[:, 0])
        s["h0"] = 0.3 * rn(B, D)
        if kind == "scan_bwd":
            s["dy"], s["d_last"] = rn(B, T, D).to(dt), rn(B, D)
            s["states"] = _states(torch.sigmoid(-s["f"].float()), s["x"].float(), s["h0"])
            s["d_x"], s["d_f"], s["d_z"] = view(torch.empty_like(proj))
        else:
            s["h_last"] = torch.empty(B, D, device=dev)
    return s


# ---------------------------------------------------------------------------------------------------
# one call
# ---------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mamba_rs_b200 as mb
    kind = s["kind"]
    if kind == "embed_fwd":
        return mb.embedding_fwd(s["table"], s["ids"], scale=s["scale"])
    if kind == "embed_bwd":
        return mb.embedding_bwd(s["ids"], s["d_out"], s["vocab"], scale=s["scale"])
    if kind == "logp":
        return mb.token_logprobs(s["logits"], s["targets"], top=s["top"], temperature=s["temperature"])
    if kind == "logp_bwd":
        return mb.token_logprobs_bwd(s["logits"], s["targets"], s["lse"], s["entropy"], s["d_logprob"], s["d_entropy"],
                                     temperature=s["temperature"])
    if kind == "step":
        y = mb.gated_scan_step(s["x"], s["f"], s["h0"], s["z"], h_last=s["h_last"])
        return dict(y=y, h_last=s["h_last"])
    if kind == "scan":
        y = mb.gated_scan_fwd(s["x"], s["f"], s["z"], h0=s["h0"], h_last=s["h_last"])
        return dict(y=y, h_last=s["h_last"])
    return mb.gated_scan_bwd(s["x"], s["f"], s["dy"], s["states"], s["z"], d_last=s["d_last"], d_x=s["d_x"], d_f=s["d_f"], d_z=s["d_z"])


def _recurrence(a, b, h0):
    """h_t = a_t h_{t-1} + b_t over dimension 1: spans of 1, 2, 4, ... steps are joined, so it takes log2(T) passes over
    whole tensors (step by step it would be T launches)."""
    b = b.clone()
    b[:, 0] += a[:, 0] * h0
    n = 1
    while n < a.shape[1]:
        b[:, n:] = b[:, n:] + a[:, n:] * b[:, :-n]
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _run_plain(s):
    kind = s["kind"]
    if kind == "embed_fwd":
        ids = s["ids"].long()
        ok = (ids >= 0) & (ids < s["table"].shape[0])
        return torch.where(ok[:, None], s["table"][torch.where(ok, ids, 0)].float() * s["scale"], 0.0)
    if kind == "embed_bwd":
        ids = s["ids"].long()
        ok = (ids >= 0) & (ids < s["vocab"])
        rows = torch.where(ok[:, None], s["d_out"].float() * s["scale"], 0.0)
        return torch.zeros(s["vocab"], rows.shape[1], device=rows.device).index_add_(0, torch.where(ok, ids, 0), rows)
    if kind in ("logp", "logp_bwd"):
        l = s["logits"].float()
        V, t = l.shape[1], s["targets"].long()
        ok = (t >= 0) & (t < V)
        t = torch.where(ok, t, 0)[:, None]
        if kind == "logp":
            m = l.amax(1, keepdim=True)
            d = (l - torch.where(torch.isinf(m), 0.0, m)) / s["temperature"]  # (a row with nothing left is -inf throughout)
            e = torch.exp(d)
            S = torch.where(torch.isinf(m), 1.0, e.sum(1, keepdim=True))
            log_s = torch.log(S)
            H = log_s - (e * torch.where(e > 0, d, 0.0)).sum(1, keepdim=True) / S
            out = dict(lse=torch.stack([m[:, 0], log_s[:, 0]]), entropy=H[:, 0],
                       logprob=torch.where(ok, (d.gather(1, t) - log_s)[:, 0], 0.0))
            if s["top"]:
                i = torch.sort(l, dim=1, descending=True, stable=True)[1]
                out.update(top_ids=i[:, :s["top"]].int(), top_logprobs=d.gather(1, i[:, :s["top"]]) - log_s)
            return out
        m, log_s = s["lse"]
        some = ~torch.isinf(m)
        logp = torch.where(some[:, None], (l - m[:, None]) / s["temperature"] - log_s[:, None], -math.inf)
        p = torch.exp(logp)
        g = torch.where(ok & some, s["d_logprob"], 0.0)[:, None]
        d = -p * (g + s["d_entropy"][:, None] * torch.where(p > 0, logp + s["entropy"][:, None], 0.0))
        d = d.scatter_add(1, t, g)
        return (d / s["temperature"]).to(s["logits"].dtype)
    dt = s["x"].dtype
    x, f = s["x"].float(), s["f"].float()
    z = s["z"].float() if s["z"] is not None else None
    u = torch.sigmoid(-f)
    if kind == "step":
        h = s["h0"] + u * (x - s["h0"])
        y = h * z * torch.sigmoid(z) if z is not None else h
        return dict(y=y.to(dt), h_last=h)
    h = _recurrence(torch.sigmoid(f), u * x, s["h0"])
    if kind == "scan":
        y = h * z * torch.sigmoid(z) if z is not None else h
        return dict(y=y.to(dt), h_last=h[:, -1].clone())
    dy = s["dy"].float()
    before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    a = torch.sigmoid(f)
    out = {}
    if z is not None:
        sz = torch.sigmoid(z)
        out["d_z"] = (dy * h * sz * (1.0 + z * (1.0 - sz))).to(dt)
        dy = dy * z * sz
    # g_t = dy_t + a_{t+1} g_{t+1}: the same recurrence from the end
    later = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _recurrence(later.flip(1), dy.flip(1), s["d_last"]).flip(1)
    out.update(d_x=(g * u).to(dt), d_f=(g * (before - x) * a * u).to(dt), d_h0=g[:, 0] * a[:, 0])
    return out


# ---------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "embed_fwd":
        table = torch.cat([s["table"].double() * case["scale"], torch.zeros(1, case["dim"], device=s["table"].device, dtype=torch.float64)])
        ids = s["ids"].long()
        ids[(ids < 0) | (ids >= case["vocab"])] = case["vocab"]
        return table[ids]
    if kind == "embed_bwd":
        ids = s["ids"].long()
        ids[(ids < 0) | (ids >= case["vocab"])] = case["vocab"]
        d = torch.zeros(case["vocab"] + 1, case["dim"], device=ids.device, dtype=torch.float64)
        return d.index_add_(0, ids, s["d_out"].double() * case["scale"])[:-1]
    if kind in ("logp", "logp_bwd"):
        parts = [_exact_rows(case, s, r, min(r + 256, case["rows"])) for r in range(0, case["rows"], 256)]
        if kind == "logp_bwd":
            return torch.cat(parts)
        out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
        return {**out, "lse": out["lse"].T.contiguous()}
    # step by step
    B, T, D = case["B"], case["T"], case["D"]
    rows = lambda t: None if t is None else t.double().reshape(B, T, D)  # noqa: E731
    x, f, z = rows(s["x"]), rows(s["f"]), rows(s["z"])
    a, u = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
    h, hs = s["h0"].double(), torch.empty_like(x)
    for t in range(T):
        h = a[:, t] * h + u[:, t] * x[:, t]
        hs[:, t] = h
    gate = None if z is None else z / (1.0 + torch.exp(-z))
    if kind != "scan_bwd":
        y = hs if z is None else hs * gate
        return dict(y=y[:, 0] if kind == "step" else y, h_last=h)
    dy = s["dy"].double()
    out = {}
    if z is not None:
        q = 1.0 / (1.0 + torch.exp(-z))
        out["d_z"] = dy * hs * (q + z * q * (1.0 - q))
        dy = dy * gate
    g, dx, df = s["d_last"].double(), torch.empty_like(x), torch.empty_like(x)
    for t in range(T - 1, -1, -1):
        g = g + dy[:, t]
        dx[:, t] = g * u[:, t]
        df[:, t] = g * ((hs[:, t - 1] if t else s["h0"].double()) - x[:, t]) * a[:, t] * u[:, t]
        g = g * a[:, t]
    out.update(d_x=dx, d_f=df, d_h0=g)
    return out


def _exact_rows(case, s, r0, r1):
    l, t = s["logits"][r0:r1].double() / case["temperature"], s["targets"][r0:r1].long()
    counted = (t >= 0) & (t < case["vocab"])
    lse = torch.logsumexp(l, 1)
    empty, m = torch.isinf(lse), l.amax(1)
    p = torch.softmax(l, 1).nan_to_num(0.0)
    logp = (l - lse[:, None]).masked_fill(empty[:, None], -math.inf)
    H = -(p * logp.masked_fill(p == 0, 0.0)).sum(1)
    hot = torch.zeros_like(l)
    hot[counted, t[counted]] = 1.0
    if case["kind"] == "logp":
        own_logp = logp.gather(1, t.clamp(min=0)[:, None])[:, 0].masked_fill(~counted, 0.0)
        out = dict(lse=torch.stack([m * case["temperature"], (lse - m).masked_fill(empty, 0.0)], 1), entropy=H, logprob=own_logp)
        if case["top"]:
            order = torch.argsort(-l, dim=1, stable=True)[:, :case["top"]]
            out.update(top_ids=order.int(), top_logprobs=logp.gather(1, order))
        return out
    d = s["d_logprob"][r0:r1, None].double() * (hot - p) * (counted & ~empty)[:, None]
    d = d - s["d_entropy"][r0:r1, None].double() * p * (logp.masked_fill(p == 0, 0.0) + H[:, None])
    return d / case["temperature"]


# ---------------------------------------------------------------------------------------------------
# what a call cannot do without
# ---------------------------------------------------------------------------------------------------

def _distinct(c):
    """Rows of the table that are expected to occur."""
    R, V = c["rows"], c["vocab"]
    if c["ids"] == "uniform":
        return V * -math.expm1(R * math.log1p(-1.0 / V))
    n = R if c["ids"] == "zipf" else R - R // 3
    return float(-torch.expm1(n * torch.log1p(-_spread(V))).sum())


def work(case):
    c, kind, e = case, case["kind"], _SIZE[case["dtype"]]
    if kind == "embed_fwd":
        R, d = c["rows"], c["dim"]
        return {"bytes": 4.0 * R + _distinct(c) * d * e + 4.0 * R * d, "flops": 1.0 * R * d}
    if kind == "embed_bwd":
        R, d = c["rows"], c["dim"]
        return {"bytes": 4.0 * R + R * d * e + 4.0 * c["vocab"] * d, "flops": 2.0 * R * d}
    if kind in ("logp", "logp_bwd"):
        n = c["rows"] * c["vocab"]
        if kind == "logp":
            return {"bytes": e * n + c["rows"] * (20.0 + 8.0 * c["top"]), "flops": 6.0 * n}
        return {"bytes": 2.0 * e * n + c["rows"] * 24.0, "flops": 8.0 * n}
    n, b = c["B"] * c["T"] * c["D"], c["B"] * c["D"]
    gates = 3 if c["z"] else 2
    if kind != "scan_bwd":
        return {"bytes": e * n * (gates + 1.0) + 8.0 * b, "flops": 14.0 * n}
    return {"bytes": e * n * (2.0 * gates + 1.0) + 4.0 * b * ((c["T"] + SAVE - 1) // SAVE + 2), "flops": 30.0 * n}
