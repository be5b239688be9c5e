"""What a retention layer's operators cost: linear attention with a decay for each head (whole texts, gradients, single tokens),
the rotation of its queries and keys by position, and the group norm with activation and gate behind it.

Each case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one call of one
operator.  With `own` false the operators are computed in elementary torch operations in 32 bits (angles in 64), with `own` true
by this framework's entry points.  Six kinds:

  step       S <- exp(g_h) S + k v^T,  o = scale S^T q            one token for each sequence, S [K, V] per sequence and head
  attn       the same over whole texts: o_t = scale sum over s <= t of exp(g_h (t - s)) (q_t . k_s) v_s + what a state adds
  attn_bwd   gradients of q, k, v and of the state that entered, from those of o and of the state that left
  rotary     pairs of columns of q and k turned by the angle position * frequency and scaled (inverse: the gradient's way)
  norm       y = act((x - mean) / sqrt(var + eps) * w + b) * SiLU(z), mean and var over a group of channels and a sample's rows
  norm_bwd   gradients of x, z, w and b from that of y
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # decoding, one sequence and a small layer: latency
        dict(name="step_b1_h4", kind="step", B=1, H=4, Hq=4, Hk=4, Hv=4, K=64, V=64, decay="retention", dtype="bf16"),
        # decoding, a full serving batch (32 heads of d_state 128 and headdim 64)
        dict(name="step_b64_h32", kind="step", B=64, H=32, Hq=32, Hk=32, Hv=32, K=128, V=64, decay="retention", dtype="bf16"),
        # a prompt of odd length that goes on from a state and leaves one
        dict(name="attn_b1_t1021_h32_state", kind="attn", B=1, T=1021, H=32, Hq=32, Hk=32, Hv=32, K=128, V=64, decay="retention",
             state=True, dtype="bf16"),
        # one layer over a training batch
        dict(name="attn_b8_t4096_h32", kind="attn", B=8, T=4096, H=32, Hq=32, Hk=32, Hv=32, K=128, V=64, decay="retention", state=False,
             dtype="bf16"),
        # a single long document: few heads, a long axis of odd length, its state kept for what follows
        dict(name="attn_b1_t32749_h12_f16", kind="attn", B=1, T=32749, H=12, Hq=12, Hk=12, Hv=12, K=64, V=64, decay="slopes", state=True,
             dtype="f16"),
        # the training batch's backward
        dict(name="attn_bwd_b8_t4096_h32", kind="attn_bwd", B=8, T=4096, H=32, Hq=32, Hk=32, Hv=32, K=128, V=64, decay="retention",
             state=False, dtype="bf16"),
        # a small f32 model at odd sizes, queries and keys shared by two heads each, text continued from a learned state
        dict(name="attn_bwd_b2_t333_shared_f32", kind="attn_bwd", B=2, T=333, H=6, Hq=3, Hk=3, Hv=6, K=40, V=56, decay="slopes", state=True,
             dtype="f32"),
        # decoding at far positions, 8 sequences
        dict(name="rotary_b8_t1_far", kind="rotary", B=8, T=1, H=32, Hk=32, D=128, R=128, interleaved=False, inverse=False, far=True,
             scaling="yarn", dtype="bf16"),
        # a training batch, half of each head turned
        dict(name="rotary_b8_t4096_part", kind="rotary", B=8, T=4096, H=32, Hk=32, D=128, R=64, interleaved=True, inverse=False, far=False,
             scaling="none", dtype="bf16"),
        # behind the attention: one group for each head of each token, gated (32 heads of 64)
        dict(name="norm_n32768_c2048_gated", kind="norm", N=32768, S=1, C=2048, G=32, act="none", gate=True, dtype="bf16"),
        # convolution features of a small f32 model: groups over a sample's whole length
        dict(name="norm_n3_s1021_c768_silu_f32", kind="norm", N=3, S=1021, C=768, G=32, act="silu", gate=False, dtype="f32"),
        # the gated norm's backward
        dict(name="norm_bwd_n32768_c2048_gated", kind="norm_bwd", N=32768, S=1, C=2048, G=32, act="none", gate=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the kinds above; sizes beyond the largest listed case's are drawn again."""
    kind = rng.choice(("step", "attn", "attn", "attn_bwd", "attn_bwd", "rotary", "norm", "norm_bwd"))
    while True:
        c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
        if kind in ("step", "attn", "attn_bwd"):
            if rng.random() < 0.8:
                K, V = 8 * _log(rng, 2, 16), 8 * _log(rng, 2, 16)
            else:
                K, V = rng.randint(9, 160), rng.randint(9, 160)
            H, share = rng.choice((1, 2, 4, 8, 12, 16, 32)), rng.choice(("none", "none", "qk", "kv"))
            part = H // rng.choice([d for d in (2, 3, 4, 8, 16) if H % d == 0] or [1])
            c.update(B=_log(rng, 1, 128 if kind == "step" else 8), H=H, Hq=part if share == "qk" else H, Hk=H if share == "none" else part,
                     Hv=part if share == "kv" else H, K=K, V=V, decay=rng.choice(("retention", "slopes", "none")))
            if kind != "step":
                c.update(T=_log(rng, 2, 32768), state=rng.random() < 0.5)
        elif kind == "rotary":
            D = rng.choice((32, 64, 80, 96, 128, 192, 256))
            H = rng.choice((1, 2, 4, 8, 12, 16, 32))
            c.update(B=_log(rng, 1, 16), T=_log(rng, 1, 32768), H=H, Hk=rng.choice([h for h in (1, 2, 4, 8, 12, 16, 32) if H % h == 0]),
                     D=D, R=2 * rng.randint(4, D // 2) if rng.random() < 0.5 else D, interleaved=rng.random() < 0.5,
                     inverse=rng.random() < 0.5, far=rng.random() < 0.3, scaling=rng.choice(("none", "linear", "ntk", "yarn")))
        else:
            per = rng.choice((4, 8, 16, 32, 64, 128)) if rng.random() < 0.8 else rng.randint(3, 97)
            G = rng.choice((1, 4, 8, 16, 32))
            S = 1 if rng.random() < 0.5 else _log(rng, 2, 16384)
            c.update(N=_log(rng, 1, 65536 if S == 1 else 32), S=S, C=per * G, G=G, act=rng.choice(("none", "silu", "gelu")), gate=rng.random() < 0.4)
        w = work(c)
        # elements that come and go, and the plain form's time where the products are in f32
        if w["bytes"] <= 5.5e8 and (not kind.startswith("attn") or c["B"] * c["T"] * c["H"] <= 8 * 4096 * 32):
            return c


# ---------------------------------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")


def _decay(c, dev):
    """Log of each head's decay a token: memories of 32 to 8192 tokens, slopes of 1.4 to 256 tokens, or none."""
    h = torch.arange(c["H"], dtype=torch.float64) / max(c["H"] - 1, 1)
    if c["decay"] == "none":
        return torch.zeros(c["H"], device=dev)
    d = torch.log1p(-torch.exp2(-5.0 - 8.0 * h)) if c["decay"] == "retention" else -torch.exp2(-0.5 - 7.5 * h)
    return d.float().to(dev)


def _columns(widths, lead, dt, rn):
    """Tensors [*lead, heads, width] as columns of one projection, and the projection."""
    proj = rn(*lead, sum(h * w for h, w in widths)).to(dt)
    out, at = [], 0
    for h, w in widths:
        out.append(proj[..., at:at + h * w].unflatten(-1, (h, w)))
        at += h * w
    return out, proj


def _frequencies(R, scaling):
    """(frequencies of the R / 2 pairs in f64, scale of the rotated columns) for texts 8 times the length trained on (8192)."""
    base, factor, trained = 10000.0, 8.0, 8192
    i = torch.arange(0, R, 2, dtype=torch.float64)
    if scaling == "ntk":
        base *= factor ** (R / max(R - 2, 1))
    f = base ** (-i / R)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":  # fast pairs as they are, slow ones interpolated, a ramp of the pair's index between
        turns = lambda n: R * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(turns(32)), 0), min(math.ceil(turns(1)), R - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    c, kind = case, case["kind"]
    dev, dt = _device(), _DT[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    s = dict(kind=kind)
    if kind in ("step", "attn", "attn_bwd"):
        B, H, K, V = c["B"], c["H"], c["K"], c["V"]
        lead = (B,) if kind == "step" else (B, c["T"])
        widths = [(c["Hq"], K), (c["Hk"], K), (c["Hv"], V)]
        (s["q"], s["k"], s["v"]), proj = _columns(widths, lead, dt, rn)
        s.update(decay=_decay(c, dev), scale=K ** -0.5, state=None, state_out=None, d_state_out=None)
        if kind == "step" or c["state"]:
            s["state"], s["state_out"] = rn(B, H, K, V), torch.empty(B, H, K, V, device=dev)
        if kind == "attn_bwd":
            s["do"] = rn(B, c["T"], H, V).to(dt)
            if c["state"]:
                s["d_state_out"] = rn(B, H, K, V)
            # the gradients are columns of the projection's
            d_proj, at = torch.empty_like(proj), 0
            for n, (h, w) in zip(("d_q", "d_k", "d_v"), widths):
                s[n] = d_proj[..., at:at + h * w].unflatten(-1, (h, w))
                at += h * w
    elif kind == "rotary":
        B, T = c["B"], c["T"]
        (s["q"], s["k"]), _ = _columns([(c["H"], c["D"]), (c["Hk"], c["D"])], (B, T), dt, rn)
        start = torch.randint(500000, 1000000, (B, 1), device=dev, generator=g) if c["far"] else torch.zeros(B, 1, device=dev, dtype=torch.long)
        s["positions"] = (start + torch.arange(T, device=dev)).int()
        freq, s["scale"] = _frequencies(c["R"], c["scaling"])
        s.update(inv_freq=freq.float().to(dev), interleaved=c["interleaved"], inverse=c["inverse"])
    else:
        N, S, C, G = c["N"], c["S"], c["C"], c["G"]
        # channels of their own means and sizes
        s["x"] = (rn(N, S, C) * (0.5 + torch.rand(C, device=dev, generator=g)) + 0.5 * rn(C)).to(dt)
        s["z"] = rn(N, S, C).to(dt) if c["gate"] else None
        s.update(weight=1.0 + 0.1 * rn(C), bias=0.1 * rn(C), groups=G, eps=1e-5, act=None if c["act"] == "none" else c["act"])
        if kind == "norm_bwd":
            s["dy"] = rn(N, S, C).to(dt)
            x = s["x"].float().view(N, S, G, C // G)  # what the forward left
            mean = x.mean((1, 3), keepdim=True)
            var = (x - mean).square().mean((1, 3))
            s["stats"] = torch.stack([mean[:, 0, :, 0], torch.rsqrt(var + s["eps"])])
    return s


# ---------------------------------------------------------------------------------------------------
# one call
# ---------------------------------------------------------------------------------------------------

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mamba_rs_b200 as mb
    kind = s["kind"]
    if kind == "step":
        o = mb.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], scale=s["scale"], state_out=s["state_out"])
        return dict(o=o, state_out=s["state_out"])
    if kind == "attn":
        o = mb.linear_attention_fwd(s["q"], s["k"], s["v"], s["decay"], scale=s["scale"], state=s["state"], state_out=s["state_out"])
        return dict(o=o) if s["state"] is None else dict(o=o, state_out=s["state_out"])
    if kind == "attn_bwd":
        return mb.linear_attention_bwd(s["q"], s["k"], s["v"], s["do"], s["decay"], scale=s["scale"], state=s["state"],
                                       d_state_out=s["d_state_out"], d_q=s["d_q"], d_k=s["d_k"], d_v=s["d_v"])
    if kind == "rotary":
        f = mb.rotary_bwd if s["inverse"] else mb.rotary_fwd
        q, k = f(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=s["interleaved"], scale=s["scale"])
        return dict(q=q, k=k)
    if kind == "norm":
        y, stats = mb.group_norm_fwd(s["x"], s["weight"], s["bias"], s["groups"], eps=s["eps"], activation=s["act"], z=s["z"])
        return dict(y=y, stats=stats)
    return mb.group_norm_bwd(s["dy"], s["x"], s["stats"], s["weight"], s["bias"], s["groups"], activation=s["act"], z=s["z"])


BLOCK = 128  # steps that the plain form takes at once


def _heads(t, H):
    """[B, T, heads, width] -> [B, H, T, width] in f32, shared heads repeated."""
    return t.float().repeat_interleave(H // t.shape[2], 2).transpose(1, 2)


def _sum_heads(t, like):
    """The gradient of _heads, in like's type."""
    B, H, T, W = t.shape
    n = like.shape[2]
    return t.transpose(1, 2).reshape(B, T, n, H // n, W).sum(3).to(like.dtype)


def _blocks(x, y, z, g, scale, S, reverse):
    """o_t = scale * sum over s <= t of exp(g (t - s)) (x_t . y_s) z_s + exp(g t) x_t S, block by block (t from 1; reverse: from the
    end, with S taken at the last step itself); and the state behind the last step, to which S counts scale-free."""
    T = x.shape[2]
    o, first = [None] * -(-T // BLOCK), True
    for i in (range(len(o) - 1, -1, -1) if reverse else range(len(o))):
        xs, ys, zs = (t[:, :, i * BLOCK:(i + 1) * BLOCK] for t in (x, y, z))
        n = xs.shape[2]
        at = torch.arange(n, device=x.device, dtype=torch.float32)
        if reverse:
            at = n - 1 - at
        d = at[:, None] - at
        L = torch.where(d >= 0, torch.exp(g[:, None, None] * d.clamp(min=0)), 0.0) * scale
        before = 0 if reverse and first else 1  # steps between S and the block's first row
        o[i] = (xs @ ys.transpose(2, 3) * L) @ zs + torch.exp(g[:, None] * (at + before))[..., None] * (xs @ S)
        S = torch.exp(g * (n - 1 + before))[:, None, None] * S + (ys * torch.exp(g[:, None] * (n - 1 - at))[..., None]).transpose(2, 3) @ zs * scale
        first = False
    return torch.cat(o, 2), S


def _run_plain(s):
    kind = s["kind"]
    if kind == "step":
        H, dt = s["decay"].shape[0], s["q"].dtype
        q, k, v = (_heads(s[n][:, None], H)[:, :, 0] for n in ("q", "k", "v"))
        S = torch.exp(s["decay"])[:, None, None] * s["state"] + k[..., None] * v[..., None, :]
        return dict(o=((q[..., None, :] @ S)[..., 0, :] * s["scale"]).to(dt), state_out=S)
    if kind in ("attn", "attn_bwd"):
        H, g, scale = s["decay"].shape[0], s["decay"], s["scale"]
        q, k, v = (_heads(s[n], H) for n in ("q", "k", "v"))
        S = s["state"] if s["state"] is not None else torch.zeros(q.shape[0], H, q.shape[3], v.shape[3], device=q.device)
        if kind == "attn":
            # (the state counts its keys and values as they are: the scale goes with the queries)
            o, last = _blocks(q * scale, k, v, g, 1.0, S, False)
            o = o.transpose(1, 2).to(s["q"].dtype)
            return dict(o=o) if s["state"] is None else dict(o=o, state_out=last)
        do = _heads(s["do"], H)
        d_q, _ = _blocks(do * scale, v, k, g, 1.0, S.transpose(2, 3), False)
        R = s["d_state_out"] if s["d_state_out"] is not None else torch.zeros_like(S)
        d_k, _ = _blocks(v, do, q, g, scale, R.transpose(2, 3), True)
        d_v, d_first = _blocks(k, q, do, g, scale, R, True)
        out = dict(d_q=_sum_heads(d_q, s["q"]), d_k=_sum_heads(d_k, s["k"]), d_v=_sum_heads(d_v, s["v"]))
        if s["state"] is not None:
            out["d_state"] = torch.exp(g)[:, None, None] * d_first
        return out
    if kind == "rotary":
        angle = s["positions"].double()[..., None] * s["inv_freq"].double()
        cos, sin = (f(angle).float()[:, :, None] * s["scale"] for f in (torch.cos, torch.sin))
        if s["inverse"]:
            sin = -sin
        out, half = {}, s["inv_freq"].shape[0]
        for n in ("q", "k"):
            t = s[n].float()
            y = t.clone()
            if s["interleaved"]:
                a, b = t[..., 0:2 * half:2], t[..., 1:2 * half:2]
                y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
            else:
                a, b = t[..., :half], t[..., half:2 * half]
                y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
            out[n] = y.to(s[n].dtype)
        return out
    N, S, C = s["x"].shape
    G, dt = s["groups"], s["x"].dtype
    x, w, b = s["x"].float().view(N, S, G, C // G), s["weight"].view(G, C // G), s["bias"].view(G, C // G)
    if kind == "norm":
        mean = x.mean((1, 3), keepdim=True)
        rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + s["eps"])
        y = _act((x - mean) * rstd * w + b, s["act"]).view(N, S, C)
        if s["z"] is not None:
            z = s["z"].float()
            y = y * z * torch.sigmoid(z)
        return dict(y=y.to(dt), stats=torch.stack([mean[:, 0, :, 0], rstd[:, 0, :, 0]]))
    mean, rstd = (t[:, None, :, None] for t in s["stats"])
    xh, dy, out = (x - mean) * rstd, s["dy"].float(), {}
    v = xh * w + b
    if s["z"] is not None:
        z = s["z"].float()
        sz = torch.sigmoid(z)
        out["d_z"] = (dy * _act(v, s["act"]).view(N, S, C) * sz * (1.0 + z * (1.0 - sz))).to(dt)
        dy = dy * z * sz
    dv = dy.view(N, S, G, C // G) * _act_slope(v, s["act"])
    dh = dv * w
    d_x = (dh - dh.mean((1, 3), keepdim=True) - xh * (dh * xh).mean((1, 3), keepdim=True)) * rstd
    out.update(d_x=d_x.view(N, S, C).to(dt), d_weight=(dv * xh).sum((0, 1)).view(C), d_bias=dv.sum((0, 1)).view(C))
    return out


def _act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v


def _act_slope(v, act):
    if act == "silu":
        q = torch.sigmoid(v)
        return q * (1.0 + v * (1.0 - q))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(v)


# ---------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    if kind in ("step", "attn", "attn_bwd"):
        return _exact_attention(c, s)
    if kind == "rotary":
        angle = s["positions"].double()[:, :, None, None] * s["inv_freq"].double()
        turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if c["inverse"] else angle)
        out, R = {}, c["R"]
        for n in ("q", "k"):
            t = s[n].double()
            pairs = t[..., :R].unflatten(-1, (R // 2, 2) if c["interleaved"] else (2, R // 2))
            if not c["interleaved"]:
                pairs = pairs.transpose(-1, -2)
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            if not c["interleaved"]:
                turned = turned.transpose(-1, -2)
            out[n] = torch.cat([turned.flatten(-2), t[..., R:]], -1)
        return out
    # one sample's group is one row
    N, S, C, G = c["N"], c["S"], c["C"], c["G"]
    rows = lambda t: t.double().reshape(N, S, G, C // G).transpose(1, 2).reshape(N * G, -1)  # noqa: E731
    back = lambda t: t.reshape(N, G, S, C // G).transpose(1, 2).reshape(N, S, C)  # noqa: E731
    per = lambda p: p.double().view(1, G, 1, C // G).expand(N, G, S, C // G).reshape(N * G, -1)  # noqa: E731
    x, w, b = rows(s["x"]), per(s["weight"]), per(s["bias"])
    if kind == "norm":
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = (var + s["eps"]) ** -0.5
    else:
        mean, rstd = (t.double().reshape(N * G, 1) for t in s["stats"])
    with torch.enable_grad():
        v = ((x - mean) * rstd * w + b).requires_grad_()
        a = {"none": v, "silu": v / (1.0 + torch.exp(-v)), "gelu": v * torch.special.ndtr(v)}[c["act"]]
        z = rows(s["z"]).requires_grad_() if c["gate"] else None
        y = a if z is None else a * z / (1.0 + torch.exp(-z))
        if kind == "norm":
            return dict(y=back(y.detach()), stats=torch.stack([mean.view(N, G), rstd.view(N, G)]))
        wrt = [v] + ([z] if z is not None else [])
        grads = torch.autograd.grad(y, wrt, rows(s["dy"]))
    xh, n = (x - mean) * rstd, x.shape[1]
    dh = grads[0] * w
    out = dict(d_z=back(grads[1])) if z is not None else {}
    out["d_x"] = back(rstd / n * (n * dh - dh.sum(1, keepdim=True) - xh * (dh * xh).sum(1, keepdim=True)))
    out["d_weight"], out["d_bias"] = back(grads[0] * xh).sum((0, 1)), back(grads[0]).sum((0, 1))
    return out


def _exact_attention(c, s):
    """Step by step."""
    B, H, K, V, T = c["B"], c["H"], c["K"], c["V"], c.get("T", 1)
    own_heads = lambda t: t.double().reshape(B, T, -1, t.shape[-1]).repeat_interleave(H // t.shape[-2], 2)  # noqa: E731
    q, k, v = own_heads(s["q"]), own_heads(s["k"]), own_heads(s["v"])
    lam = torch.exp(s["decay"].double())[None, :, None, None]
    S = torch.zeros(B, H, K, V, device=q.device, dtype=torch.float64) if s["state"] is None else s["state"].double()
    do = own_heads(s["do"]) if c["kind"] == "attn_bwd" else None
    out = torch.empty_like(v if do is None else q)
    for t in range(T):
        S = torch.addcmul(lam * S, k[:, t, :, :, None], v[:, t, :, None, :])
        out[:, t] = torch.matmul(q[:, t, :, None], S)[:, :, 0] if do is None else torch.matmul(S, do[:, t, :, :, None])[..., 0]
    out *= s["scale"]
    if c["kind"] == "step":
        return dict(o=out[:, 0], state_out=S)
    if do is None:
        return dict(o=out) if s["state"] is None else dict(o=out, state_out=S)
    R = torch.zeros_like(S) if s["d_state_out"] is None else s["d_state_out"].double()
    d_k, d_v = torch.empty_like(k), torch.empty_like(v)
    for t in range(T - 1, -1, -1):
        R = torch.addcmul(R, q[:, t, :, :, None], do[:, t, :, None, :], value=s["scale"])
        d_k[:, t] = torch.matmul(R, v[:, t, :, :, None])[..., 0]
        d_v[:, t] = torch.matmul(k[:, t, :, None], R)[:, :, 0]
        R = lam * R
    shared = lambda d, n: d.reshape(B, T, n, H // n, -1).sum(3)  # noqa: E731
    res = dict(d_q=shared(out, c["Hq"]), d_k=shared(d_k, c["Hk"]), d_v=shared(d_v, c["Hv"]))
    if s["state"] is not None:
        res["d_state"] = R
    return res


# ---------------------------------------------------------------------------------------------------
# what a call cannot do without
# ---------------------------------------------------------------------------------------------------

def work(case):
    c, kind, e = case, case["kind"], _SIZE[case["dtype"]]
    if kind in ("step", "attn", "attn_bwd"):
        n, K, V = c["B"] * c.get("T", 1), c["K"], c["V"]
        qkv = e * n * (K * (c["Hq"] + c["Hk"]) + V * c["Hv"])
        o = e * n * c["H"] * V
        states = 8.0 * c["B"] * c["H"] * K * V if kind == "step" or c["state"] else 0.0
        flops = 4.0 * n * c["H"] * K * V  # a token's part in a state and what is read from it
        if kind == "attn_bwd":
            return {"bytes": 2.0 * qkv + o + 1.5 * states, "flops": 2.5 * flops}
        return {"bytes": float(qkv + o) + states, "flops": flops}
    if kind == "rotary":
        n = c["B"] * c["T"]
        return {"bytes": 2.0 * e * n * (c["H"] + c["Hk"]) * c["D"] + 4.0 * n, "flops": 3.0 * n * (c["H"] + c["Hk"]) * c["R"]}
    n = c["N"] * c["S"] * c["C"]
    gate = 1 if c["gate"] else 0
    if kind == "norm":
        return {"bytes": e * n * (2.0 + gate) + 8.0 * (c["N"] * c["G"] + c["C"]), "flops": 10.0 * n}
    return {"bytes": e * n * (3.0 + 2.0 * gate) + 8.0 * c["N"] * c["G"] + 16.0 * c["C"], "flops": 20.0 * n}
