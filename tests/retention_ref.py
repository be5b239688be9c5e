"""Plain implementations in 64 bits of linear attention, rotation and group norm, for the tests of their kernels."""
import math

import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}           # and absolute


def spread(t, H):
    """[B,T,heads,W] -> [B,T,H,W] in f64, shared heads repeated."""
    return t.double().repeat_interleave(H // t.shape[2], 2)


def gather(d, n):
    """Sums the gradients of heads that share one of n."""
    B, T, H, W = d.shape
    return d.reshape(B, T, n, H // n, W).sum(3)


def attention(q, k, v, decay, scale, state=None):
    """(o, last state), token by token."""
    H = decay.shape[0]
    q, k, v = (spread(t, H) for t in (q, k, v))
    lam = torch.exp(decay.double())[None, :, None, None]
    S = torch.zeros(q.shape[0], H, q.shape[3], v.shape[3], dtype=torch.float64, device=q.device) if state is None else state.double()
    o = torch.empty_like(v)
    for t in range(q.shape[1]):
        S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * torch.einsum("bhk,bhkv->bhv", q[:, t], S)
    return o, S


def attention_grads(q, k, v, do, decay, scale, state=None, d_last=None):
    """d_q, d_k, d_v, d_state, token by token."""
    H, n = decay.shape[0], [t.shape[2] for t in (q, k, v)]
    q, k, v, do = (spread(t, H) for t in (q, k, v, do))
    lam = torch.exp(decay.double())[None, :, None, None]
    S = torch.zeros(q.shape[0], H, q.shape[3], v.shape[3], dtype=torch.float64, device=q.device) if state is None else state.double()
    R = torch.zeros_like(S) if d_last is None else d_last.double()
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    for t in range(q.shape[1]):
        S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * torch.einsum("bhkv,bhv->bhk", S, do[:, t])
    for t in range(q.shape[1] - 1, -1, -1):
        R = R + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = torch.einsum("bhkv,bhv->bhk", R, v[:, t])
        dv[:, t] = torch.einsum("bhkv,bhk->bhv", R, k[:, t])
        R = lam * R
    return gather(dq, n[0]), gather(dk, n[1]), gather(dv, n[2]), R


def rotary(x, positions, inv_freq, interleaved, scale, inverse=False):
    B, T, _, D = x.shape
    n = inv_freq.shape[0]
    angle = (positions.double().expand(B, T)[..., None] * inv_freq.double())[:, :, None]
    if inverse:
        angle = -angle
    x, y = x.double(), x.double().clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., a] = scale * (x[..., a] * angle.cos() - x[..., b] * angle.sin())
    y[..., b] = scale * (x[..., b] * angle.cos() + x[..., a] * angle.sin())
    return y


def group_norm(x, weight, bias, groups, eps, activation, z):
    """(y, mean, rstd) of [N,S,C] in f64; differentiable."""
    N, S, C = x.shape
    g = x.view(N, S, groups, C // groups)
    mean = g.mean((1, 3), keepdim=True)
    rstd = 1.0 / ((g - mean) ** 2).mean((1, 3), keepdim=True).add(eps).sqrt()
    v = ((g - mean) * rstd).view(N, S, C) * weight + bias
    y = {None: lambda: v, "silu": lambda: v * torch.sigmoid(v), "gelu": lambda: v * 0.5 * torch.erfc(-v * math.sqrt(0.5))}[activation]()
    return (y if z is None else y * z * torch.sigmoid(z)), mean[:, 0, :, 0], rstd[:, 0, :, 0]


def fro(got, want):
    """Distance relative to the wanted values' norm."""
    d = (got.double() - want).norm()
    return float(d / want.norm().clamp(min=1e-300))
