"""Operator layer over the C ABI, on torch CUDA tensors.

Names and argument meaning follow the reference's launch sites
(src/mamba_ssm/gpu/forward_mixed.rs:433-758, prefill.rs:676-961): activations
are ``[B, T, D]`` row-major views (a last-dim stride of 1 and any row stride, so
the x / z halves of ``proj[B*T, 2D]`` and the B / C columns of ``xdbl`` are
passed in place), state tensors are f32.  torch is used for device memory and
streams only; every compute call goes through ``libmamba_b200.so``.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import ffi

__all__ = ["selective_scan_fwd", "selective_scan_fwd_workspace_bytes", "selective_scan_bwd",
           "selective_scan_bwd_workspace_bytes",
           "residual_rmsnorm_fwd", "residual_rmsnorm_bwd", "embedding_gather", "softmax_xent", "adamw_step",
           "ssm_parallel_scan_fwd_nosave", "ssm_scan_fwd_save", "ssm_scan_bwd", "conv1d_fwd_nosave", "selective_scan_step", "conv1d_fwd", "conv1d_bwd", "m3_ssd_fwd", "m3_ssd_fwd_fused_kq", "m3_ssd_bwd", "dtype_code",
           "embedding_fwd", "embedding_bwd", "embedding_bwd_workspace_bytes", "token_logprobs", "token_logprobs_bwd",
           "gated_scan_fwd", "gated_scan_bwd", "gated_scan_step", "gated_scan_states",
           "gated_scan_workspace_bytes",
           "linear_attention_fwd", "linear_attention_bwd", "linear_attention_step", "linear_attention_workspace_bytes",
           "rotary_fwd", "rotary_bwd", "rotary_frequencies", "group_norm_fwd", "group_norm_bwd", "group_norm_workspace_bytes"]


_DTYPES = {torch.float32: ffi.F32, torch.float16: ffi.F16, torch.bfloat16: ffi.BF16}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPES[dt]
    except KeyError:
        raise TypeError(f"unsupported storage dtype {dt} (WeightDtype is f32 / f16 / bf16)")


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("mamba_rs_b200 ops take CUDA tensors only (no CPU fallback)")


def _rows(t: torch.Tensor, name: str) -> int:
    """Row stride (elements) of a [B, T, C] or [B*T, C] activation view."""
    if t.stride(-1) != 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    ld = t.stride(-2)
    if t.dim() == 3 and t.shape[0] > 1 and t.stride(0) != t.shape[1] * ld:
        raise ValueError(f"{name}: batch stride must equal T * row stride")
    return ld


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(dev):
    """The current stream of a device as the integer the C ABI takes (no Stream object is built)."""
    return torch._C._cuda_getCurrentRawStream(dev.index or 0)


class _on:
    """``with torch.cuda.device(dev)`` that costs nothing when the device is current already."""

    __slots__ = ("dev", "guard")

    def __init__(self, dev):
        self.dev, self.guard = dev, None

    def __enter__(self):
        if torch._C._cuda_getDevice() != (self.dev.index or 0):
            self.guard = torch.cuda.device(self.dev)
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def selective_scan_fwd(x, delta, Bm, Cm, a_neg, Dp, z=None, *, z_mode=None,
                       delta_softplus=True, conv_w=None, conv_b=None, conv_state=None,
                       ssm_state=None, y=None, u_out=None, chunk_states=None, save_stride=0,
                       workspace=None, handle=None):
    """Fused forward ``[conv1d+SiLU] -> softplus -> scan -> +D*u -> *SiLU(z)``.

    x, delta, z: [B,T,D]; Bm, Cm: [B,T,N]; a_neg [D,N] f32; Dp [D] f32.
    conv_state [B,D,K] / ssm_state [B,D,N] f32 are updated in place.
    workspace: optional uint8 scratch of selective_scan_fwd_workspace_bytes(...)
    bytes; with it a small batch is cut into time segments that run side by side.
    Returns y [B,T,D] in the storage dtype of x."""
    _require_cuda(x, delta, Bm, Cm, a_neg, Dp, z, conv_w, conv_b, conv_state, ssm_state, y, u_out)
    Bsz, T, D = delta.shape
    N = a_neg.shape[1]
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    if y is None:
        y = torch.empty((Bsz, T, D), dtype=x.dtype, device=dev)
    if z_mode is None:
        z_mode = 0 if z is None else 1
    a = ffi.SscanFwdArgs()
    a.dtype = dtype_code(x.dtype)
    for t, nm in ((delta, "delta"), (Bm, "B"), (Cm, "C"), (z, "z"), (y, "y"), (u_out, "u_out")):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{nm} dtype {t.dtype} != x dtype {x.dtype}")
    for t, nm in ((a_neg, "a_neg"), (Dp, "D"), (conv_w, "conv_w"), (conv_b, "conv_b"),
                  (conv_state, "conv_state"), (ssm_state, "ssm_state"), (chunk_states, "chunk_states")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise TypeError(f"{nm} must be contiguous float32")
    a.B, a.T, a.D, a.N = Bsz, T, D, N
    a.x, a.ld_x = _ptr(x), _rows(x, "x")
    a.delta, a.ld_delta, a.delta_softplus = _ptr(delta), _rows(delta, "delta"), int(delta_softplus)
    if _rows(Bm, "B") != _rows(Cm, "C"):
        raise ValueError("B and C must share a row stride")
    a.Bm, a.Cm, a.ld_bc = _ptr(Bm), _ptr(Cm), _rows(Bm, "B")
    a.z, a.ld_z, a.z_mode = _ptr(z), (_rows(z, "z") if z is not None else 0), int(z_mode)
    a.a_neg, a.Dp = _ptr(a_neg), _ptr(Dp)
    a.conv_w, a.conv_b, a.conv_state = _ptr(conv_w), _ptr(conv_b), _ptr(conv_state)
    a.K = conv_w.shape[1] if conv_w is not None else 0
    a.ssm_state = _ptr(ssm_state)
    a.y, a.ld_y = _ptr(y), _rows(y, "y")
    a.u_out, a.ld_u = _ptr(u_out), (_rows(u_out, "u_out") if u_out is not None else 0)
    a.chunk_states, a.save_stride = _ptr(chunk_states), int(save_stride)
    if workspace is not None:
        _require_cuda(workspace)
        a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel() * workspace.element_size()
    with _on(dev):
        rc = ffi.lib().mamba_b200_sscan_fwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_sscan_fwd")
    return y


def ssm_parallel_scan_fwd_nosave(h_state, y_out, delta, u, Bm, Cm, a_neg, Dp, *, handle=None):
    """Drop-in for the reference kernel ``ssm_parallel_scan_fwd_nosave_{dt}``
    (kernels/mamba_ssm_parallel.cu:544-553): contiguous tensors, delta already
    softplus'ed, ``h_state`` [B,D,N] f32 updated in place, ``y_out`` written."""
    _require_cuda(h_state, y_out, delta, u, Bm, Cm, a_neg, Dp)
    Bsz, T, D = delta.shape
    N = a_neg.shape[1]
    dev = delta.device
    hd = handle or ffi.default_handle(dev.index or 0)
    for t in (y_out, delta, u, Bm, Cm, a_neg, Dp, h_state):
        if not t.is_contiguous():
            raise ValueError("compat entry point takes contiguous tensors")
    fn = ffi.lib().mamba_b200_ssm_scan_fwd_nosave
    with _on(dev):
        rc = fn(hd.ptr, _stream(dev), dtype_code(delta.dtype), _ptr(h_state), _ptr(y_out),
                _ptr(delta), _ptr(u), _ptr(Bm), _ptr(Cm), _ptr(a_neg), _ptr(Dp), Bsz,
                T, D, N)
    hd.check(rc, "mamba_b200_ssm_scan_fwd_nosave")
    return y_out


def ssm_scan_fwd_save(h_state, y_out, h_saved, delta, u, Bm, Cm, a_neg, Dp, *, handle=None):
    """Drop-in for the reference's saving forward ``ssm_parallel_scan_fwd_{dt}``
    (kernels/mamba_ssm_parallel.cu:777-790): same tensors; of ``h_saved``
    [B, T+1, D, N] only rows 0, 32, 64, ... are written (what ssm_scan_bwd reads)."""
    _require_cuda(h_state, y_out, h_saved, delta, u, Bm, Cm, a_neg, Dp)
    Bsz, T, D = delta.shape
    N = a_neg.shape[1]
    dev = delta.device
    hd = handle or ffi.default_handle(dev.index or 0)
    if tuple(h_saved.shape) != (Bsz, T + 1, D, N) or h_saved.dtype != torch.float32 or not h_saved.is_contiguous():
        raise ValueError("h_saved must be contiguous float32 [B, T+1, D, N]")
    for t in (y_out, delta, u, Bm, Cm, a_neg, Dp, h_state):
        if not t.is_contiguous():
            raise ValueError("compat entry point takes contiguous tensors")
    with _on(dev):
        rc = ffi.lib().mamba_b200_ssm_scan_fwd_save(
            hd.ptr, _stream(dev), dtype_code(delta.dtype), _ptr(h_state), _ptr(y_out), _ptr(h_saved),
            _ptr(delta), _ptr(u), _ptr(Bm), _ptr(Cm), _ptr(a_neg), _ptr(Dp), Bsz, T, D, N)
    hd.check(rc, "mamba_b200_ssm_scan_fwd_save")
    return y_out


def ssm_scan_bwd(h_saved, delta, u, Bm, Cm, a_neg, Dp, dy, *, d_D=None, d_a_log=None, workspace=None,
                 handle=None):
    """Drop-in for ``ssm_parallel_scan_bwd_{dt}`` / ``ssm_backward_local_{dt}`` plus the four
    reducers (kernels/mamba_ssm_parallel.cu:1182-1200, kernels/mamba_ssm.cu:466-763), on the
    reference's own buffers.  Returns dict(d_delta, d_u, dB, dC, dD, dA_log); d_D / d_a_log
    are accumulated into the tensors passed in (zeros otherwise)."""
    _require_cuda(h_saved, delta, u, Bm, Cm, a_neg, Dp, dy, d_D, d_a_log, workspace)
    Bsz, T, D = delta.shape
    N = a_neg.shape[1]
    dev = delta.device
    hd = handle or ffi.default_handle(dev.index or 0)
    for t in (h_saved, delta, u, Bm, Cm, a_neg, Dp, dy):
        if not t.is_contiguous():
            raise ValueError("compat entry point takes contiguous tensors")
    f32 = dict(dtype=torch.float32, device=dev)
    d_delta, d_u = torch.empty_like(delta), torch.empty_like(u)
    dB, dC = torch.empty((Bsz, T, N), **f32), torch.empty((Bsz, T, N), **f32)
    d_D = torch.zeros(D, **f32) if d_D is None else d_D
    d_a_log = torch.zeros((D, N), **f32) if d_a_log is None else d_a_log
    if workspace is None:
        workspace = torch.empty(max(selective_scan_bwd_workspace_bytes(Bsz, T, D, N), 1), dtype=torch.uint8,
                                device=dev)
    with _on(dev):
        rc = ffi.lib().mamba_b200_ssm_scan_bwd(
            hd.ptr, _stream(dev), dtype_code(delta.dtype), _ptr(h_saved), _ptr(delta), _ptr(u), _ptr(Bm),
            _ptr(Cm), _ptr(a_neg), _ptr(Dp), _ptr(dy), _ptr(d_delta), _ptr(d_u), _ptr(dB), _ptr(dC), _ptr(d_D),
            _ptr(d_a_log), Bsz, T, D, N, _ptr(workspace), workspace.numel())
    hd.check(rc, "mamba_b200_ssm_scan_bwd")
    return dict(d_delta=d_delta, d_u=d_u, dB=dB, dC=dC, dD=d_D, dA_log=d_a_log)


def conv1d_fwd_nosave(u_out, state, x, conv_w, conv_b, *, handle=None):
    """Drop-in for ``conv1d_burnin_forward_nosave_{dt}`` (kernels/conv1d.cu:284-296)."""
    _require_cuda(u_out, state, x, conv_w, conv_b)
    Bsz, T, D = x.shape
    dev = x.device
    hd = handle or ffi.default_handle(dev.index or 0)
    for t in (u_out, state, x, conv_w, conv_b):
        if not t.is_contiguous():
            raise ValueError("compat entry point takes contiguous tensors")
    with _on(dev):
        rc = ffi.lib().mamba_b200_conv1d_fwd_nosave(hd.ptr, _stream(dev), dtype_code(x.dtype), _ptr(u_out),
                                                    _ptr(state), _ptr(x), _ptr(conv_w), _ptr(conv_b), Bsz, T, D,
                                                    conv_w.shape[1])
    hd.check(rc, "mamba_b200_conv1d_fwd_nosave")
    return u_out


def selective_scan_fwd_workspace_bytes(B, T, D, N) -> int:
    """Bytes of the optional forward scratch (segment hand-over states)."""
    return int(ffi.lib().mamba_b200_sscan_fwd_workspace_bytes(B, T, D, N))


def selective_scan_bwd_workspace_bytes(B, T, D, N) -> int:
    """Bytes of caller-owned scratch the backward needs (per-tile dB/dC partials
    and per-sample dA_log / dD partials)."""
    return int(ffi.lib().mamba_b200_sscan_bwd_workspace_bytes(B, T, D, N))


def selective_scan_bwd(u, delta, Bm, Cm, a_neg, Dp, dy, chunk_states, save_stride, z=None, *,
                       z_mode=None, delta_softplus=True, dA_log=None, dD=None, workspace=None,
                       handle=None):
    """Fused backward (BPTT by recomputation from the saved block-boundary
    states).  Returns dict(d_u, d_delta, d_z, dB, dC, dA_log, dD); dA_log and
    dD are accumulated into the tensors passed in (zeros if none are passed)."""
    _require_cuda(u, delta, Bm, Cm, a_neg, Dp, dy, chunk_states, z)
    Bsz, T, D = delta.shape
    N = a_neg.shape[1]
    dev = u.device
    h = handle or ffi.default_handle(dev.index or 0)
    if z_mode is None:
        z_mode = 0 if z is None else 1
    f32 = dict(dtype=torch.float32, device=dev)
    d_u = torch.empty((Bsz, T, D), dtype=u.dtype, device=dev)
    d_delta = torch.empty((Bsz, T, D), dtype=u.dtype, device=dev)
    d_z = torch.empty((Bsz, T, D), dtype=u.dtype, device=dev) if z_mode else None
    dB = torch.empty((Bsz, T, N), **f32)
    dC = torch.empty((Bsz, T, N), **f32)
    dA_log = torch.zeros((D, N), **f32) if dA_log is None else dA_log
    dD = torch.zeros((D,), **f32) if dD is None else dD
    need = selective_scan_bwd_workspace_bytes(Bsz, T, D, N)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    a = ffi.SscanBwdArgs()
    a.dtype = dtype_code(u.dtype)
    a.B, a.T, a.D, a.N = Bsz, T, D, N
    a.u, a.ld_u = _ptr(u), _rows(u, "u")
    a.delta, a.ld_delta, a.delta_softplus = _ptr(delta), _rows(delta, "delta"), int(delta_softplus)
    a.Bm, a.Cm, a.ld_bc = _ptr(Bm), _ptr(Cm), _rows(Bm, "B")
    a.z, a.ld_z, a.z_mode = _ptr(z), (_rows(z, "z") if z is not None else 0), int(z_mode)
    a.a_neg, a.Dp = _ptr(a_neg), _ptr(Dp)
    a.chunk_states, a.save_stride = _ptr(chunk_states), int(save_stride)
    a.dy, a.ld_dy = _ptr(dy), _rows(dy, "dy")
    a.d_u, a.ld_du = _ptr(d_u), D
    a.d_delta, a.ld_ddelta = _ptr(d_delta), D
    a.d_z, a.ld_dz = _ptr(d_z), D
    a.dBm, a.dCm, a.dA_log, a.dD = _ptr(dB), _ptr(dC), _ptr(dA_log), _ptr(dD)
    a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel()
    with _on(dev):
        rc = ffi.lib().mamba_b200_sscan_bwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_sscan_bwd")
    return dict(d_u=d_u, d_delta=d_delta, d_z=d_z, dB=dB, dC=dC, dA_log=dA_log, dD=dD)


def selective_scan_step(x, delta, Bm, Cm, a_neg, Dp, ssm_state, z=None, *, z_mode=None,
                        delta_softplus=True, conv_w=None, conv_b=None, conv_state=None, y=None,
                        u_out=None, handle=None):
    """T = 1 decode step (GpuMambaBackbone::step inner kernels).  x, delta, z:
    [B,D]; Bm, Cm: [B,N] (views of xdbl are fine); states updated in place."""
    _require_cuda(x, delta, Bm, Cm, a_neg, Dp, ssm_state, z, conv_w, conv_b, conv_state)
    Bsz, D = delta.shape
    N = a_neg.shape[1]
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    if y is None:
        y = torch.empty((Bsz, D), dtype=x.dtype, device=dev)
    if z_mode is None:
        z_mode = 0 if z is None else 1
    a = ffi.SscanStepArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.D, a.N = Bsz, D, N
    a.x, a.ld_x = _ptr(x), x.stride(0)
    a.delta, a.ld_delta, a.delta_softplus = _ptr(delta), delta.stride(0), int(delta_softplus)
    a.Bm, a.Cm, a.ld_bc = _ptr(Bm), _ptr(Cm), Bm.stride(0)
    a.z, a.ld_z, a.z_mode = _ptr(z), (z.stride(0) if z is not None else 0), int(z_mode)
    a.a_neg, a.Dp = _ptr(a_neg), _ptr(Dp)
    a.conv_w, a.conv_b, a.conv_state = _ptr(conv_w), _ptr(conv_b), _ptr(conv_state)
    a.K = conv_w.shape[1] if conv_w is not None else 0
    a.ssm_state = _ptr(ssm_state)
    a.y, a.ld_y = _ptr(y), y.stride(0)
    a.u_out, a.ld_u = _ptr(u_out), (u_out.stride(0) if u_out is not None else 0)
    with _on(dev):
        rc = ffi.lib().mamba_b200_sscan_step(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_sscan_step")
    return y


def conv1d_fwd(x, conv_w, conv_b, conv_state=None, u=None, *, handle=None):
    """Depthwise causal conv1d + SiLU over [B,T,D]; conv_state [B,D,K] in/out."""
    _require_cuda(x, conv_w, conv_b, conv_state, u)
    Bsz, T, D = x.shape
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    if u is None:
        u = torch.empty((Bsz, T, D), dtype=x.dtype, device=dev)
    a = ffi.Conv1dArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.T, a.D, a.K = Bsz, T, D, conv_w.shape[1]
    a.x, a.ld_x = _ptr(x), _rows(x, "x")
    a.conv_w, a.conv_b, a.conv_state = _ptr(conv_w), _ptr(conv_b), _ptr(conv_state)
    a.u, a.ld_u = _ptr(u), _rows(u, "u")
    with _on(dev):
        rc = ffi.lib().mamba_b200_conv1d_fwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_conv1d_fwd")
    return u


def conv1d_bwd(x, conv_w, conv_b, d_u, conv_state0=None, *, dconv_w=None, dconv_b=None,
               workspace=None, handle=None):
    """Backward of conv1d + SiLU by recomputation.  Returns dict(d_x, dconv_w,
    dconv_b); the parameter gradients are accumulated into the tensors given."""
    _require_cuda(x, conv_w, conv_b, d_u, conv_state0)
    Bsz, T, D = x.shape
    K = conv_w.shape[1]
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    d_x = torch.empty((Bsz, T, D), dtype=x.dtype, device=dev)
    dconv_w = torch.zeros((D, K), dtype=torch.float32, device=dev) if dconv_w is None else dconv_w
    dconv_b = torch.zeros((D,), dtype=torch.float32, device=dev) if dconv_b is None else dconv_b
    need = int(ffi.lib().mamba_b200_conv1d_bwd_workspace_bytes(Bsz, T, D, K))
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    a = ffi.Conv1dArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.T, a.D, a.K = Bsz, T, D, K
    a.x, a.ld_x = _ptr(x), _rows(x, "x")
    a.conv_w, a.conv_b, a.conv_state = _ptr(conv_w), _ptr(conv_b), _ptr(conv_state0)
    a.d_u, a.ld_du = _ptr(d_u), _rows(d_u, "d_u")
    a.d_x, a.ld_dx = _ptr(d_x), D
    a.dconv_w, a.dconv_b = _ptr(dconv_w), _ptr(dconv_b)
    a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel()
    with _on(dev):
        rc = ffi.lib().mamba_b200_conv1d_bwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_conv1d_bwd")
    return dict(d_x=d_x, dconv_w=dconv_w, dconv_b=dconv_b)


def m3_ssd_fwd(x, K, Q, dt, trap, adt, Dh, *, ssm_state=None, k_state=None, v_state=None,
               carry_in=False, force_sequential=False, y=None, handle=None):
    """Mamba-3 SISO SSD forward.  x [B,T,nh*hd], K/Q [B,T,nh,N] in the storage
    dtype (contiguous); dt, trap, adt [B,T,nh] and Dh [nh] f32.  State tensors
    (f32) receive the state after the window; with carry_in they are read first."""
    _require_cuda(x, K, Q, dt, trap, adt, Dh, ssm_state, k_state, v_state, y)
    Bsz, T, nh, N = K.shape
    hd = x.shape[2] // nh
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    for t, nm in ((x, "x"), (K, "K"), (Q, "Q")):
        if not t.is_contiguous() or t.dtype != x.dtype:
            raise ValueError(f"{nm} must be contiguous and share x's dtype")
    for t, nm in ((dt, "dt"), (trap, "trap"), (adt, "adt"), (Dh, "Dh"), (ssm_state, "ssm_state"),
                  (k_state, "k_state"), (v_state, "v_state")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise TypeError(f"{nm} must be contiguous float32")
    if y is None:
        y = torch.empty_like(x)
    a = ffi.M3SsdArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.T, a.nh, a.hd, a.N = Bsz, T, nh, hd, N
    a.x, a.K, a.Q = _ptr(x), _ptr(K), _ptr(Q)
    a.dt, a.trap, a.adt, a.Dh = _ptr(dt), _ptr(trap), _ptr(adt), _ptr(Dh)
    a.y = _ptr(y)
    a.ssm_state, a.k_state, a.v_state = _ptr(ssm_state), _ptr(k_state), _ptr(v_state)
    a.carry_in, a.force_sequential = int(carry_in), int(force_sequential)
    with _on(dev):
        rc = ffi.lib().mamba_b200_m3_ssd_fwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_m3_ssd_fwd")
    return y


def m3_ssd_fwd_fused_kq(x, Bn, Cn, b_bias, c_bias, angle_vel, dt, trap, adt, Dh, *, angle_state=None,
                        ssm_state=None, k_state=None, v_state=None, y=None, handle=None):
    """Mamba-3 SISO SSD forward with the per-head K / Q built inside the kernel (bias add +
    RoPE with the running angle) from the group-level rows.  x [B,T,nh*hd], Bn / Cn
    [B,T,ng,N] in the 16-bit storage dtype; b_bias, c_bias [nh,N], angle_vel [B,T,n_angles]
    (= tanh(angles_raw) * pi; None = no rotation), dt, trap, adt [B,T,nh], Dh [nh] f32;
    angle_state [B,nh,n_angles] f32 is read and overwritten with the angle after the window."""
    _require_cuda(x, Bn, Cn, b_bias, c_bias, angle_vel, dt, trap, adt, Dh, angle_state, ssm_state, k_state,
                  v_state, y)
    Bsz, T, ng, N = Bn.shape
    nh = b_bias.shape[0]
    hd = x.shape[2] // nh
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    for t, nm in ((x, "x"), (Bn, "Bn"), (Cn, "Cn")):
        if not t.is_contiguous() or t.dtype != x.dtype:
            raise ValueError(f"{nm} must be contiguous and share x's dtype")
    for t, nm in ((b_bias, "b_bias"), (c_bias, "c_bias"), (angle_vel, "angle_vel"), (dt, "dt"), (trap, "trap"),
                  (adt, "adt"), (Dh, "Dh"), (angle_state, "angle_state"), (ssm_state, "ssm_state"),
                  (k_state, "k_state"), (v_state, "v_state")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise TypeError(f"{nm} must be contiguous float32")
    if y is None:
        y = torch.empty_like(x)
    a = ffi.M3SsdArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.T, a.nh, a.hd, a.N = Bsz, T, nh, hd, N
    a.x = _ptr(x)
    a.dt, a.trap, a.adt, a.Dh = _ptr(dt), _ptr(trap), _ptr(adt), _ptr(Dh)
    a.y = _ptr(y)
    a.ssm_state, a.k_state, a.v_state = _ptr(ssm_state), _ptr(k_state), _ptr(v_state)
    a.Bn, a.Cn, a.b_bias, a.c_bias = _ptr(Bn), _ptr(Cn), _ptr(b_bias), _ptr(c_bias)
    a.angle_vel, a.angle_state = _ptr(angle_vel), _ptr(angle_state)
    a.ng, a.n_angles = ng, (angle_vel.shape[2] if angle_vel is not None else 0)
    with _on(dev):
        rc = ffi.lib().mamba_b200_m3_ssd_fwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_m3_ssd_fwd")
    return y


def m3_ssd_bwd(x, K, Q, dt, trap, adt, Dh, dy, *, dD=None, workspace=None, handle=None):
    """Mamba-3 SISO SSD backward for a window that started from a zero state.
    Returns dx (storage dtype), dK, dQ, d_adt, d_dt, d_trap (f32) and dD (f32,
    accumulated into the tensor passed in, or a fresh zero one).  d_dt is the
    direct path only; the caller adds A * d_adt (src/mamba3_siso/gpu/backward.rs:420-457)."""
    _require_cuda(x, K, Q, dt, trap, adt, Dh, dy, dD, workspace)
    Bsz, T, nh, N = K.shape
    hd = x.shape[2] // nh
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    for t, nm in ((x, "x"), (K, "K"), (Q, "Q"), (dy, "dy")):
        if not t.is_contiguous() or t.dtype != x.dtype:
            raise ValueError(f"{nm} must be contiguous and share x's dtype")
    for t, nm in ((dt, "dt"), (trap, "trap"), (adt, "adt"), (Dh, "Dh"), (dD, "dD")):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous()):
            raise TypeError(f"{nm} must be contiguous float32")
    need = ffi.lib().mamba_b200_m3_ssd_bwd_workspace_bytes_for(dtype_code(x.dtype), Bsz, T, nh, hd, N)
    if workspace is None:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    f32 = dict(dtype=torch.float32, device=dev)
    dx = torch.empty_like(x)
    dK = torch.empty((Bsz, T, nh, N), **f32)
    dQ = torch.empty((Bsz, T, nh, N), **f32)
    d_adt = torch.empty((Bsz, T, nh), **f32)
    d_dt = torch.empty((Bsz, T, nh), **f32)
    d_trap = torch.empty((Bsz, T, nh), **f32)
    if dD is None:
        dD = torch.zeros(nh, **f32)
    a = ffi.M3SsdBwdArgs()
    a.dtype = dtype_code(x.dtype)
    a.B, a.T, a.nh, a.hd, a.N = Bsz, T, nh, hd, N
    a.x, a.K, a.Q, a.dy = _ptr(x), _ptr(K), _ptr(Q), _ptr(dy)
    a.dt, a.trap, a.adt, a.Dh = _ptr(dt), _ptr(trap), _ptr(adt), _ptr(Dh)
    a.dx, a.dK, a.dQ = _ptr(dx), _ptr(dK), _ptr(dQ)
    a.d_adt, a.d_dt, a.d_trap, a.dD = _ptr(d_adt), _ptr(d_dt), _ptr(d_trap), _ptr(dD)
    a.workspace, a.workspace_bytes = _ptr(workspace), workspace.numel()
    with _on(dev):
        rc = ffi.lib().mamba_b200_m3_ssd_bwd(h.ptr, _stream(dev), C.byref(a))
    h.check(rc, "mamba_b200_m3_ssd_bwd")
    return dict(dx=dx, dK=dK, dQ=dQ, d_adt=d_adt, d_dt=d_dt, d_trap=d_trap, dD=dD)


def residual_rmsnorm_fwd(residual, branch, scale, *, eps=1e-5, out_dtype=None, y=None, rms_out=None, handle=None):
    """residual [rows, dim] f32 += branch (storage dtype, or None); returns
    (y = rmsnorm(residual) * scale in the storage dtype, rms [rows] f32)."""
    _require_cuda(residual, branch, scale, y, rms_out)
    rows, dim = residual.shape
    dev = residual.device
    h = handle or ffi.default_handle(dev.index or 0)
    if residual.dtype != torch.float32 or not residual.is_contiguous() or not scale.is_contiguous():
        raise TypeError("residual and scale are contiguous float32")
    dt = branch.dtype if branch is not None else (out_dtype or torch.bfloat16)
    if branch is not None and (not branch.is_contiguous() or tuple(branch.shape) != (rows, dim)):
        raise ValueError("branch must be contiguous [rows, dim]")
    if y is None:
        y = torch.empty((rows, dim), dtype=dt, device=dev)
    if rms_out is None:
        rms_out = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        rc = ffi.lib().mamba_b200_residual_rmsnorm_fwd(h.ptr, _stream(dev), dtype_code(dt), _ptr(residual), _ptr(branch),
                                                       _ptr(scale), _ptr(y), _ptr(rms_out), rows, dim, float(eps))
    h.check(rc, "mamba_b200_residual_rmsnorm_fwd")
    return y, rms_out


def residual_rmsnorm_bwd(dy, x, scale, rms_saved, d_residual, d_scale, *, workspace=None, handle=None):
    """d_residual [rows, dim] f32 += dx of the RMSNorm; d_scale [dim] f32 += its scale
    gradient.  x is the f32 residual the forward normalised, rms_saved its per-row rms."""
    _require_cuda(dy, x, scale, rms_saved, d_residual, d_scale, workspace)
    rows, dim = x.shape
    dev = x.device
    h = handle or ffi.default_handle(dev.index or 0)
    need = int(ffi.lib().mamba_b200_residual_rmsnorm_bwd_workspace_bytes(rows, dim))
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    with _on(dev):
        rc = ffi.lib().mamba_b200_residual_rmsnorm_bwd(h.ptr, _stream(dev), dtype_code(dy.dtype), _ptr(dy), _ptr(x),
                                                       _ptr(scale), _ptr(rms_saved), _ptr(d_residual), _ptr(d_scale),
                                                       rows, dim, _ptr(workspace), workspace.numel())
    h.check(rc, "mamba_b200_residual_rmsnorm_bwd")
    return d_residual, d_scale


def embedding_gather(table, ids, out=None, *, handle=None):
    """out [rows, dim] f32 = table[ids] (table [vocab, dim] in the storage dtype, ids int32)."""
    _require_cuda(table, ids, out)
    vocab, dim = table.shape
    dev = table.device
    h = handle or ffi.default_handle(dev.index or 0)
    ids = ids.reshape(-1)
    if ids.dtype != torch.int32 or not ids.is_contiguous() or not table.is_contiguous():
        raise TypeError("ids are contiguous int32, the table is contiguous")
    if out is None:
        out = torch.empty((ids.numel(), dim), dtype=torch.float32, device=dev)
    with _on(dev):
        rc = ffi.lib().mamba_b200_embedding_gather(h.ptr, _stream(dev), dtype_code(table.dtype), _ptr(table), _ptr(ids),
                                                   _ptr(out), ids.numel(), dim, vocab)
    h.check(rc, "mamba_b200_embedding_gather")
    return out


def softmax_xent(logits, targets, *, grad_scale=1.0, want_grad=True, dlogits=None, handle=None):
    """Per-row cross-entropy of logits [rows, V] against int32 targets (negative = not
    counted).  Returns (loss_rows f32 [rows], d_logits in the logits' dtype or None)."""
    _require_cuda(logits, targets, dlogits)
    rows, V = logits.shape
    dev = logits.device
    h = handle or ffi.default_handle(dev.index or 0)
    if logits.stride(1) != 1 or targets.dtype != torch.int32 or not targets.is_contiguous():
        raise TypeError("logits rows are contiguous, targets are contiguous int32")
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    if want_grad and dlogits is None:
        dlogits = torch.empty_strided(logits.shape, logits.stride(), dtype=logits.dtype, device=dev)
    with _on(dev):
        rc = ffi.lib().mamba_b200_softmax_xent(h.ptr, _stream(dev), dtype_code(logits.dtype), _ptr(logits), _ptr(targets),
                                               _ptr(loss), _ptr(dlogits if want_grad else None), float(grad_scale),
                                               rows, V, logits.stride(0))
    h.check(rc, "mamba_b200_softmax_xent")
    return loss, (dlogits if want_grad else None)


def adamw_step(param, grad, m, v, bias_factors, *, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0,
               param_lp=None, handle=None):
    """In-place AdamW on flat f32 arenas; bias_factors is a 2-float device tensor
    {1/(1-beta1^t), 1/(1-beta2^t)}; param_lp (f16 / bf16) receives the compute copy."""
    _require_cuda(param, grad, m, v, bias_factors, param_lp)
    dev = param.device
    h = handle or ffi.default_handle(dev.index or 0)
    for t in (param, grad, m, v, bias_factors):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise TypeError("AdamW state is contiguous float32")
    with _on(dev):
        rc = ffi.lib().mamba_b200_adamw_step(h.ptr, _stream(dev), _ptr(param), _ptr(grad), _ptr(m), _ptr(v), float(lr),
                                             float(beta1), float(beta2), float(eps), float(weight_decay),
                                             _ptr(bias_factors), _ptr(param_lp),
                                             dtype_code(param_lp.dtype) if param_lp is not None else ffi.BF16,
                                             param.numel())
    h.check(rc, "mamba_b200_adamw_step")
    return param


def _device_index(*ts):
    """The index of the CUDA device that all the tensors (None aside) are on."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != index:
            index = -1
            break
    if index < 0:
        _require_cuda(*ts)
        raise ValueError(f"tensors on several devices: {', '.join(sorted({str(t.device) for t in ts if t is not None}))}")
    return index


def _new(like, dtype, rows, width):
    """An empty [rows, width] on like's device (half the host time of torch.empty)."""
    return torch.empty_strided((rows, width), (width, 1), dtype=dtype, device=like.device)


def _row(t, width):
    """Row stride of a matrix (of one row: any that is no narrower than the row)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)


def _launch(fn, index, handle, *args):
    """fn(handle, current stream of the device, *args) with the device current; failures as the library words them."""
    h = handle or ffi.default_handle(index)
    if torch._C._cuda_getDevice() == index:
        rc = fn(h.ptr, torch._C._cuda_getCurrentRawStream(index), *args)
    else:
        with torch.cuda.device(index):
            rc = fn(h.ptr, torch._C._cuda_getCurrentRawStream(index), *args)
    if rc:
        h.check(rc, fn.__name__)


def embedding_fwd(table, ids, *, scale=1.0, out=None, out_dtype=torch.float32, handle=None):
    """out [rows, dim] = scale * table[ids]: table [vocab, dim] in the storage dtype (any row stride), ids int32 of any
    shape; out in float32 (the residual stream) or the table's dtype.  An id outside the table gives a row of zeros."""
    dev = _device_index(table, ids, out)
    if table.dim() != 2 or table.stride(1) != 1 or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise TypeError("the table is [vocab, dim] with contiguous rows, ids are contiguous int32")
    vocab, dim = table.shape
    rows = ids.numel()
    if out is None:
        out, ld_out = _new(table, out_dtype, rows, dim), dim
    elif tuple(out.shape) != (rows, dim) or out.stride(1) != 1:
        raise ValueError(f"out is [{rows}, {dim}] with contiguous rows")
    else:
        out_dtype, ld_out = out.dtype, _row(out, dim)
    _launch(ffi.lib().mamba_b200_embedding_fwd, dev, handle, dtype_code(table.dtype), table.data_ptr(), _row(table, dim), ids.data_ptr(),
            dtype_code(out_dtype), out.data_ptr(), ld_out, rows, dim, vocab, scale)
    return out


def embedding_bwd_workspace_bytes(rows, dim, vocab) -> int:
    """Bytes of scratch the table's gradient needs (rows sorted by token, sums of rows that go on)."""
    return int(ffi.lib().mamba_b200_embedding_bwd_workspace_bytes(rows, dim, vocab))


def embedding_bwd(ids, d_out, vocab=None, *, d_table=None, scale=1.0, workspace=None, handle=None):
    """Gradient of embedding_fwd's table: scale * the sums of d_out's rows by token, f32 [vocab, dim].  Accumulated into
    d_table when it is given, else a fresh tensor.  ids int32 of any shape, d_out [ids.numel(), dim] in a storage dtype (any
    row stride).  The order of the sums is fixed: the same inputs give the same bits."""
    dev = _device_index(ids, d_out, d_table, workspace)
    rows = ids.numel()
    if ids.dtype != torch.int32 or not ids.is_contiguous():
        raise TypeError("ids are contiguous int32")
    if d_out.dim() != 2 or d_out.shape[0] != rows or d_out.stride(1) != 1:
        raise ValueError(f"d_out is [{rows}, dim] with contiguous rows")
    dim = d_out.shape[1]
    accumulate = d_table is not None
    if accumulate:
        if d_table.dtype != torch.float32 or not d_table.is_contiguous():
            raise TypeError("d_table is contiguous float32")
        if d_table.dim() != 2 or d_table.shape[1] != dim or (vocab is not None and vocab != d_table.shape[0]):
            raise ValueError(f"d_table is [vocab, {dim}], not {list(d_table.shape)}")
        vocab = d_table.shape[0]
    elif vocab is None:
        raise ValueError("the vocabulary's size or a table to accumulate into is needed")
    else:
        d_table = _new(d_out, torch.float32, vocab, dim)
    lib = ffi.lib()
    if workspace is None:
        need = lib.mamba_b200_embedding_bwd_workspace_bytes(rows, dim, vocab)
        workspace = torch.empty(need, dtype=torch.uint8, device=d_out.device) if need else None
    elif not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous")
    _launch(lib.mamba_b200_embedding_bwd, dev, handle, dtype_code(d_out.dtype), d_out.data_ptr(), _row(d_out, dim), ids.data_ptr(),
            d_table.data_ptr(), accumulate, rows, dim, vocab, scale, _ptr(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size())
    return d_table


def _logit_rows(logits, targets):
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise TypeError("logits are [rows, V] with contiguous rows")
    if targets is not None and (targets.dtype != torch.int32 or not targets.is_contiguous() or targets.numel() != logits.shape[0]):
        raise TypeError(f"targets are {logits.shape[0]} contiguous int32")


def token_logprobs(logits, targets=None, *, top=0, temperature=1.0, handle=None):
    """Per row of logits [rows, V] / temperature: dict(entropy [rows], lse [2, rows]), with targets (int32 [rows]; outside
    the vocabulary: not counted, 0) also logprob [rows], all f32; with top > 0 (at most 32) also top_ids int32 and
    top_logprobs f32 [rows, top], by falling probability, equal ones by rising index.  lse holds the largest
    logit M and the log of the sum of exp((logits - M) / temperature): the log-sum-exp is M / temperature plus that.  Logits of -inf are tokens that are ruled out."""
    dev = _device_index(logits, targets)
    _logit_rows(logits, targets)
    rows, V = logits.shape
    if not 0 <= top <= min(32, V):
        raise ValueError(f"{top} alternatives of {V} tokens (at most 32)")
    # (a tensor of its own costs the host half of what a slice does)
    lse = _new(logits, torch.float32, 2, rows)
    entropy = lse.new_empty(rows)
    out = dict(lse=lse, entropy=entropy)
    tp = lp = ip = vp = None
    if targets is not None:
        out["logprob"] = logprob = torch.empty_like(entropy)
        tp, lp = targets.data_ptr(), logprob.data_ptr()
    if top:
        out["top_logprobs"] = val = _new(logits, torch.float32, rows, top)
        out["top_ids"] = ids = torch.empty_like(val, dtype=torch.int32)
        ip, vp = ids.data_ptr(), val.data_ptr()
    _launch(ffi.lib().mamba_b200_token_logprobs, dev, handle, dtype_code(logits.dtype), logits.data_ptr(), _row(logits, V), tp,
            temperature, lse.data_ptr(), entropy.data_ptr(), lp, top, ip, vp, rows, V)
    return out


def token_logprobs_bwd(logits, targets, lse, entropy, d_logprob=None, d_entropy=None, *, temperature=1.0, dlogits=None,
                       handle=None):
    """Gradient of the logits from those of logprob and entropy (f32 [rows], either may be None), with lse and entropy as
    token_logprobs returned them.  dlogits in the logits' dtype; it may be the logits themselves.  Where the row strides of the two
    differ by no multiple of 16 bytes (a padded head's logits[:, :V] and a result that is made here), elements are moved one by one,
    at a third of the speed: a dlogits with the logits' own stride avoids it."""
    dev = _device_index(logits, targets, lse, entropy, d_logprob, d_entropy, dlogits)
    _logit_rows(logits, targets)
    rows, V = logits.shape
    for t, nm, n in ((lse, "lse", 2), (entropy, "entropy", 1), (d_logprob, "d_logprob", 1), (d_entropy, "d_entropy", 1)):
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != n * rows):
            raise TypeError(f"{nm} is contiguous float32, {n} x {rows}")
    if dlogits is None:
        dlogits = _new(logits, logits.dtype, rows, V)
    elif dlogits.dtype != logits.dtype or dlogits.shape != logits.shape or dlogits.stride(1) != 1:
        raise TypeError("dlogits has the logits' dtype and shape and contiguous rows")
    _launch(ffi.lib().mamba_b200_token_logprobs_bwd, dev, handle, dtype_code(logits.dtype), logits.data_ptr(), _row(logits, V),
            _ptr(targets), temperature, lse.data_ptr(), _ptr(entropy), _ptr(d_logprob), _ptr(d_entropy), dlogits.data_ptr(),
            _row(dlogits, V), rows, V)
    return dlogits


def gated_scan_states(B, T, D):
    """Shape of the chunk_states that gated_scan_fwd keeps for gated_scan_bwd."""
    return (B, -(-T // ffi.GATED_SCAN_SAVE), D)


def gated_scan_workspace_bytes(B, T, D) -> int:
    """Bytes of the scratch that lets a long axis of few channels run as segments side by side (0: it is not cut)."""
    return int(ffi.lib().mamba_b200_gated_scan_workspace_bytes(B, T, D))


def _gated_workspace(workspace, x):
    """(tensor, address, bytes) of the scratch for x: the caller's, or one of its own where it is needed."""
    if workspace is None:
        need = ffi.lib().mamba_b200_gated_scan_workspace_bytes(*x.shape)
        if not need:
            return None, None, 0
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    elif not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _gated_rows(t, name, like):
    """Row stride of a [B, T, D] view whose rows are one after another: any stride where there is but one row."""
    if t.dtype != like.dtype or t.shape != like.shape:
        raise TypeError(f"{name} has x's dtype and shape: {list(like.shape)} {like.dtype}")
    B, T, D = t.shape
    s0, s1, s2 = t.stride()
    if s2 != 1 and D > 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    if T <= 1:
        s1 = s0 if B > 1 and T else D
    elif B > 1 and s0 != T * s1:
        raise ValueError(f"{name}: batch stride must equal T * row stride")
    return s1


def _gated_state(t, name, x, shape=None):
    shape = shape or (x.shape[0], x.shape[2])
    if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous()):
        raise TypeError(f"{name} is contiguous float32 {list(shape)}")
    return _ptr(t)


def gated_scan_fwd(x, f, z=None, *, h0=None, h_last=None, y=None, chunk_states=None, workspace=None, handle=None):
    """Gated linear recurrence: u = sigmoid(-f), h_t = h_{t-1} + u_t (x_t - h_{t-1}), y = h * SiLU(z) (y = h without z).
    x, f, z, y [B,T,D] in a storage dtype, any row stride; h0 (zeros if None) and h_last (written if given, may be h0)
    [B,D] f32; chunk_states f32 of gated_scan_states(B,T,D) receives what gated_scan_bwd needs.  workspace: scratch of
    gated_scan_workspace_bytes(B,T,D) bytes (made here if None).  Returns y."""
    dev = _device_index(x, f, z, h0, h_last, y, chunk_states, workspace)
    if y is None:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
    B, T, D = x.shape
    a = ffi.GatedScanArgs(dtype_code(x.dtype), B, T, D, x.data_ptr(), _gated_rows(x, "x", x), f.data_ptr(), _gated_rows(f, "f", x),
                          _ptr(z), 0 if z is None else _gated_rows(z, "z", x), _gated_state(h0, "h0", x),
                          _gated_state(h_last, "h_last", x), y.data_ptr(), _gated_rows(y, "y", x),
                          _gated_state(chunk_states, "chunk_states", x, gated_scan_states(B, T, D)))
    if T > 8:
        workspace, a.workspace, a.workspace_bytes = _gated_workspace(workspace, x)
    _launch(ffi.lib().mamba_b200_gated_scan_fwd, dev, handle, C.byref(a))
    return y


def gated_scan_step(x, f, h0, z=None, *, h_last=None, y=None, handle=None):
    """One token per sequence: x, f, z, y [B,D]; the state h0 [B,D] f32 is updated in place, or h_last receives it."""
    dev = _device_index(x, f, h0, z, h_last, y)
    dtype = x.dtype
    B, D = shape = x.shape
    if y is None:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)

    def row(t, name):
        if t.dtype != dtype or t.shape != shape:
            raise TypeError(f"{name} has x's dtype and shape: {list(shape)} {dtype}")
        ld, one = t.stride()
        if one != 1 and D > 1:
            raise ValueError(f"{name}: last dimension must be contiguous")
        return ld if B > 1 else D

    for t, name in ((h0, "h0"), (h_last, "h_last")):
        if t is not None and (t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous()):
            raise TypeError(f"{name} is contiguous float32 {list(shape)}")
    h = h0.data_ptr()
    a = ffi.GatedScanArgs(dtype_code(dtype), B, 1, D, x.data_ptr(), row(x, "x"), f.data_ptr(), row(f, "f"), _ptr(z),
                          0 if z is None else row(z, "z"), h, h if h_last is None else h_last.data_ptr(), y.data_ptr(), row(y, "y"))
    _launch(ffi.lib().mamba_b200_gated_scan_fwd, dev, handle, C.byref(a))
    return y


def gated_scan_bwd(x, f, dy, chunk_states, z=None, *, d_last=None, d_h0=None, d_x=None, d_f=None, d_z=None, workspace=None,
                   handle=None):
    """Backward of gated_scan_fwd from its chunk_states.  d_last [B,D] f32: gradient of the state that left (None: zeros).
    Returns dict(d_x, d_f, d_z (with z), d_h0 f32); the outputs may be given (columns of one projection's gradient, say)."""
    dev = _device_index(x, f, z, dy, chunk_states, d_last, d_h0, d_x, d_f, d_z, workspace)
    B, T, D = x.shape
    new = lambda t: torch.empty_like(x, memory_format=torch.contiguous_format) if t is None else t  # noqa: E731
    d_x, d_f = new(d_x), new(d_f)
    d_z = new(d_z) if z is not None else None
    if d_h0 is None:
        d_h0 = _new(x, torch.float32, B, D)
    a = ffi.GatedScanArgs(dtype_code(x.dtype), B, T, D, x.data_ptr(), _gated_rows(x, "x", x), f.data_ptr(), _gated_rows(f, "f", x),
                          _ptr(z), 0 if z is None else _gated_rows(z, "z", x), None, None, None, 0,
                          _gated_state(chunk_states, "chunk_states", x, gated_scan_states(B, T, D)),
                          dy.data_ptr(), _gated_rows(dy, "dy", x), _gated_state(d_last, "d_last", x), _gated_state(d_h0, "d_h0", x),
                          d_x.data_ptr(), _gated_rows(d_x, "d_x", x), d_f.data_ptr(), _gated_rows(d_f, "d_f", x),
                          _ptr(d_z), 0 if d_z is None else _gated_rows(d_z, "d_z", x))
    workspace, a.workspace, a.workspace_bytes = _gated_workspace(workspace, x)
    _launch(ffi.lib().mamba_b200_gated_scan_bwd, dev, handle, C.byref(a))
    out = dict(d_x=d_x, d_f=d_f, d_h0=d_h0)
    if d_z is not None:
        out["d_z"] = d_z
    return out


def _head_strides(t, name, shape, dtype):
    """Strides of batch, step and head of a [B, T, heads, width] view with contiguous columns."""
    if t.dtype != dtype or t.shape != shape:
        raise TypeError(f"{name} is {list(shape)} {dtype}, not {list(t.shape)} {t.dtype}")
    b, s, h, one = t.stride()
    if one != 1 and shape[3] > 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    return b, s, h


def _written(t, name):
    """Refuses an output whose elements share memory (an expanded view)."""
    if 0 in t.stride() and t.numel() and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name}: an expanded tensor cannot be written")


def _heads_of(t, B, T, heads, width):
    """A contiguous [B, T, heads, width] like t (half the host time of torch.empty)."""
    row = heads * width
    return torch.empty_strided((B, T, heads, width), (T * row, row, width, 1), dtype=t.dtype, device=t.device)


def _attention_args(q, k, v, decay, scale, state):
    """LinearAttentionArgs with what forward and backward share, and the shape of a state."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v are [B, T, heads, width]")
    dtype = q.dtype
    B, T, Hq, K = qs = q.shape
    Hk = k.shape[2]
    _, _, Hv, V = v.shape
    if decay.dtype != torch.float32 or decay.dim() != 1 or not decay.is_contiguous():
        raise TypeError("decay is contiguous float32 [heads]")
    H = decay.shape[0]
    for n, h in (("q", Hq), ("k", Hk), ("v", Hv)):
        if h < 1 or H % h:
            raise ValueError(f"{n}: {h} heads are not shared by {H} evenly")
    if not 1 <= K <= 256 or not 1 <= V <= 256:
        raise ValueError(f"K {K} and V {V} are 1 to 256")
    shape = (B, H, K, V)
    a = ffi.LinearAttentionArgs(dtype_code(dtype), B, T, H, K, V, Hq, Hk, Hv, K ** -0.5 if scale is None else scale, decay.data_ptr(),
                                q.data_ptr(), *_head_strides(q, "q", qs, dtype), k.data_ptr(), *_head_strides(k, "k", (B, T, Hk, K), dtype),
                                v.data_ptr(), *_head_strides(v, "v", (B, T, Hv, V), dtype), _attention_state(state, "state", shape))
    return a, shape


def _attention_state(t, name, shape):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise TypeError(f"{name} is contiguous float32 {list(shape)}")
    return t.data_ptr()


def _scratch(a, need, workspace, like):
    """Gives an argument struct its workspace (the caller's, or one made here); the tensor has to outlive the call."""
    if workspace is None:
        if not need:
            return None
        workspace = torch.empty(need, dtype=torch.uint8, device=like.device)
    elif not workspace.is_contiguous():
        raise ValueError("the workspace is contiguous")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return workspace


def linear_attention_workspace_bytes(B, T, H, K, V, *, Hq=None, Hk=None, Hv=None, backward=False) -> int:
    """Bytes of the scratch of linear_attention_fwd (backward: _bwd): states between the segments that a long text of few heads
    is cut into, and the parts of shared heads' gradients.  0: none is needed."""
    a = ffi.LinearAttentionArgs(B=B, T=T, H=H, K=K, V=V, Hq=Hq or H, Hk=Hk or H, Hv=Hv or H)
    return int(ffi.lib().mamba_b200_linear_attention_workspace_bytes(C.byref(a), int(backward)))


def linear_attention_fwd(q, k, v, decay, *, scale=None, state=None, state_out=None, o=None, workspace=None, handle=None):
    """Linear attention with a decay for each head: S_t = exp(decay) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t.
    q [B,T,Hq,K], k [B,T,Hk,K], v [B,T,Hv,V] in a storage dtype with any strides of batch, step and head; decay [H] f32, the log of
    each head's factor a token; Hq, Hk and Hv divide H (fewer heads are shared by consecutive ones); K, V <= 256; scale: K ** -0.5
    if None.  state [B,H,K,V] f32 enters (zeros if None), state_out receives what leaves (may be state).  workspace: scratch of
    linear_attention_workspace_bytes(...) bytes (made here if None).  Returns o [B,T,H,V] in q's dtype.  An infinite or NaN input
    changes no earlier token's output; what depends on it may be NaN where the formula has an infinity.  16-bit types keep a state that
    leaves in more digits than one that does not, so the last bits of o depend on whether state_out is asked for."""
    dev = _device_index(q, k, v, decay, state, state_out, o, workspace)
    a, shape = _attention_args(q, k, v, decay, scale, state)
    B, H, _, V = shape
    T = q.shape[1]
    if o is None:
        o = _heads_of(q, B, T, H, V)
        a.o_b, a.o_t, a.o_h = T * H * V, H * V, V
    else:
        a.o_b, a.o_t, a.o_h = _head_strides(o, "o", (B, T, H, V), q.dtype)
        _written(o, "o")
    a.o = o.data_ptr()
    a.state_out = _attention_state(state_out, "state_out", shape)
    lib = ffi.lib()
    if T > 1:
        workspace = _scratch(a, lib.mamba_b200_linear_attention_workspace_bytes(C.byref(a), 0), workspace, q)
    _launch(lib.mamba_b200_linear_attention_fwd, dev, handle, C.byref(a))
    return o


def linear_attention_step(q, k, v, decay, state, *, scale=None, state_out=None, o=None, handle=None):
    """One token for each sequence: q [B,Hq,K], k [B,Hk,K], v [B,Hv,V], o [B,H,V]; the state [B,H,K,V] f32 is updated in place, or
    state_out receives it."""
    dev = _device_index(q, k, v, decay, state, state_out, o)
    dtype = q.dtype
    B, Hq, K = q.shape
    (_, Hk, K2), (_, Hv, V), H = k.shape, v.shape, decay.shape[0]
    if k.dtype != dtype or v.dtype != dtype or k.shape[0] != B or v.shape[0] != B or K2 != K:
        raise TypeError(f"k and v have q's dtype and sequences, k its width: {list(q.shape)} {dtype}")
    if decay.dtype != torch.float32 or decay.dim() != 1 or not decay.is_contiguous():
        raise TypeError("decay is contiguous float32 [heads]")
    shape = (B, H, K, V)
    for t, name in ((state, "state"), (state_out, "state_out")):
        if t is not None and (t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous()):
            raise TypeError(f"{name} is contiguous float32 {list(shape)}")
    if o is None:
        o = torch.empty_strided((B, H, V), (H * V, V, 1), dtype=dtype, device=q.device)
    elif o.dtype != dtype or o.shape != (B, H, V):
        raise TypeError(f"o is {[B, H, V]} {dtype}")
    else:
        _written(o, "o")

    def at(t, name):
        b, h, one = t.stride()
        if one != 1 and t.shape[2] > 1:
            raise ValueError(f"{name}: last dimension must be contiguous")
        return t.data_ptr(), b, 0, h

    s = state.data_ptr()
    a = ffi.LinearAttentionArgs(dtype_code(dtype), B, 1, H, K, V, Hq, Hk, Hv, K ** -0.5 if scale is None else scale, decay.data_ptr(),
                                *at(q, "q"), *at(k, "k"), *at(v, "v"), s, s if state_out is None else state_out.data_ptr(), *at(o, "o"))
    _launch(ffi.lib().mamba_b200_linear_attention_fwd, dev, handle, C.byref(a))
    return o


def linear_attention_bwd(q, k, v, do, decay, *, scale=None, state=None, d_state_out=None, d_q=None, d_k=None, d_v=None, d_state=None,
                         workspace=None, handle=None):
    """Backward of linear_attention_fwd from its inputs alone.  do [B,T,H,V] in q's dtype, d_state_out [B,H,K,V] f32 the gradient of the
    state that left (zeros if None).  Returns dict(d_q, d_k, d_v) in q's dtype (they may be given: columns of one projection's
    gradient, say; those of shared heads are sums) and, with a state or a d_state to fill, d_state f32, the gradient of the state that
    entered.  The decays have no gradient here."""
    dev = _device_index(q, k, v, do, decay, state, d_state_out, d_q, d_k, d_v, d_state, workspace)
    a, shape = _attention_args(q, k, v, decay, scale, state)
    B, H, _, V = shape
    new = lambda t, like: _heads_of(like, *like.shape) if t is None else t  # noqa: E731
    d_q, d_k, d_v = new(d_q, q), new(d_k, k), new(d_v, v)
    if d_state is None and state is not None:
        d_state = torch.empty(shape, dtype=torch.float32, device=q.device)
    a.d_o = do.data_ptr()
    a.do_b, a.do_t, a.do_h = _head_strides(do, "do", (B, q.shape[1], H, V), q.dtype)
    a.d_state_out, a.d_state = _attention_state(d_state_out, "d_state_out", shape), _attention_state(d_state, "d_state", shape)
    a.d_q, (a.dq_b, a.dq_t, a.dq_h) = d_q.data_ptr(), _head_strides(d_q, "d_q", q.shape, q.dtype)
    a.d_k, (a.dk_b, a.dk_t, a.dk_h) = d_k.data_ptr(), _head_strides(d_k, "d_k", k.shape, q.dtype)
    a.d_v, (a.dv_b, a.dv_t, a.dv_h) = d_v.data_ptr(), _head_strides(d_v, "d_v", v.shape, q.dtype)
    for t, n in ((d_q, "d_q"), (d_k, "d_k"), (d_v, "d_v")):
        _written(t, n)
    lib = ffi.lib()
    workspace = _scratch(a, lib.mamba_b200_linear_attention_workspace_bytes(C.byref(a), 1), workspace, q)
    _launch(lib.mamba_b200_linear_attention_bwd, dev, handle, C.byref(a))
    out = dict(d_q=d_q, d_k=d_k, d_v=d_v)
    if d_state is not None:
        out["d_state"] = d_state
    return out


def rotary_frequencies(dim, base=10000.0, *, scaling=None, factor=1.0, trained=None, beta_fast=32.0, beta_slow=1.0, device=None):
    """(inv_freq f32 [dim / 2], scale) for rotary_fwd: base ** (-2 i / dim) for pair i, for texts `factor` times as long as the `trained`
    ones by scaling
      "linear"  positions interpolated: every frequency divided by factor
      "ntk"     a larger base, so that the slowest pair is divided by factor and the fastest stays (dim > 2)
      "yarn"    pairs of more than beta_fast turns over `trained` positions stay, those of less than beta_slow are divided by factor, a
                ramp between; scale = 0.1 ln(factor) + 1, once for q and once for k (Peng et al., YaRN, 2023, equations 17 to 22)
    Computed in 64 bits on the host, rounded once."""
    if dim < 2 or dim % 2:
        raise ValueError(f"{dim} columns are no pairs")
    if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError(f"base {base} and factor {factor} are positive")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("one pair has no slowest one beside its fastest")
        base = base * factor ** (dim / (dim - 2))
    pair = torch.arange(dim // 2, dtype=torch.float64)
    freq, scale = base ** (-2.0 * pair / dim), 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if trained is None or trained < 1 or base <= 1 or not 0 < beta_slow < beta_fast:
            raise ValueError("yarn needs the length trained on, a base above 1, and beta_slow below beta_fast")
        # the pair that makes n turns over the trained length: trained * base ** (-2 i / dim) = 2 pi n
        at = [dim * math.log(trained / (2 * math.pi * n)) / (2 * math.log(base)) for n in (beta_fast, beta_slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        slow = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * slow + freq * (1 - slow)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq.to(torch.float32).to(device or "cpu"), scale


def _rotary(q, k, positions, inv_freq, interleaved, scale, inverse, q_out, k_out, handle):
    dev = _device_index(q, k, positions, inv_freq, q_out, k_out)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k are [B, T, heads, width]")
    dtype = q.dtype
    B, T, Hq, D = qs = q.shape
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() or 2 * inv_freq.shape[0] > D:
        raise TypeError(f"inv_freq is contiguous float32 of at most {D // 2} pairs")
    if positions.dtype != torch.int32 or not positions.is_contiguous() or positions.shape not in ((T,), (B, T)):
        raise TypeError(f"positions are contiguous int32 [{T}] or [{B}, {T}]")

    def result(out, name, heads, shape):
        if out is None:
            return _heads_of(q, B, T, heads, D), (T * heads * D, heads * D, D)
        _written(out, name)
        return out, _head_strides(out, name, shape, dtype)

    q_out, to = result(q_out, "q_out", Hq, qs)
    ks, Hk = (), 0
    if k is not None:
        shape = B, T, Hk, D = (B, T, k.shape[2], D)
        k_in = _head_strides(k, "k", shape, dtype)
        k_out, k_to = result(k_out, "k_out", Hk, shape)
        ks = (k.data_ptr(), *k_in, k_out.data_ptr(), *k_to)
    a = ffi.RotaryArgs(dtype_code(dtype), B, T, Hq, Hk, D, 2 * inv_freq.shape[0], bool(interleaved), inverse, scale, positions.data_ptr(),
                       T if positions.dim() == 2 else 0, inv_freq.data_ptr(), q.data_ptr(), *_head_strides(q, "q", qs, dtype),
                       q_out.data_ptr(), *to, *ks)
    _launch(ffi.lib().mamba_b200_rotary, dev, handle, C.byref(a))
    return q_out, k_out


def rotary_fwd(q, k, positions, inv_freq, *, interleaved=False, scale=1.0, q_out=None, k_out=None, handle=None):
    """Rotation by position: pair i of each head's first 2 len(inv_freq) columns is turned by positions * inv_freq[i] (64 bits before
    sine and cosine) and multiplied by scale; the columns behind are handed on.  Pairs are columns 2i, 2i + 1 (interleaved) or i and
    i + len(inv_freq).  q [B,T,Hq,D], k [B,T,Hk,D] (or None) in a storage dtype with any strides of batch, step and head; positions int32
    [T] or [B,T]; inv_freq f32 (rotary_frequencies makes one).  q_out / k_out may be q / k themselves.  Returns (q_out, k_out)."""
    return _rotary(q, k, positions, inv_freq, interleaved, scale, False, q_out, k_out, handle)


def rotary_bwd(d_q, d_k, positions, inv_freq, *, interleaved=False, scale=1.0, q_out=None, k_out=None, handle=None):
    """Gradients of rotary_fwd's q and k from those of its results: the rotation the other way, with the same scale."""
    return _rotary(d_q, d_k, positions, inv_freq, interleaved, scale, True, q_out, k_out, handle)


def group_norm_workspace_bytes(N, S, C_, G, backward=False) -> int:
    """Bytes of the scratch of group_norm_fwd (backward: _bwd): sums of blocks of rows."""
    return int(ffi.lib().mamba_b200_group_norm_workspace_bytes(N, S, C_, G, int(backward)))


def _norm_rows(t, name, like):
    """Row stride of an [N, S, C] (or [N, C]) view whose rows are one after another."""
    if t.dtype != like.dtype or t.shape != like.shape:
        raise TypeError(f"{name} has x's dtype and shape: {list(like.shape)} {like.dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    C_ = t.shape[-1]
    if t.dim() == 2:
        return t.stride(0) if t.shape[0] > 1 else C_
    N, S = t.shape[:2]
    if S <= 1:
        return t.stride(0) if N > 1 and S else C_
    if N > 1 and t.stride(0) != S * t.stride(1):
        raise ValueError(f"{name}: sample stride must equal S * row stride")
    return t.stride(1)


def _rows_like(x):
    """A contiguous tensor of x's shape and dtype."""
    if x.dim() == 2:
        return torch.empty_strided(x.shape, (x.shape[1], 1), dtype=x.dtype, device=x.device)
    _, S, C_ = x.shape
    return torch.empty_strided(x.shape, (S * C_, C_, 1), dtype=x.dtype, device=x.device)


def _norm_args(x, z, weight, bias, groups, activation, eps):
    if x.dim() not in (2, 3):
        raise ValueError("x is [N, S, C] or [N, C]")
    shape = x.shape
    N, C_ = shape[0], shape[-1]
    if groups < 1 or C_ < 1 or C_ % groups:
        raise ValueError(f"{C_} channels are no {groups} groups")
    if activation not in ffi.ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    for t, n in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.dtype != torch.float32 or t.shape != (C_,) or not t.is_contiguous()):
            raise TypeError(f"{n} is contiguous float32 [{C_}]")
    return ffi.GroupNormArgs(dtype_code(x.dtype), N, 1 if len(shape) == 2 else shape[1], C_, groups, ffi.ACTIVATIONS[activation], eps,
                             x.data_ptr(), _norm_rows(x, "x", x), _ptr(z), 0 if z is None else _norm_rows(z, "z", x), _ptr(weight), _ptr(bias))


def group_norm_fwd(x, weight, bias, groups, *, eps=1e-5, activation=None, z=None, y=None, stats=None, workspace=None, handle=None):
    """Group norm with channels last: y = act((x - mean) / sqrt(var + eps) * weight + bias) * SiLU(z).  x, z, y [N,S,C] in a storage dtype
    (any row stride), mean and var over a sample's S rows and the C / groups channels of a group; [N,C] is S = 1, each row by itself
    (a group for each head, say).  weight, bias [C] f32 or None; activation None, "silu" or "gelu" (by erf); z None: no gate.  y may be
    x or z.
    Returns (y, stats): mean and rstd f32 [2,N,groups], which group_norm_bwd takes."""
    dev = _device_index(x, weight, bias, z, y, stats, workspace)
    a = _norm_args(x, z, weight, bias, groups, activation, eps)
    N = a.N
    if y is None:
        y, a.ld_y = _rows_like(x), a.C
    else:
        a.ld_y = _norm_rows(y, "y", x)
        _written(y, "y")
    if stats is None:
        stats = torch.empty_strided((2, N, groups), (N * groups, groups, 1), dtype=torch.float32, device=x.device)
    elif stats.dtype != torch.float32 or stats.shape != (2, N, groups) or not stats.is_contiguous():
        raise TypeError(f"stats is contiguous float32 {[2, N, groups]}")
    a.stats, a.y = stats.data_ptr(), y.data_ptr()
    lib = ffi.lib()
    workspace = _scratch(a, lib.mamba_b200_group_norm_workspace_bytes(a.N, a.S, a.C, a.G, 0), workspace, x)
    _launch(lib.mamba_b200_group_norm_fwd, dev, handle, C.byref(a))
    return y, stats


def group_norm_bwd(dy, x, stats, weight, bias, groups, *, activation=None, z=None, d_x=None, d_z=None, d_weight=None, d_bias=None,
                   workspace=None, handle=None):
    """Backward of group_norm_fwd from its inputs and stats.  Returns dict(d_x, d_weight, d_bias f32 [C], d_z (with z)).  d_x and d_z may
    be given and are overwritten (d_x may be dy or x, d_z may be z); d_weight and d_bias, given both, are added to (a gradient arena),
    else made."""
    dev = _device_index(x, dy, stats, weight, bias, z, d_x, d_z, d_weight, d_bias, workspace)
    a = _norm_args(x, z, weight, bias, groups, activation, 0.0)
    if stats.dtype != torch.float32 or stats.shape != (2, a.N, groups) or not stats.is_contiguous():
        raise TypeError(f"stats is contiguous float32 {[2, a.N, groups]}")
    if (d_weight is None) != (d_bias is None):
        raise ValueError("d_weight and d_bias are given both or neither")
    if d_weight is None:
        d_weight = torch.empty_strided((a.C,), (1,), dtype=torch.float32, device=x.device)
        d_bias = torch.empty_like(d_weight)
    else:
        a.accumulate = 1
        for t, n in ((d_weight, "d_weight"), (d_bias, "d_bias")):
            if t.dtype != torch.float32 or t.shape != (a.C,) or not t.is_contiguous():
                raise TypeError(f"{n} is contiguous float32 [{a.C}]")
    new = lambda t: _rows_like(x) if t is None else t  # noqa: E731
    d_x = new(d_x)
    a.stats, a.dy, a.ld_dy = stats.data_ptr(), dy.data_ptr(), _norm_rows(dy, "dy", x)
    a.d_x, a.ld_dx, a.d_weight, a.d_bias = d_x.data_ptr(), _norm_rows(d_x, "d_x", x), d_weight.data_ptr(), d_bias.data_ptr()
    _written(d_x, "d_x")
    out = dict(d_x=d_x, d_weight=d_weight, d_bias=d_bias)
    if z is not None:
        out["d_z"] = d_z = new(d_z)
        a.d_z, a.ld_dz = d_z.data_ptr(), _norm_rows(d_z, "d_z", x)
        _written(d_z, "d_z")
    lib = ffi.lib()
    workspace = _scratch(a, lib.mamba_b200_group_norm_workspace_bytes(a.N, a.S, a.C, a.G, 1), workspace, x)
    _launch(lib.mamba_b200_group_norm_bwd, dev, handle, C.byref(a))
    return out
