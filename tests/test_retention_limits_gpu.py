"""What the entry points of linear attention, rotation and group norm refuse before anything is launched.  The calls of the C entries here
lack a pointer that they need or ask for what no call may, so none of them could run."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu
NEAR = 2 ** 31 - 1 - 65535  # the first size that 32-bit loops could step past


@pytest.fixture()
def refused(cuda_dev):
    from mamba_rs_b200 import ffi
    h = ffi.default_handle(0)

    def call(name, a):
        rc = getattr(ffi.lib(), "mamba_b200_" + name)(h.ptr, None, C.byref(a))
        assert rc < 0
        return ffi.lib().mamba_b200_last_error(h.ptr).decode()
    return call


def attention(**kw):
    from mamba_rs_b200 import ffi
    return ffi.LinearAttentionArgs(**{**dict(dtype=0, B=1, T=2, H=1, K=8, V=8, Hq=1, Hk=1, Hv=1, scale=1.0), **kw})


def rotary(**kw):
    from mamba_rs_b200 import ffi
    return ffi.RotaryArgs(**{**dict(dtype=0, B=1, T=2, Hq=1, Hk=1, D=8, R=8, scale=1.0), **kw})


def norm(**kw):
    from mamba_rs_b200 import ffi
    C_ = kw.get("C", 8)
    return ffi.GroupNormArgs(**{**dict(dtype=0, N=1, S=2, C=C_, G=1, eps=1e-5, ld_x=C_, ld_z=C_, ld_y=C_, ld_dy=C_, ld_dx=C_, ld_dz=C_), **kw})


def test_sizes(refused):
    for big in (NEAR, 2 ** 31 - 1):
        for name in ("linear_attention_fwd", "linear_attention_bwd"):
            assert "too many steps" in refused(name, attention(T=big))
            assert "too many sequences" in refused(name, attention(B=big))
            assert "too many sequences" in refused(name, attention(H=big))
        assert "too many" in refused("rotary", rotary(T=big)) and "too many" in refused("rotary", rotary(B=big))
        for name in ("group_norm_fwd", "group_norm_bwd"):
            assert "too many" in refused(name, norm(N=big)) and "too many" in refused(name, norm(S=big)) and "too many" in refused(name, norm(C=big))
    for name in ("linear_attention_fwd", "linear_attention_bwd"):
        assert "null" in refused(name, attention(T=NEAR - 1)) and "null" in refused(name, attention(B=1000, H=1000, Hq=1000))
        assert "too many" in refused(name, attention(B=1001, H=1000))
        for bad in (dict(B=-1), dict(T=-1), dict(H=0), dict(K=0), dict(V=0), dict(K=257), dict(V=257)):
            assert "K" in refused(name, attention(**bad)), bad
        for bad in (dict(Hq=0), dict(Hk=-1), dict(H=6, Hv=4), dict(H=6, Hq=12)):
            assert "shared" in refused(name, attention(**bad)), bad
        assert "dtype" in refused(name, attention(dtype=7))
        for bad in (float("inf"), float("nan")):
            assert "scale" in refused(name, attention(scale=bad))
    for bad in (dict(R=7), dict(R=-2), dict(R=10)):
        assert "pairs" in refused("rotary", rotary(**bad))
    for bad in (dict(B=-1), dict(T=-1), dict(Hq=0), dict(D=0), dict(D=1025, R=0)):
        assert "heads" in refused("rotary", rotary(**bad)), bad
    assert "scale" in refused("rotary", rotary(scale=float("nan"))) and "dtype" in refused("rotary", rotary(dtype=-1))
    for name in ("group_norm_fwd", "group_norm_bwd"):
        for bad in (dict(N=-1), dict(S=-1), dict(C=0), dict(G=0), dict(G=3)):
            assert "N " in refused(name, norm(**bad)), bad
        assert "activation" in refused(name, norm(activation=9)) and "dtype" in refused(name, norm(dtype=9))
        for bad in (-1e-5, float("inf"), float("nan")):
            assert "eps" in refused(name, norm(eps=bad)), bad


def test_null_and_narrow(refused):
    from mamba_rs_b200 import ffi
    p = C.c_void_p(4096)
    need = {"linear_attention_fwd": (attention, ("decay", "q", "k", "v", "o")),
            "linear_attention_bwd": (attention, ("decay", "q", "k", "v", "d_o", "d_q", "d_k", "d_v")),
            "rotary": (rotary, ("positions", "inv_freq", "q", "q_out")),
            "group_norm_fwd": (norm, ("x", "y")), "group_norm_bwd": (norm, ("x", "dy", "d_x", "stats"))}
    for name, (make, pointers) in need.items():
        for missing in pointers:
            only = dict(Hk=0) if name == "rotary" else {}
            assert "null" in refused(name, make(**only, **{n: p for n in pointers if n != missing})), (name, missing)
    assert "null" in refused("rotary", rotary(positions=p, inv_freq=p, q=p, q_out=p, k=p))
    assert "null" in refused("group_norm_bwd", norm(x=p, dy=p, d_x=p, stats=p, z=p))
    for n in ("ld_x", "ld_y"):
        assert "narrower" in refused("group_norm_fwd", norm(x=p, y=p, **{n: 7}))
    for n in ("ld_x", "ld_dy", "ld_dx"):
        assert "narrower" in refused("group_norm_bwd", norm(x=p, dy=p, d_x=p, stats=p, **{n: 7}))
    assert "narrower" in refused("group_norm_fwd", norm(x=p, y=p, z=p, ld_z=7))
    # a workspace that is too small or starts between lines
    q = dict(decay=p, q=p, k=p, v=p, d_o=p, d_q=p, d_k=p, d_v=p)
    apart = {n: C.c_void_p(4096 * (i + 1)) for i, n in enumerate(q)}
    assert "need a workspace" in refused("linear_attention_bwd", attention(H=2, Hq=2, Hv=2, workspace=p, workspace_bytes=16, **apart))
    assert "misaligned workspace" in refused("linear_attention_fwd", attention(decay=p, q=p, k=p, v=p, o=p, workspace=C.c_void_p(4096 + 128)))
    assert "misaligned workspace" in refused("group_norm_bwd", norm(S=1, x=p, dy=p, d_x=p, stats=p, workspace=C.c_void_p(4096 + 128)))
    big = norm(S=100000, x=p, y=p)
    assert ffi.lib().mamba_b200_group_norm_workspace_bytes(1, 100000, 8, 1, 0) > 0 and "workspace" in refused("group_norm_fwd", big)
    assert "same memory" in refused("linear_attention_bwd", attention(d_state=p, d_state_out=p, **q))
    for t in ("q", "k"):
        a = dict(positions=p, inv_freq=p, q=p, q_out=C.c_void_p(8192), k=p, k_out=C.c_void_p(8192), q_t=8, k_t=8, qo_t=8, ko_t=8)
        assert "other strides" in refused("rotary", rotary(**{**a, t + "_out": p, t + "o_t": 16}))


def test_pointers_between_elements(refused):
    from mamba_rs_b200 import ffi
    p = C.c_void_p(4096)
    for dtype, odd in ((ffi.F32, 2), (ffi.BF16, 1), (ffi.F16, 1)):
        store, words = C.c_void_p(4096 + odd), C.c_void_p(4096 + 2)
        for name, make, stores, w in (("linear_attention_fwd", attention, ("q", "k", "v", "o"), ("decay", "state", "state_out")),
                                      ("linear_attention_bwd", attention, ("q", "k", "v", "d_o", "d_q", "d_k", "d_v"),
                                       ("decay", "state", "d_state", "d_state_out")),
                                      ("rotary", rotary, ("q", "q_out", "k", "k_out"), ("positions", "inv_freq")),
                                      ("group_norm_fwd", norm, ("x", "y", "z"), ("weight", "bias", "stats")),
                                      ("group_norm_bwd", norm, ("x", "dy", "d_x", "z", "d_z"), ("weight", "bias", "stats", "d_weight", "d_bias"))):
            base = {n: p for n in stores + tuple(n for n in w if n in ("decay", "positions", "inv_freq", "stats"))}
            for n in stores + w:
                assert "misaligned" in refused(name, make(dtype=dtype, **{**base, n: store if n in stores else words})), (name, n)


def test_results_in_the_place_of_what_others_read(refused):
    """(At one step more than the decode step's, at it, and for each pair; every other pointer is a place of its own.)"""
    def places(names):
        return {n: C.c_void_p(4096 * (i + 1)) for i, n in enumerate(names)}
    for T in (1, 2):
        p = places(("decay", "q", "k", "v", "o"))
        for n in ("q", "k", "v"):
            assert "same memory" in refused("linear_attention_fwd", attention(T=T, **{**p, "o": p[n]})), n
        p = places(("decay", "q", "k", "v", "d_o", "d_q", "d_k", "d_v"))
        for out in ("d_q", "d_k", "d_v"):
            for n in p:
                if n not in (out, "decay"):
                    assert "same memory" in refused("linear_attention_bwd", attention(T=T, **{**p, out: p[n]})), (out, n)
        p = places(("decay", "q", "k", "v", "d_o", "d_q", "d_k", "d_v", "state"))
        assert "same memory" in refused("linear_attention_bwd", attention(T=T, d_state=p["state"], **p))
    p = places(("positions", "inv_freq", "q", "q_out", "k", "k_out"))
    for out, n in (("q_out", "k"), ("k_out", "q"), ("q_out", "k_out")):
        assert "memory" in refused("rotary", rotary(**{**p, out: p[n]})), out
    p = places(("x", "dy", "stats", "z", "d_x", "d_z"))
    assert "same memory" in refused("group_norm_bwd", norm(**{**p, "d_z": p["d_x"]}))
