"""Linear attention, rotation and group norm at the boundary: laid out alike on both sides, refused without a device; the tables of
frequencies, which the host makes."""
import ctypes
import math
import os
import re
import subprocess

import pytest

import mamba_rs_b200 as mb
from mamba_rs_b200 import ffi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mamba_b200.h")


@pytest.mark.parametrize("cls,name", [(ffi.LinearAttentionArgs, "linear_attention"), (ffi.RotaryArgs, "rotary"), (ffi.GroupNormArgs, "group_norm")])
def test_argument_structs_are_laid_out_alike(tmp_path, cls, name):
    name = f"mamba_b200_{name}_args"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({name}));']
    lines += [f'printf("%zu\\n", offsetof({name}, {n}));' for n, _ in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.check_call(["gcc", "-std=c11", "-o", str(tmp_path / "t"), str(src)])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, n).offset for n, _ in cls._fields_]
    # and no member is missing
    body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name, open(HEADER).read(), re.S).group(1)
    members = re.findall(r"(\w+)\s*(?=[,;])", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
    assert members == [n for n, _ in cls._fields_]


def test_every_entry_point_is_bound_and_null_is_an_error():
    lib = ffi.lib()
    for name in set(re.findall(r"\b(mamba_b200_(?:linear|rotary|group)\w*)\s*\(", open(HEADER).read())):
        assert getattr(lib, name).argtypes, name
    for name, cls in (("linear_attention_fwd", ffi.LinearAttentionArgs), ("linear_attention_bwd", ffi.LinearAttentionArgs), ("rotary", ffi.RotaryArgs),
                      ("group_norm_fwd", ffi.GroupNormArgs), ("group_norm_bwd", ffi.GroupNormArgs)):
        a = cls()
        assert getattr(lib, "mamba_b200_" + name)(None, None, ctypes.byref(a)) < 0
    assert lib.mamba_b200_linear_attention_workspace_bytes(None, 0) == 0


def test_sizes_without_a_device():
    big = 2 ** 31 - 1
    assert mb.linear_attention_workspace_bytes(1, 1, 1, 64, 64) == 0
    assert mb.linear_attention_workspace_bytes(1, 100000, 1, 64, 64) > 0 == mb.linear_attention_workspace_bytes(64, 100000, 16, 64, 64)
    # parts of shared heads, f32
    assert mb.linear_attention_workspace_bytes(64, 10, 16, 64, 32, Hk=4, backward=True) == 64 * 10 * 16 * 64 * 4
    for bad in ((0, 1, 1, 1, 1), (1, big, 1, 8, 8), (1, 8, 1, 257, 8), (1, 8, 1, 8, 257), (big, 8, big, 8, 8), (1, -1, 1, 8, 8)):
        assert mb.linear_attention_workspace_bytes(*bad, backward=True) == 0
    assert mb.group_norm_workspace_bytes(10, 1, 64, 4) == 0 < mb.group_norm_workspace_bytes(10, 1, 64, 4, backward=True)
    for bad in ((1, big, 8, 1), (1, 1, 8, 3), (0, 1, 8, 1), (1, 1, 0, 1), (1, 1, 8, 0)):
        assert mb.group_norm_workspace_bytes(*bad, backward=True) == 0
    # a scratch does not grow with the rows without bound
    assert mb.group_norm_workspace_bytes(100000, 1, 2048, 32, backward=True) < 2 ** 24


def test_compute_refuses_cpu_tensors():
    import torch
    x = torch.zeros(1, 4, 2, 8)
    f, s, n = torch.zeros(2), torch.zeros(1, 2, 8, 8), torch.zeros(2, 1, 2)
    for call in (lambda: mb.linear_attention_fwd(x, x, x, f), lambda: mb.linear_attention_step(x[0], x[0], x[0], f, s),
                 lambda: mb.linear_attention_bwd(x, x, x, x, f), lambda: mb.rotary_fwd(x, x, f.int(), f), lambda: mb.rotary_bwd(x, None, f.int(), f),
                 lambda: mb.group_norm_fwd(x[0], None, None, 2), lambda: mb.group_norm_bwd(x[0], x[0], n, None, None, 2)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_frequencies():
    import torch
    f, scale = mb.rotary_frequencies(8)
    assert f.dtype == torch.float32 and scale == 1.0 and f.tolist() == torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64).float().tolist()
    assert torch.equal(mb.rotary_frequencies(8, scaling="linear", factor=4.0)[0], torch.tensor([0.25, 0.025, 0.0025, 0.00025], dtype=torch.float64).float())
    f, _ = mb.rotary_frequencies(64, scaling="ntk", factor=8.0)
    plain = mb.rotary_frequencies(64)[0].double()
    assert f[0] == 1.0 and abs(float(f[-1] * 8 / plain[-1]) - 1) < 2.0 ** -22
    # fast pairs as they were, slow ones divided, between them a ramp; turns over the trained length tell which
    f, scale = mb.rotary_frequencies(128, scaling="yarn", factor=16.0, trained=4096)
    plain = mb.rotary_frequencies(128)[0].double()
    turns, ratio = 4096 * plain / (2 * math.pi), f.double() / plain
    assert ((ratio[turns > 40] - 1).abs() < 2.0 ** -22).all() and ((ratio[turns < 0.8] - 1 / 16).abs() < 2.0 ** -22).all()
    assert (ratio.diff() <= 2.0 ** -22).all() and ((ratio > 0.1) & (ratio < 0.9)).sum() > 5
    assert scale == 0.1 * math.log(16.0) + 1.0
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, base=-1.0), dict(dim=8, factor=0.0), dict(dim=2, scaling="ntk"),
                dict(dim=8, scaling="yarn"), dict(dim=8, scaling="yarn", trained=8, beta_slow=33.0)):
        with pytest.raises(ValueError):
            mb.rotary_frequencies(**bad)
