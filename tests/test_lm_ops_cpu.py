"""The token table, token log probabilities and the gated scan at the boundary: exported, laid out alike on both sides,
refused where there is no device."""
import ctypes
import os
import re
import subprocess

import pytest

import mamba_rs_b200 as mb
from mamba_rs_b200 import ffi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mamba_b200.h")


def test_argument_struct_is_laid_out_alike(tmp_path):
    cls, name = ffi.GatedScanArgs, "mamba_b200_gated_scan_args"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'printf("%zu\\n", sizeof({name}));',
             'printf("%d\\n", MAMBA_B200_GATED_SCAN_SAVE);']
    lines += [f'printf("%zu\\n", offsetof({name}, {n}));' for n, _ in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.check_call(["gcc", "-std=c11", "-o", str(tmp_path / "t"), str(src)])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    assert got == [ctypes.sizeof(cls), ffi.GATED_SCAN_SAVE] + [getattr(cls, n).offset for n, _ in cls._fields_]


def test_every_entry_point_is_bound():
    declared = re.findall(r"\b(mamba_b200_(?:embedding|token|gated)\w*)\s*\(", open(HEADER).read())
    lib = ffi.lib()
    for name in set(declared) - {"mamba_b200_embedding_gather"}:
        assert getattr(lib, name).argtypes, name


def test_null_handles_are_an_error_not_a_crash():
    lib = ffi.lib()
    assert lib.mamba_b200_embedding_fwd(None, None, 0, None, 1, None, 0, None, 1, 1, 1, 1, 1.0) < 0
    assert lib.mamba_b200_embedding_bwd(None, None, 0, None, 1, None, None, 0, 1, 1, 1, 1.0, None, 0) < 0
    assert lib.mamba_b200_token_logprobs(None, None, 0, None, 1, None, 1.0, None, None, None, 0, None, None, 1, 1) < 0
    assert lib.mamba_b200_token_logprobs_bwd(None, None, 0, None, 1, None, 1.0, None, None, None, None, None, 1, 1, 1) < 0
    a = ffi.GatedScanArgs()
    assert lib.mamba_b200_gated_scan_fwd(None, None, ctypes.byref(a)) < 0
    assert lib.mamba_b200_gated_scan_bwd(None, None, ctypes.byref(a)) < 0


def test_sizes_without_a_device():
    assert mb.gated_scan_states(2, 0, 8) == (2, 0, 8)
    assert mb.gated_scan_states(2, 64, 8) == (2, 1, 8) and mb.gated_scan_states(2, 65, 8) == (2, 2, 8)
    for rows, dim, vocab in ((0, 1, 1), (1, 1, 1), (65536, 2560, 50280), (2 ** 31 - 1, 64, 2 ** 31 - 1)):
        assert mb.embedding_bwd_workspace_bytes(rows, dim, vocab) >= 0


def test_compute_refuses_cpu_tensors():
    import torch
    t, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: mb.embedding_fwd(t, ids), lambda: mb.embedding_bwd(ids, t, 4), lambda: mb.token_logprobs(t, ids),
                 lambda: mb.token_logprobs_bwd(t, ids, t[:, 0], t[:, 0]), lambda: mb.gated_scan_fwd(t[None], t[None]),
                 lambda: mb.gated_scan_step(t, t, t), lambda: mb.gated_scan_bwd(t[None], t[None], t[None], t[None])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
