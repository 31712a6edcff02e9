"""CPU only: the serving operators at the ends of what they take: the columns their loads touch, scratch and grids of calls
of unusual shape, what their outputs must not share, tensors that carry gradients."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from test_serving_host import P, Packed, refused

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def test_loads_stay_inside_their_rows(tmp_path):
    """tests/native/serving_columns_test.cpp: the columns that decoding loads of a cache row, load widths included."""
    exe = str(tmp_path / "serving_columns_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                           os.path.join(ROOT, "tests", "native", "serving_columns_test.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("q_heads", [1, 2, 4, 8, 16])
def test_scratch_of_packed_prompts_follows_from_sizes(fa, q_heads, causal):
    """The size query gives one answer for the same sizes, whichever offsets the call comes with, and the call takes
    scratch of that size (the launch itself is kept from happening by an address that is not aligned)."""
    L = fa.lib()
    for n in (1536, 1700, 2048, 3000, 4095):
        for sequences in (1, 2, 3, 8):
            a = dict(q=P, k=P, v=P, o=P, sequences=sequences, total_q=n, total_k=n, q_heads=q_heads, kv_heads=1, d=64, qt=q_heads * 64, qh=64, kt=64,
                     kh=64, vt=64, vh=64, ot=q_heads * 64, oh=64, softmax_scale=0.125, causal=causal, dtype=0)
            need = L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**a)))
            assert need < 70 << 20
            for cu in (dict(cu_q=P, cu_k=P), dict(cu_q=P, cu_k=P + 4096)):
                call = Packed(**a, **cu)
                assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(call)) == need
                assert refused(fa, L.flash_fwd_packed(ctypes.byref(call), P + 8, need, None), "aligned")
                if need > 0:
                    assert refused(fa, L.flash_fwd_packed(ctypes.byref(call), P + 8, need - 1, None), "too small")
