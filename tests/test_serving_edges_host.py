"""CPU only: the serving operators at the ends of what they take: the columns their loads touch, scratch and grids of calls
of unusual shape, what their outputs must not share, tensors that carry gradients."""
import ctypes
import importlib.util
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from test_serving_host import P, Append, Packed, cache, refused

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


def test_grids_that_no_launch_takes_are_refused(fa):
    """2^24 workgroups of 256 threads and more along one dimension."""
    L = fa.lib()
    a = dict(q=P, k=P, v=P, o=P, cu_q=P, cu_k=P, total_q=6, total_k=6, q_heads=4, kv_heads=2, d=64, qt=256, qh=64, kt=128, kh=64, vt=128,
             vh=64, ot=256, oh=64, softmax_scale=0.125, causal=1, dtype=0)
    for sequences in (1 << 24, 1 << 30):
        assert refused(fa, L.flash_fwd_packed(ctypes.byref(Packed(**a, sequences=sequences)), None, 0, None), "too many")
        assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**a, sequences=sequences))) == -1
    for sequences, heads in ((1 << 20, 64), ((1 << 24) - 1, 4), (1, 4)):      # heads have a dimension of their own
        call = Packed(**{**a, "sequences": sequences, "q_heads": heads, "qt": heads * 64, "ot": heads * 64})
        assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(call)) == 0
        assert refused(fa, L.flash_fwd_packed(ctypes.byref(call), P + 8, 0, None), "aligned")
    one_row = dict(k=P, v=P, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, cu_seqlens=P, dtype=0)
    for tokens in ((1 << 29) - 32, 1 << 29, 1 << 30):
        x = Append(**one_row, tokens=tokens)
        assert refused(fa, L.flash_cache_append(ctypes.byref(x), ctypes.byref(cache()), None), "tokens")
    x = Append(**{**one_row, "k": P + 8}, tokens=(1 << 29) - 33)
    assert refused(fa, L.flash_cache_append(ctypes.byref(x), ctypes.byref(cache()), None), "16-byte")


def test_the_serving_operators_are_compiled_with_nans():
    """Masked places may hold NaN, and rows that see one are computed with it: no unit of theirs may be compiled as if there
    were none.  The pipelined kernel's running maximum, which would quiet every score, is one of integers there."""
    spec = importlib.util.spec_from_file_location("fa_build", os.path.join(ROOT, "flash-attention_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    for unit in ("flash_packed", "flash_serve"):
        for flag in build.HIP_FLAGS + build.HIP_UNITS[unit][0]:
            assert not any(x in flag for x in ("nans", "fast", "finite", "infinities")), (unit, flag)
    text = open(os.path.join(ROOT, "flash-attention_amd", "csrc", "flash_packed.hip")).read()
    assert text.index("#define FLASH_M16_HONOR_NANS") < text.index("#include")
