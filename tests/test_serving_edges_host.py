"""CPU only: the serving operators at the ends of what they take: the columns their loads touch, scratch and grids of calls
of unusual shape, what their outputs must not share, tensors that carry gradients."""
import os
import subprocess

import pytest
import torch

from conftest import ROOT

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def test_loads_stay_inside_their_rows(tmp_path):
    """tests/native/serving_columns_test.cpp: the columns that decoding loads of a cache row, load widths included."""
    exe = str(tmp_path / "serving_columns_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                           os.path.join(ROOT, "tests", "native", "serving_columns_test.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
