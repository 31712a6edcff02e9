"""CPU only: the serving operators at the ends of what they take: the columns their loads touch, scratch and grids of calls
of unusual shape, what their outputs must not share, tensors that carry gradients."""
import ctypes
import importlib.util
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from test_serving_host import P, Append, Decode, Packed, cache, caches, packed, paged, refused

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("name", ["serving_columns_test", "serving_overlap_test"])
def test_index_arithmetic(tmp_path, name):
    """tests/native/serving_columns_test.cpp: the columns that decoding loads of a cache row, load widths included;
    serving_overlap_test.cpp: rows of an output that share an element."""
    exe = str(tmp_path / name)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                           os.path.join(ROOT, "tests", "native", name + ".cpp"), "-o", exe])
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


def overlapping(shape, dtype=F16):
    """Tensors of this shape whose rows share memory."""
    room = torch.zeros(1 << 14, dtype=dtype)
    dense = torch.zeros(shape, dtype=dtype).stride()
    out = [torch.zeros((1,) + shape[1:], dtype=dtype).expand(shape)]
    for i in range(len(shape) - 1):
        out.append(room.as_strided(shape, dense[:i] + (0,) + dense[i + 1:]))       # one place for all of a dimension
        out.append(room.as_strided(shape, dense[:i] + (shape[-1] // 2,) + dense[i + 1:]))  # half a row further each
    return out


def test_outputs_whose_rows_overlap_are_refused(fa):
    for out in overlapping((6, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            fa.forward_packed(**packed(out=out))
    for out in overlapping((2, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            fa.decode_paged(**paged(out=out))
    # (the same strides are no reason to refuse what is read: these calls come as far as the device)
    for x in overlapping((5, 2, 16, 64)):
        with pytest.raises(ValueError, match="no CPU path"):
            fa.decode_paged(**paged(k_cache=x, v_cache=x))
    for out in (torch.zeros(6, 8, 64, dtype=F16)[:, ::2], torch.zeros(4, 6, 64, dtype=F16).transpose(0, 1), torch.zeros(6, 4, 72, dtype=F16)[..., :64]):
        with pytest.raises(ValueError, match="no CPU path"):
            fa.forward_packed(**packed(out=out))


def test_written_caches_whose_rows_overlap_are_refused(fa):
    L = fa.lib()
    a = Append(k=P, v=P, tokens=2, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, dtype=0)
    for change in (dict(page_stride=0), dict(head_stride=0), dict(slot_stride=0), dict(slot_stride=32), dict(head_stride=960), dict(page_stride=1024)):
        assert refused(fa, L.flash_cache_append(ctypes.byref(a), ctypes.byref(cache(**change)), None), "overlap"), change
    d = Decode(q=P, o=P, q_heads=4, q_batch_stride=256, q_head_stride=64, o_batch_stride=256, o_head_stride=64, softmax_scale=0.125, dtype=0)
    assert L.flash_decode_paged_workspace_bytes(ctypes.byref(d), ctypes.byref(cache(page_stride=0))) > 0      # read only
    for change in (dict(o_batch_stride=0), dict(o_head_stride=0), dict(o_batch_stride=192), dict(o_head_stride=56)):
        bad = Decode(**{f: getattr(d, f) for f, _ in Decode._fields_ if f not in change}, **change)
        assert refused(fa, L.flash_decode_paged(ctypes.byref(bad), ctypes.byref(cache()), P, 1 << 40, None), "overlap"), change
    # layouts as caches have them: heads or tokens first, K and V side by side, a layer of several
    for change in (dict(head_stride=64, slot_stride=128), dict(head_stride=2048, slot_stride=128, page_stride=4096),
                   dict(page_stride=1 << 30), dict(head_stride=5 * 16 * 64, page_stride=16 * 64)):
        y = Append(k=P, v=P, tokens=0, cu_seqlens=P, dtype=0)
        assert L.flash_cache_append(ctypes.byref(y), ctypes.byref(cache(**change)), None) == 0


E4M3_CACHES = caches(5, 2, 16, 64, dtype=E4M3)


@pytest.mark.parametrize("how", ["backward", "forward"])
@pytest.mark.parametrize("call,name,tensor", [
    ("forward_packed", "q", None), ("forward_packed", "v", None), ("forward_packed", "out", torch.zeros(6, 4, 64, dtype=F16)),
    ("decode_paged", "q", None), ("decode_paged", "v_cache", None), ("decode_paged", "out", torch.zeros(2, 4, 64, dtype=F16)),
    ("decode_paged", "k_scale", torch.ones(2)), ("decode_paged", "v_scale", torch.ones(2)), ("decode_paged", "workspace", torch.zeros(1 << 22)),
    ("cache_append", "k", torch.zeros(2, 2, 64, dtype=F16)), ("cache_append", "v_cache", None), ("cache_append", "k_scale", torch.ones(2)),
])
def test_tensors_that_carry_gradients_are_refused(fa, call, name, tensor, how):
    """Whatever the argument: a gradient that would not be computed, or a tangent that would be lost."""
    a = packed() if call == "forward_packed" else paged(**(E4M3_CACHES if "scale" in name else {}))
    if call == "cache_append":
        a.pop("q")
        a.update(k=torch.zeros(2, 2, 64, dtype=F16), v=torch.zeros(2, 2, 64, dtype=F16))
    x = (a[name] if tensor is None else tensor).detach().clone()
    run = getattr(fa, call)
    if how == "backward":
        a[name] = x.requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            run(**a)
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            run(**a)
    else:
        with torch.autograd.forward_ad.dual_level():
            a[name] = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(ValueError, match="forward-mode"):
                run(**a)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                run(**a)
            a[name] = x
            with pytest.raises(ValueError, match="no CPU path"):
                run(**a)


@pytest.mark.parametrize("name", ["forward_packed", "decode_paged"])
def test_schemas_say_what_results_alias(fa, name):
    """A result is a new tensor, or, in the form of its own that takes an output, that output."""
    fa.load_pyflash()
    op = getattr(torch.ops.pyflash, name)
    assert not any(a.name == "out" for a in op.default._schema.arguments)
    assert all(r.alias_info is None for r in op.default._schema.returns)
    given = next(a for a in op.out._schema.arguments if a.name == "out")
    result = op.out._schema.returns[0]
    assert given.alias_info.is_write and result.alias_info.is_write
    assert given.alias_info.before_set == result.alias_info.before_set
    assert all(r.alias_info is None for r in op.out._schema.returns[1:])
    # every way of calling it comes as far as the device
    a = packed() if name == "forward_packed" else paged()
    for more in ({}, {"out": None}, {"out": torch.zeros_like(a["q"])}):
        for call in (op, getattr(fa, name)):
            with pytest.raises(ValueError, match="no CPU path"):
                call(*a.values(), **more)
    with pytest.raises(ValueError, match="out must have"):
        op(*a.values(), out=torch.zeros(1, 4, 64, dtype=F16))


def test_releasing_scratch_needs_no_device(fa):
    fa.release_workspaces()
    fa.release_workspaces()
