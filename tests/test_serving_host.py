"""CPU only: what the serving operators refuse, through the operators (CPU tensors: everything but the device is looked
at first) and through the C ABI, the workspace query, and the kernels' index arithmetic walked on the host."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def test_index_arithmetic(tmp_path):
    """tests/native/serving_index_test.cpp: lengths, offsets and page tables of any content never lead outside the
    tensors, and decoding workgroups cover every sequence once."""
    exe = str(tmp_path / "serving_index_test")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                           os.path.join(ROOT, "tests", "native", "serving_index_test.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr


def packed(**change):
    a = dict(q=torch.zeros(6, 4, 64, dtype=F16), k=torch.zeros(6, 2, 64, dtype=F16), v=torch.zeros(6, 2, 64, dtype=F16),
             cu_seqlens_q=torch.tensor([0, 2, 6], dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(6, 64, dtype=F16)), "q must be"),
    (dict(q=torch.zeros(6, 4, 64)), "float16 or bfloat16"),
    (dict(k=torch.zeros(6, 2, 64, dtype=BF16)), "one dtype"),
    (dict(v=torch.zeros(5, 2, 64, dtype=F16)), "shape of k"),
    (dict(k=torch.zeros(6, 2, 32, dtype=F16), v=torch.zeros(6, 2, 32, dtype=F16)), "same head dim"),
    (dict(q=torch.zeros(6, 5, 64, dtype=F16)), "multiple of the 2 K/V heads"),
    (dict(q=torch.zeros(6, 4, 128, dtype=F16)[:, :, ::2]), "adjacent"),
    (dict(cu_seqlens_q=torch.tensor([0, 2, 6])), "int32"),
    (dict(cu_seqlens_q=torch.tensor([[0, 6]], dtype=torch.int32)), "1 dimension"),
    (dict(cu_seqlens_q=torch.zeros(0, dtype=torch.int32)), "one entry more"),
    (dict(cu_seqlens_k=torch.tensor([0, 6], dtype=torch.int32)), "one entry more"),
    (dict(k=torch.zeros(7, 2, 64, dtype=F16), v=torch.zeros(7, 2, 64, dtype=F16)), "as many keys as queries"),
    (dict(softmax_scale=0.0), "softmax_scale"),
    (dict(softmax_scale=float("nan")), "softmax_scale"),
    (dict(out=torch.zeros(6, 4, 64, dtype=BF16)), "out must have"),
    (dict(out=torch.zeros(5, 4, 64, dtype=F16)), "out must have"),
    (dict(q=torch.zeros(6, 4, 64, dtype=F16, requires_grad=True)), "no backward"),
    (dict(), "no CPU path"),
])
def test_packed_refusals(fa, change, match):
    with pytest.raises(ValueError, match=match):
        fa.forward_packed(**packed(**change))


@pytest.mark.parametrize("d", [136, 100, 4, 256])
def test_head_dims(fa, d):
    x = torch.zeros(6, 2, d, dtype=F16)
    with pytest.raises(ValueError, match="head dim"):
        fa.forward_packed(x, x, x, torch.tensor([0, 6], dtype=torch.int32))


def paged(**change):
    a = dict(q=torch.zeros(2, 4, 64, dtype=F16), k_cache=torch.zeros(5, 2, 16, 64, dtype=F16), v_cache=torch.zeros(5, 2, 16, 64, dtype=F16),
             page_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32))
    a.update(change)
    return a


def caches(*shape, dtype=F16):
    return dict(k_cache=torch.zeros(*shape, dtype=dtype), v_cache=torch.zeros(*shape, dtype=dtype))


CACHE_REFUSALS = [
    (caches(5, 2, 64), "k_cache must be"),
    (dict(v_cache=torch.zeros(5, 2, 32, 64, dtype=F16)), "shape and type of k_cache"),
    (dict(v_cache=torch.zeros(5, 16, 2, 64, dtype=F16).transpose(1, 2)), "strides of k_cache"),
    (caches(5, 2, 16, 64, dtype=torch.float32), "float8_e4m3fn"),
    (caches(5, 2, 16, 64, dtype=torch.float8_e5m2), "float8_e4m3fn"),
    (dict(page_table=torch.zeros(2, 3)), "int32"),
    (dict(page_table=torch.zeros(3, dtype=torch.int32)), "2 dimension"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), "adjacent"),
    (dict(seq_lens=torch.zeros(2)), "int32"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "one entry for each"),
    (dict(k_scale=torch.ones(2)), "float8_e4m3fn cache only"),
    (dict(k_scale=torch.ones(3), **caches(5, 2, 16, 64, dtype=E4M3)), "2 entries"),
    (dict(v_scale=torch.ones(2, dtype=F16), **caches(5, 2, 16, 64, dtype=E4M3)), "2 entries"),
    (dict(), "no CPU path"),
]


@pytest.mark.parametrize("change,match", CACHE_REFUSALS + [
    (dict(q=torch.zeros(2, 64, dtype=F16)), "q must be"),
    (dict(q=torch.zeros(3, 4, 64, dtype=F16)), "one row for each"),
    (dict(q=torch.zeros(2, 4, 32, dtype=F16)), "same head dim"),
    (dict(q=torch.zeros(2, 3, 64, dtype=F16)), "multiple of the 2 K/V heads"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF16)), "type of the other tensors"),
    (caches(5, 2, 12, 64), "power of two"),
    (caches(0, 2, 16, 64), "pages"),
    (dict(softmax_scale=-1.0), "softmax_scale"),
    (dict(out=torch.zeros(2, 4, 32, dtype=F16)), "out must have"),
    (dict(page_table=torch.zeros(2, 4096, dtype=torch.int32), workspace=torch.zeros(16, dtype=torch.uint8)), "workspace"),
    (dict(q=torch.zeros(2, 4, 64, dtype=F16, requires_grad=True)), "no backward"),
])
def test_decode_refusals(fa, change, match):
    with pytest.raises(ValueError, match=match):
        fa.decode_paged(**paged(**change))


@pytest.mark.parametrize("change,match", CACHE_REFUSALS + [
    (dict(k=torch.zeros(2, 64, dtype=F16)), "k must be"),
    (dict(k=torch.zeros(2, 4, 64, dtype=F16), v=torch.zeros(2, 4, 64, dtype=F16)), "like the cache's rows"),
    (dict(v=torch.zeros(3, 2, 64, dtype=F16)), "shape and type of k"),
    (dict(cu_seqlens=torch.tensor([0, 2], dtype=torch.int32)), "3 entries"),
    (dict(cu_seqlens=torch.tensor([0, 1, 2])), "int32"),
    (dict(k=torch.zeros(2, 2, 64, dtype=F16, requires_grad=True)), "no backward"),
])
def test_append_refusals(fa, change, match):
    a = paged(**change)
    a.pop("q")
    a.setdefault("k", torch.zeros(2, 2, 64, dtype=F16))
    a.setdefault("v", torch.zeros(2, 2, 64, dtype=F16))
    with pytest.raises(ValueError, match=match):
        fa.cache_append(**a)


def test_workspace_query(fa):
    """No scratch where no sequence can be cut; otherwise two parts for each of at most 768 workgroups at the largest head
    dim, and a ticket for each sequence and K/V head."""
    a = paged()
    assert fa.decode_workspace_bytes(a["q"], a["k_cache"], a["page_table"]) == 0
    wide = torch.zeros(2, 4096, dtype=torch.int32)
    need = fa.decode_workspace_bytes(a["q"], a["k_cache"], wide)
    assert need == 2 * 768 * 16 * (128 * 4 + 8) + 16
    assert fa.decode_workspace_bytes(a["q"], a["k_cache"], torch.zeros(2, 1 << 22, dtype=torch.int32)) == need


class Cache(ctypes.Structure):
    _fields_ = ([("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] +
                [(n, ctypes.c_int64) for n in ("num_pages", "kv_heads", "page_size", "d", "page_stride", "head_stride", "slot_stride")] +
                [("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("page_table", ctypes.c_void_p)] +
                [(n, ctypes.c_int64) for n in ("sequences", "table_width", "table_stride")] +
                [("seq_lens", ctypes.c_void_p), ("dtype", ctypes.c_int32)])


class Append(ctypes.Structure):
    _fields_ = ([("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] +
                [(n, ctypes.c_int64) for n in ("tokens", "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")] +
                [("cu_seqlens", ctypes.c_void_p), ("dtype", ctypes.c_int32)])


class Decode(ctypes.Structure):
    _fields_ = ([("q", ctypes.c_void_p), ("o", ctypes.c_void_p), ("lse", ctypes.c_void_p)] +
                [(n, ctypes.c_int64) for n in ("q_heads", "q_batch_stride", "q_head_stride", "o_batch_stride", "o_head_stride")] +
                [("softmax_scale", ctypes.c_float), ("dtype", ctypes.c_int32)])


class Packed(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "cu_q", "cu_k")] +
                [(n, ctypes.c_int64) for n in ("sequences", "total_q", "total_k", "q_heads", "kv_heads", "d", "qt", "qh", "kt", "kh", "vt", "vh", "ot", "oh")] +
                [("softmax_scale", ctypes.c_float), ("causal", ctypes.c_int32), ("dtype", ctypes.c_int32)])


P = 1 << 20   # an aligned address that is never read: every call here is refused, or has nothing to do


def cache(**change):
    a = dict(k=P, v=P, num_pages=5, kv_heads=2, page_size=16, d=64, page_stride=2048, head_stride=1024, slot_stride=64, page_table=P, sequences=2,
             table_width=300, table_stride=300, seq_lens=P, dtype=0)
    a.update(change)
    return Cache(**a)


def refused(fa, rc, match):
    text = fa.lib().flash_hip_last_error().decode()
    return rc in (-1, -2) and match in text


@pytest.mark.parametrize("change,match", [
    (dict(page_size=24), "power of two"), (dict(page_size=0), "power of two"), (dict(num_pages=0), "pages"), (dict(num_pages=1 << 31), "pages"),
    (dict(kv_heads=3), "multiple"), (dict(kv_heads=0), "head counts"), (dict(d=60), "head dim"), (dict(d=136), "head dim"), (dict(k=None), "null"),
    (dict(k=P + 8), "16-byte"), (dict(head_stride=1028), "16-byte"), (dict(slot_stride=60), "16-byte"), (dict(page_stride=2044), "16-byte"),
    (dict(head_stride=-1024), "negative"), (dict(page_stride=-2048), "negative"), (dict(dtype=1), "type"), (dict(dtype=5), "type"),
    (dict(k_scale=P), "e4m3"), (dict(page_table=None), "null page table"), (dict(seq_lens=None), "null page table"),
    (dict(table_width=1 << 28), "positions"), (dict(sequences=-1), "page table"), (dict(dtype=2, k=P + 4), "8-byte"),
])
def test_cache_refusals_through_the_abi(fa, change, match):
    c = cache(**change)
    d = Decode(q=P, o=P, q_heads=4, q_batch_stride=256, q_head_stride=64, o_batch_stride=256, o_head_stride=64, softmax_scale=0.125, dtype=0)
    L = fa.lib()
    assert refused(fa, L.flash_decode_paged(ctypes.byref(d), ctypes.byref(c), P, 1 << 40, None), match)
    if match != "multiple":
        a = Append(k=P, v=P, tokens=2, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, dtype=0)
        assert refused(fa, L.flash_cache_append(ctypes.byref(a), ctypes.byref(c), None), match)


def test_decode_and_append_refusals_through_the_abi(fa):
    L = fa.lib()
    c = cache()
    good = dict(q=P, o=P, q_heads=4, q_batch_stride=256, q_head_stride=64, o_batch_stride=256, o_head_stride=64, softmax_scale=0.125, dtype=0)
    for change, match in ((dict(q=None), "null"), (dict(o=P + 2), "16-byte"), (dict(q_batch_stride=252), "16-byte"), (dict(dtype=2), "float16"),
                          (dict(softmax_scale=float("inf")), "softmax_scale"), (dict(q_heads=70000), "head counts")):
        d = Decode(**{**good, **change})
        assert refused(fa, L.flash_decode_paged(ctypes.byref(d), ctypes.byref(c), P, 1 << 40, None), match), change
    d = Decode(**good)
    assert refused(fa, L.flash_decode_paged(ctypes.byref(d), ctypes.byref(c), None, 0, None), "workspace")
    assert refused(fa, L.flash_decode_paged(ctypes.byref(d), ctypes.byref(c), P + 8, 1 << 40, None), "workspace")
    assert refused(fa, L.flash_decode_paged(None, ctypes.byref(c), P, 1 << 40, None), "null")
    assert refused(fa, L.flash_decode_paged(ctypes.byref(d), None, P, 1 << 40, None), "null")
    assert L.flash_decode_paged_workspace_bytes(ctypes.byref(d), None) == -1
    assert L.flash_decode_paged(ctypes.byref(d), ctypes.byref(cache(sequences=0)), None, 0, None) == 0     # nothing to do
    a = dict(k=P, v=P, tokens=2, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, dtype=0)
    for change, match in ((dict(k=None), "null"), (dict(tokens=3), "one token per sequence"), (dict(tokens=-1), "tokens"), (dict(v=P + 2), "16-byte"),
                          (dict(k_head_stride=60), "16-byte"), (dict(dtype=1), "type")):
        x = Append(**{**a, **change})
        assert refused(fa, L.flash_cache_append(ctypes.byref(x), ctypes.byref(c), None), match), change
    x = Append(**{**a, "tokens": 0, "cu_seqlens": P})
    assert L.flash_cache_append(ctypes.byref(x), ctypes.byref(c), None) == 0


def test_packed_refusals_through_the_abi(fa):
    L = fa.lib()
    good = dict(q=P, k=P, v=P, o=P, cu_q=P, cu_k=P, sequences=2, total_q=6, total_k=6, q_heads=4, kv_heads=2, d=64, qt=256, qh=64, kt=128, kh=64, vt=128,
                vh=64, ot=256, oh=64, softmax_scale=0.125, causal=1, dtype=0)
    for change, match in ((dict(q=None), "null"), (dict(k=None), "null"), (dict(cu_k=None), "cu_seqlens"), (dict(q=P + 4), "16-byte"), (dict(vt=124), "16-byte"),
                          (dict(oh=-64), "negative"), (dict(dtype=2), "float16"), (dict(causal=2), "causal"), (dict(d=52), "head dim"),
                          (dict(q_heads=5), "multiple"), (dict(total_q=-1), "between"), (dict(total_k=1 << 31), "between"), (dict(softmax_scale=0.0), "softmax_scale"),
                          (dict(softmax_scale=3e38), "softmax_scale")):
        p = Packed(**{**good, **change})
        assert refused(fa, L.flash_fwd_packed(ctypes.byref(p), None, 0, None), match), change
    # a workspace, where one is of use: few rows over many keys
    few = Packed(**{**good, "total_k": 4096})
    need = L.flash_fwd_packed_workspace_bytes(ctypes.byref(few))
    assert need > 2048
    assert refused(fa, L.flash_fwd_packed(ctypes.byref(few), P, need - 1, None), "too small")
    assert refused(fa, L.flash_fwd_packed(ctypes.byref(few), P + 8, need, None), "aligned")
    assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**good))) == 0                                     # few keys
    assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**{**good, "total_k": 4096, "total_q": 1 << 20}))) == 0  # many rows
    assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**{**good, "total_q": 0}))) == 0
    assert L.flash_fwd_packed_workspace_bytes(ctypes.byref(Packed(**{**good, "d": 52}))) == -1
    assert L.flash_fwd_packed_workspace_bytes(None) == -1
    assert refused(fa, L.flash_fwd_packed(None, None, 0, None), "null")
    assert L.flash_fwd_packed(ctypes.byref(Packed(**{**good, "sequences": 0, "q": None})), None, 0, None) == 0
    assert L.flash_fwd_packed(ctypes.byref(Packed(**{**good, "total_q": 0, "q": None})), None, 0, None) == 0
