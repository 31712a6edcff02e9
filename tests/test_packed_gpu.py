"""GPU: attention over packed prompts (fa.forward_packed) against a plain float64 form, head by head.  The bounds are
derived from the kernels' arithmetic in serving_reference.bound."""
import math

import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(q_lens, k_lens, hq, hk, d, dtype, seed=0, fused=False):
    gen = torch.Generator().manual_seed(seed)
    tq, tk = sum(q_lens), sum(k_lens)
    if fused:
        x = torch.randn(tq, hq + 2 * hk, d, generator=gen).to(dtype)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], x
    q = torch.randn(tq, hq, d, generator=gen).to(dtype)
    k, v = (torch.randn(tk, hk, d, generator=gen).to(dtype) for _ in range(2))
    return q, k, v, None


def call(fa, q, k, v, q_lens, k_lens=None, **more):
    cu_k = None if k_lens is None else ref.offsets(k_lens).cuda()
    return fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), ref.offsets(q_lens).cuda(), cu_k, **more)


CASES = [
    # q_lens, k_lens (None: the same), Hq, Hkv, d, dtype
    ([1], None, 1, 1, 64, F16),
    ([2, 1, 3], None, 2, 1, 128, BF16),
    ([17], None, 4, 2, 64, BF16),
    ([63, 64, 65, 1, 0, 31, 32, 33], None, 3, 1, 128, F16),
    ([255, 256, 257], None, 2, 2, 128, BF16),
    ([255, 256, 257, 511], None, 2, 1, 64, F16),
    ([700, 13, 1100], None, 4, 2, 128, F16),
    ([300, 5], None, 6, 2, 40, BF16),
    ([129, 140], None, 5, 5, 72, F16),
    ([90], None, 2, 1, 8, BF16),
    ([200, 333], None, 7, 1, 112, BF16),
    # keys that reach back before the first query: later pieces of prompts
    ([5, 64, 300], [700, 129, 301], 4, 2, 128, BF16),
    ([1, 1, 1, 1], [1, 64, 65, 999], 4, 1, 64, F16),
    ([77], [1357], 2, 2, 96, F16),
    # more queries than keys: the first ones see nothing; sequences without keys, without queries
    ([10, 300, 70, 0, 33], [4, 40, 0, 50, 33], 2, 1, 128, F16),
    ([130], [1], 2, 2, 64, BF16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{'-'.join(map(str, c[0]))}_k{c[1] and '-'.join(map(str, c[1]))}_{c[2]}x{c[3]}_d{c[4]}_{str(c[5])[6:]}")
def test_against_float64(fa, case, causal):
    q_lens, k_lens, hq, hk, d, dtype = case
    q, k, v, _ = make(q_lens, k_lens or q_lens, hq, hk, d, dtype, seed=sum(q_lens))
    got = call(fa, q, k, v, q_lens, k_lens, causal=causal)
    assert got.dtype == dtype and got.shape == q.shape and got.is_contiguous()
    ref.check_packed(got, q, k, v, q_lens, k_lens or q_lens, causal, d ** -0.5)


def test_many_short_sequences(fa):
    lens = [n % 5 for n in range(200)] + [40]
    q, k, v, _ = make(lens, lens, 2, 1, 64, BF16, seed=3)
    ref.check_packed(call(fa, q, k, v, lens), q, k, v, lens, lens, True, 64 ** -0.5)


@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 128, BF16), (4, 4, 64, F16)])
def test_long_prompt(fa, hq, hk, d, dtype):
    lens = [4099, 700]
    q, k, v, _ = make(lens, lens, hq, hk, d, dtype, seed=9)
    ref.check_packed(call(fa, q, k, v, lens), q, k, v, lens, lens, True, d ** -0.5, heads=[0, hq - 1])


def test_slices_of_a_fused_projection_and_strided_output(fa):
    lens, hq, hk, d = [150, 260], 4, 2, 128
    q, k, v, whole = make(lens, lens, hq, hk, d, F16, seed=4, fused=True)
    x = whole.cuda()
    room = torch.full((sum(lens), hq + 1, d), 7.0, dtype=F16, device="cuda")
    out = room[:, :hq]
    got = fa.forward_packed(x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], ref.offsets(lens).cuda(), out=out)
    assert got.data_ptr() == room.data_ptr() and bool((room[:, hq] == 7.0).all())
    ref.check_packed(out, q, k, v, lens, lens, True, d ** -0.5)
    # head-major tensors, as the other operators of this package take them
    t = [a.transpose(0, 1).contiguous().cuda().transpose(0, 1) for a in (q, k, v)]
    assert torch.equal(fa.forward_packed(*t, ref.offsets(lens).cuda()), out)


def test_rows_behind_the_last_sequence_are_left_as_they_were(fa):
    lens, pad = [100, 33], 91
    q, k, v, _ = make([sum(lens) + pad], [sum(lens) + pad], 2, 1, 128, BF16, seed=5)
    k[sum(lens):] = float("nan")
    v[sum(lens):] = float("inf")
    out = torch.full_like(q, 3.0).cuda()
    call(fa, q, k, v, lens, out=out)
    assert bool((out[sum(lens):] == 3.0).all())
    ref.check_packed(out[:sum(lens)], q[:sum(lens)], k[:sum(lens)], v[:sum(lens)], lens, lens, True, 128 ** -0.5)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, F16), (72, BF16)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_masked_places_may_hold_anything(fa, d, dtype, poison):
    """Keys and values that a query does not see do not reach it, whatever they hold, although they share a tile with
    some it sees; those that see a non-finite value get what the formula gives."""
    lens = [333, 290]
    q, k, v, _ = make(lens, lens, 2, 1, d, dtype, seed=6)
    bad = torch.finfo(dtype).min if poison == "lowest" else poison
    for row in (40, 201, 330, 333 + 250):
        v[row, 0, 3::7] = bad
    got = call(fa, q, k, v, lens)
    ref.check_packed(got, q, k, v, lens, lens, True, d ** -0.5)
    k[332] = bad                  # the last key of the first sequence: only the last query sees it
    got2 = call(fa, q, k, v, lens)
    assert torch.equal(got2[:332].view(torch.int16), got[:332].view(torch.int16))
    assert torch.equal(got2[333:].view(torch.int16), got[333:].view(torch.int16))


def test_scores_far_apart(fa):
    """Rows whose largest score stands far above the first ones seen, and far below."""
    lens, d = [600], 128
    q, k, v, _ = make(lens, lens, 2, 2, d, F16, seed=7)
    k *= 0.2
    for j, gain in ((70, 4.0), (200, 12.0), (401, 25.0), (599, 40.0)):
        k[j] = q[j] * (gain / 11.0)
    ref.check_packed(call(fa, q, k, v, lens), q, k, v, lens, lens, True, d ** -0.5)
    ref.check_packed(call(fa, q, -k, v, lens), q, -k, v, lens, lens, True, d ** -0.5)


def test_scale_argument(fa):
    lens = [50]
    q, k, v, _ = make(lens, lens, 1, 1, 64, BF16, seed=8)
    for scale in (0.03, 0.5):
        ref.check_packed(call(fa, q, k, v, lens, softmax_scale=scale), q, k, v, lens, lens, True, scale)


def test_offsets_beyond_the_tensors_stay_inside(fa):
    """Offsets are cut to the tensors: a sequence that runs past the end ends there, one that runs backwards is empty."""
    q, k, v, _ = make([64], [64], 1, 1, 64, F16, seed=10)
    out = torch.full_like(q, 5.0).cuda()
    cu = torch.tensor([0, 20, 10, 500], dtype=torch.int32).cuda()
    fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), cu, out=out)
    # sequences: rows 0..20, nothing, rows 10..64 (which overwrite the first one's rows 10..20)
    ref.check_packed(out[:10], q[:10], k[:10], v[:10], [10], [10], True, 0.125)
    whole = ref.attention(q[10:, 0], k[10:, 0], v[10:, 0], ref.visible_keys(54, 54, True), 0.125)
    ref.assert_within(out[20:, 0], whole[0][10:], ref.bound(whole[0], whole[2], whole[3], 54, 64, F16, True)[10:], "cut sequence")


def test_empty_calls(fa):
    q = torch.empty(0, 4, 64, dtype=F16, device="cuda")
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert fa.forward_packed(q, q[:, :2], q[:, :2], cu).shape == (0, 4, 64)
    q = torch.randn(5, 4, 64, device="cuda").half()
    none = q[:0, :2]
    out = fa.forward_packed(q, none, none, torch.tensor([0, 5], dtype=torch.int32, device="cuda"),
                            torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    assert bool((out == 0).all())


def test_captured_and_replayed_with_other_lengths(fa):
    """The lengths are read on the device: one graph serves every split of the same rows."""
    total, hq, hk, d = 640, 4, 2, 128
    q, k, v, _ = make([total], [total], hq, hk, d, BF16, seed=11)
    qd, kd, vd, cu = q.cuda(), k.cuda(), v.cuda(), ref.offsets([300, 340]).cuda()
    out = torch.empty_like(qd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fa.forward_packed(qd, kd, vd, cu, out=out, sync=False)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            fa.forward_packed(qd, kd, vd, cu, out=out, sync=False)
    for lens in ([300, 340], [640, 0], [1, 639], [320, 320]):
        cu.copy_(ref.offsets(lens))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fa.forward_packed(qd, kd, vd, cu)), lens
    ref.check_packed(out, q, k, v, [320, 320], [320, 320], True, d ** -0.5, heads=[1])


def test_runs_on_the_current_stream(fa):
    lens = [512]
    q, k, v, _ = make(lens, lens, 4, 4, 128, F16, seed=12)
    want = call(fa, q, k, v, lens)
    side = torch.cuda.Stream()
    src = [x.cuda() for x in (q, k, v)]
    cu = ref.offsets(lens).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        moved = [torch.empty_like(x) for x in src]
        for a, b in zip(moved, src):
            a.copy_(b)              # behind this on the same stream, in front of it on any other
        got = fa.forward_packed(*moved, cu, sync=False)
    side.synchronize()
    assert torch.equal(got, want)


def test_same_bits_every_time(fa):
    lens = [1000, 300]
    q, k, v, _ = make(lens, lens, 4, 2, 128, BF16, seed=13)
    first = call(fa, q, k, v, lens)
    for _ in range(3):
        assert torch.equal(call(fa, q, k, v, lens), first)


def test_one_piece_or_several(fa):
    """A prompt worked off in pieces, each over all keys so far, gives the rows of the whole."""
    n, hq, hk, d = 700, 4, 2, 64
    q, k, v, _ = make([n], [n], hq, hk, d, F16, seed=14)
    for a, b in ((0, 256), (256, 257), (257, 700)):
        part = call(fa, q[a:b], k[:b], v[:b], [b - a], [b])
        ref.check_packed(part, q[a:b], k[:b], v[:b], [b - a], [b], True, d ** -0.5, heads=[0, 3])


def test_needs_no_gradient(fa):
    q = torch.randn(4, 2, 64, device="cuda").half().requires_grad_()
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="no backward"):
        fa.forward_packed(q, q, q, cu)
    with torch.no_grad():
        out = fa.forward_packed(q, q, q, cu)
    assert not out.requires_grad and math.isfinite(float(out.float().sum()))


# few rows over many keys: the keys of a row are dealt to several workgroups
CUT_CASES = [
    ([130], [4200], 2, 1, 128, BF16),
    ([300, 40], [2600, 1500], 4, 2, 64, F16),
    ([5, 64, 300], [700, 129, 3001], 6, 2, 128, F16),
    ([1], [9000], 2, 1, 72, BF16),
    ([1, 0, 1, 200], [1024, 77, 0, 2047], 4, 1, 96, F16),
    ([2500], [2500], 2, 1, 64, BF16),
    ([1500], [1100], 2, 2, 128, BF16),
    ([1900], [1700], 2, 2, 128, BF16),
    ([333], [3333], 5, 1, 40, F16),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CUT_CASES, ids=lambda c: f"q{'-'.join(map(str, c[0]))}_k{'-'.join(map(str, c[1]))}_{c[2]}x{c[3]}_d{c[4]}_{str(c[5])[6:]}")
def test_few_rows_over_many_keys(fa, case, causal):
    q_lens, k_lens, hq, hk, d, dtype = case
    q, k, v, _ = make(q_lens, k_lens, hq, hk, d, dtype, seed=sum(k_lens))
    got = call(fa, q, k, v, q_lens, k_lens, causal=causal)
    ref.check_packed(got, q, k, v, q_lens, k_lens, causal, d ** -0.5, heads=[0, hq - 1])
    for _ in range(3):
        assert torch.equal(call(fa, q, k, v, q_lens, k_lens, causal=causal), got)


def _packed_args(q, k, v, out, cu_q, cu_k, causal=True):
    import ctypes

    class Packed(ctypes.Structure):
        _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "cu_q", "cu_k")] +
                    [(n, ctypes.c_int64) for n in ("sequences", "total_q", "total_k", "q_heads", "kv_heads", "d", "qt", "qh", "kt", "kh", "vt", "vh", "ot", "oh")] +
                    [("softmax_scale", ctypes.c_float), ("causal", ctypes.c_int32), ("dtype", ctypes.c_int32)])
    strides = [s for x in (q, k, v, out) for s in x.stride()[:2]]
    return Packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), len(cu_q) - 1, q.shape[0], k.shape[0],
                  q.shape[1], k.shape[1], q.shape[2], *strides, q.shape[2] ** -0.5, int(causal), {F16: 0, BF16: 1}[q.dtype])


def test_cut_with_a_workspace_and_whole_without(fa):
    """Through the C entry: one workspace, whose parts hold NaN in front of each call, for calls of several shapes; and none."""
    import ctypes
    L = fa.lib()
    work = torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    for q_lens, k_lens, hq, hk, d, dtype in CUT_CASES[:4]:
        q, k, v, _ = make(q_lens, k_lens, hq, hk, d, dtype, seed=3)
        dev = [x.cuda() for x in (q, k, v)] + [torch.full_like(q, 5.0).cuda(), ref.offsets(q_lens).cuda(), ref.offsets(k_lens).cuda()]
        a = _packed_args(*dev)
        need = L.flash_fwd_packed_workspace_bytes(ctypes.byref(a))
        assert need > 2048
        assert need <= work.numel()
        work[2048:] = 255               # (an earlier call may have needed more)
        stream = torch.cuda.current_stream().cuda_stream
        assert L.flash_fwd_packed(ctypes.byref(a), work.data_ptr(), need, stream) == 0, L.flash_hip_last_error()
        torch.cuda.synchronize()
        assert not bool(work[:2048].any())
        assert bool((work[need:] == 255).all())
        ref.check_packed(dev[3], q, k, v, q_lens, k_lens, True, d ** -0.5, heads=[0])
        dev[3].fill_(5.0)
        assert L.flash_fwd_packed(ctypes.byref(a), None, 0, stream) == 0, L.flash_hip_last_error()
        ref.check_packed(dev[3], q, k, v, q_lens, k_lens, True, d ** -0.5, heads=[0])


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_cut_rows_and_masked_places(fa, poison):
    """As test_masked_places_may_hold_anything, with the diagonal in the last of several parts, and values in the first
    part that every row sees."""
    nq, nk, d = 150, 2300, 128
    q, k, v, _ = make([nq], [nk], 2, 1, d, BF16, seed=21)
    bad = torch.finfo(BF16).min if poison == "lowest" else poison
    for row in (nk - 149, nk - 70, nk - 3):
        v[row, 0, 3::7] = bad
    got = call(fa, q, k, v, [nq], [nk])
    ref.check_packed(got, q, k, v, [nq], [nk], True, d ** -0.5)
    k[nk - 1] = bad
    got2 = call(fa, q, k, v, [nq], [nk])
    assert torch.equal(got2[:nq - 1].view(torch.int16), got[:nq - 1].view(torch.int16))
    v[100, 0, 5] = bad
    k[nk - 1] = 0.0
    got = call(fa, q, k, v, [nq], [nk])
    ref.check_packed(got, q, k, v, [nq], [nk], True, d ** -0.5)


def test_cut_rows_in_a_graph_beside_eager_calls(fa):
    """A captured call has scratch of its own: replays on one stream beside eager calls, and another graph, on others."""
    hq, hk, d, total_q, total_k = 4, 2, 64, 260, 4000
    q, k, v, _ = make([total_q], [total_k], hq, hk, d, F16, seed=22)
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    cu_q, cu_k = ref.offsets([130, 130]).cuda(), ref.offsets([2000, 2000]).cuda()
    outs = [torch.empty_like(qd) for _ in range(3)]
    sides = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    torch.cuda.synchronize()
    for out, side in zip(outs[:2], sides):
        with torch.cuda.stream(side):
            fa.forward_packed(qd, kd, vd, cu_q, cu_k, out=out, sync=False)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                fa.forward_packed(qd, kd, vd, cu_q, cu_k, out=out, sync=False)
        graphs.append(graph)
    for q_lens, k_lens in (([130, 130], [2000, 2000]), ([260, 0], [3000, 1000]), ([3, 257], [10, 3990])):
        cu_q.copy_(ref.offsets(q_lens))
        cu_k.copy_(ref.offsets(k_lens))
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, side in zip(graphs, sides):
                with torch.cuda.stream(side):
                    graph.replay()
            with torch.cuda.stream(sides[2]):
                fa.forward_packed(qd, kd, vd, cu_q, cu_k, out=outs[2], sync=False)
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, outs[0])
        ref.check_packed(outs[0], q, k, v, q_lens, k_lens, True, d ** -0.5, heads=[0, 3])


@pytest.mark.parametrize("d,dtype,causal", [(128, BF16, True), (64, F16, False), (40, BF16, True)])
def test_rows_far_apart(fa, d, dtype, causal):
    """Rows more than 4 MiB apart (one row of a wide array per token)."""
    q_lens, k_lens = [5, 70], [40, 130]
    q, k, v, _ = make(q_lens, k_lens, 2, 1, d, dtype, seed=23)
    wide = torch.zeros(sum(k_lens), (1 << 21) + 64, dtype=dtype, device="cuda")
    kd = wide[:, :d].unflatten(1, (1, d))
    kd.copy_(k)
    got = fa.forward_packed(q.cuda(), kd, v.cuda(), ref.offsets(q_lens).cuda(), ref.offsets(k_lens).cuda(), causal=causal)
    ref.check_packed(got, q, k, v, q_lens, k_lens, causal, d ** -0.5)


@pytest.mark.parametrize("sequences,same,causal,d", [(65, True, True, 128), (64, False, True, 64), (300, False, True, 128), (300, False, False, 64), (4500, True, True, 64)])
def test_more_sequences_than_a_scan_covers(fa, sequences, same, causal, d):
    gen = torch.Generator().manual_seed(sequences)
    q_lens = torch.randint(0, 9, (sequences,), generator=gen).tolist()
    q_lens[::29] = [200 + b % 70 for b in range(len(q_lens[::29]))]
    k_lens = q_lens if same else [n + int(x) for n, x in zip(q_lens, torch.randint(-3, 90, (sequences,), generator=gen))]
    k_lens = [max(0, n) for n in k_lens]
    q, k, v, _ = make(q_lens, k_lens, 2, 1, d, BF16, seed=25)
    got = call(fa, q, k, v, q_lens, None if same else k_lens, causal=causal)
    ref.check_packed(got, q, k, v, q_lens, k_lens, causal, d ** -0.5, heads=[1])
