"""GPU: the paged key-value cache: fa.cache_append bit for bit, fa.decode_paged against a plain float64 form with the
bounds of serving_reference, and both with fa.forward_packed in one run as a server makes it."""
import pytest
import torch

import serving_reference as ref

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def bits(x):
    return x.view({1: torch.uint8, 2: torch.int16}[x.element_size()])


def filled(lens, page, hk, d, cache_dtype, seed=0, token_major=False, width=None):
    """A pool with random rows in every sequence's positions (16-bit, or what an e4m3 code stands for), NaN elsewhere."""
    gen = torch.Generator().manual_seed(seed)
    kc, vc, table = ref.page_pool(lens, page, hk, d, cache_dtype, token_major=token_major, seed=seed, width=width)
    rows = [[torch.randn(n, hk, d, generator=gen).mul(20 if cache_dtype == E4M3 else 1).to(cache_dtype) for n in lens] for _ in range(2)]
    ref.fill(kc, table, rows[0], page)
    ref.fill(vc, table, rows[1], page)
    return kc, vc, table, rows


def on_gpu(x):
    """To the device with the strides kept."""
    return x.transpose(1, 2).contiguous().cuda().transpose(1, 2) if not x.is_contiguous() else x.cuda()


def check_decode(got, lse, q, rows, lens, scale, ks=None, vs=None, heads=None, what=""):
    hq, d = q.shape[1:]
    hk = rows[0][0].shape[1]
    for b, n in enumerate(lens):
        for h in range(hq) if heads is None else heads:
            g = h // (hq // hk)
            k = rows[0][b][:, g].double() * (1.0 if ks is None else float(ks[g]))
            v = rows[1][b][:, g].double() * (1.0 if vs is None else float(vs[g]))
            out, want_lse, spread, rise = ref.attention(q[b:b + 1, h], k, v, torch.ones(1, n, dtype=torch.bool), scale)
            ref.assert_within(got[b:b + 1, h], out, ref.bound(out, spread, rise, n, d, q.dtype, False), f"{what} sequence {b} (length {n}), head {h}")
            if lse is not None:
                ref.assert_within(lse[b, h].reshape(1), want_lse, ref.lse_bound(want_lse, rise, n, d), f"{what} lse, sequence {b} (length {n}), head {h}")


CASES = [
    # lens, page, Hq, Hkv, d, dtype, cache, token-major
    ([1], 16, 1, 1, 64, F16, F16, False),
    ([1, 0, 2], 16, 2, 1, 128, BF16, BF16, False),
    ([15, 16, 17, 31, 32, 33], 16, 4, 2, 128, F16, F16, False),
    ([127, 128, 129, 255, 256, 257], 32, 4, 1, 64, BF16, BF16, True),
    ([127, 128, 129, 600], 64, 8, 2, 128, BF16, BF16, False),
    ([1023], 16, 32, 8, 128, BF16, BF16, False),
    ([0, 0], 16, 4, 4, 128, F16, F16, False),
    ([2500, 3, 700], 128, 3, 3, 128, F16, F16, True),
    ([300, 41], 1, 2, 1, 64, F16, F16, False),          # pages of one token
    ([300, 41], 2, 5, 1, 128, BF16, BF16, True),
    ([99, 1000], 8, 7, 1, 72, BF16, BF16, False),
    ([513, 77], 256, 6, 2, 40, F16, F16, False),
    ([200], 16, 4, 2, 8, BF16, BF16, False),
    ([700, 90], 16, 17, 1, 128, F16, F16, False),       # more than 16 query heads on a K/V head
    ([700, 90], 16, 96, 1, 112, BF16, BF16, False),
    ([350, 5], 16, 40, 2, 64, F16, F16, True),
    ([1, 255, 256, 257, 1111], 16, 8, 2, 128, BF16, E4M3, False),
    ([300, 0, 65], 32, 4, 4, 64, F16, E4M3, True),
    ([300, 65], 64, 6, 1, 72, BF16, E4M3, False),
    ([555], 4, 20, 1, 120, F16, E4M3, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"n{'-'.join(map(str, c[0]))}_p{c[1]}_{c[2]}x{c[3]}_d{c[4]}_{str(c[5])[6:]}_{str(c[6])[6:]}")
def test_decode_against_float64(fa, case):
    lens, page, hq, hk, d, dtype, cache_dtype, token_major = case
    kc, vc, table, rows = filled(lens, page, hk, d, cache_dtype, seed=sum(lens), token_major=token_major)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    scales = [torch.rand(hk, generator=torch.Generator().manual_seed(s)) * 0.03 + 0.02 for s in (2, 3)] if cache_dtype == E4M3 else [None, None]
    dev = [None if s is None else s.cuda() for s in scales]
    got, lse = fa.decode_paged(q.cuda(), on_gpu(kc), on_gpu(vc), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                               k_scale=dev[0], v_scale=dev[1], return_lse=True)
    assert got.dtype == dtype and got.is_contiguous() and lse.dtype == torch.float32
    check_decode(got, lse, q, rows, lens, d ** -0.5, *scales)
    if cache_dtype == E4M3:      # scales default to 1
        got = fa.decode_paged(q.cuda(), on_gpu(kc), on_gpu(vc), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softmax_scale=0.002)
        check_decode(got, None, q, rows, lens, 0.002)


def test_decode_long_and_ragged(fa):
    """Sequences cut over many workgroups beside sequences that share one."""
    lens = [30001, 5, 0, 129, 4096, 1, 777] + [60] * 70
    kc, vc, table, rows = filled(lens, 16, 2, 128, BF16, seed=21)
    q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(1)).to(BF16)
    got, lse = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check_decode(got, lse, q, rows, lens, 128 ** -0.5, heads=[0, 3, 4, 7])


@pytest.mark.parametrize("sequences", [64, 65, 700, 4500])
def test_decode_many_sequences(fa, sequences):
    """More sequences than a wave has lanes, some of them long and some empty."""
    gen = torch.Generator().manual_seed(sequences)
    lens = torch.randint(0, 20, (sequences,), generator=gen).tolist()
    lens[sequences // 2] = 900
    lens[-1] = 300
    kc, vc, table, rows = filled(lens, 16, 2, 64, F16, seed=33)
    q = torch.randn(sequences, 4, 64, generator=gen).half()
    got, lse = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check_decode(got, lse, q, rows, lens, 0.125, heads=[3])


def test_lengths_decide_and_not_the_table(fa):
    """Positions behind a sequence's length hold NaN, in its last page and in pages that the table names already."""
    lens, page = [37, 130], 16
    kc, vc, table, rows = filled([400, 400], page, 2, 64, F16, seed=22)
    for b, n in enumerate(lens):
        ref.fill(kc, table[b:b + 1], [torch.cat([rows[0][b][:n], torch.full((400 - n, 2, 64), float("nan"), dtype=F16)])], page)
        ref.fill(vc, table[b:b + 1], [torch.cat([rows[1][b][:n], torch.full((400 - n, 2, 64), float("inf"), dtype=F16)])], page)
    cut = [[r[:n] for r, n in zip(rows[s], lens)] for s in range(2)]
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(1)).half()
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    check_decode(got, None, q, cut, lens, 0.125)


def test_pages_outside_the_cache_hold_no_keys(fa):
    lens, page, d = [100, 64], 16, 64
    kc, vc, table, rows = filled(lens, page, 1, d, F16, seed=23)
    bad = table.clone()
    bad[0, 1], bad[0, 3], bad[1, 2] = kc.shape[0], -7, 2 ** 31 - 1
    keep = [[j for j in range(n) if 0 <= int(bad[b, j // page]) < kc.shape[0]] for b, n in enumerate(lens)]
    cut = [[r[i] for r, i in zip(rows[s], keep)] for s in range(2)]
    q = torch.randn(2, 4, d, generator=torch.Generator().manual_seed(1)).half()
    got, lse = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), bad.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), return_lse=True)
    check_decode(got, lse, q, cut, [len(i) for i in keep], 0.125)
    # lengths beyond the table's reach and negative ones are cut to it
    kc, vc, table, rows = filled([64, 64], page, 1, d, F16, seed=24)
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32).cuda())
    check_decode(got, None, q, [[r[0], r[1][:0]] for r in rows], [64, 0], 0.125)


def test_values_at_the_ends_of_the_range(fa):
    """Live infinities and NaN give what the formula gives; scores of the type's lowest value are no special case."""
    d, lens = 64, [50, 50, 50]
    kc, vc, table, rows = filled(lens, 16, 1, d, BF16, seed=25)
    rows[1][0][7, 0, 5] = float("inf")
    rows[1][1][9, 0, 3] = float("nan")
    rows[0][2][11, 0] = torch.finfo(BF16).min / 1e3
    q = torch.randn(3, 2, d, generator=torch.Generator().manual_seed(1)).to(BF16).abs()
    ref.fill(kc, table, rows[0], 16)
    ref.fill(vc, table, rows[1], 16)
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    check_decode(got, None, q, rows, lens, 0.125, heads=[0, 1])


def test_offsets_past_32_bits(fa):
    """A cache of more than 4 GiB, with pages near both of its ends."""
    page, hk, d, pages = 64, 8, 128, 36000
    kc = torch.zeros((pages, hk, page, d), dtype=F16, device="cuda")      # 4.7 GB
    vc = torch.zeros_like(kc)
    gen = torch.Generator().manual_seed(1)
    lens = [150, 100]
    table = torch.tensor([[pages - 1, 0, 33333], [20000, pages - 2, -1]], dtype=torch.int32)
    new = torch.randn(2, sum(lens), hk, d, generator=gen).half()
    cu, n = ref.offsets(lens).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    fa.cache_append(new[0].cuda(), new[1].cuda(), kc, vc, table.cuda(), n, cu)
    assert torch.equal(kc[pages - 1, :, :64].cpu(), new[0][:64].transpose(0, 1))
    assert torch.equal(vc[33333, :, :22].cpu(), new[1][128:150].transpose(0, 1)) and not bool(vc[33333, :, 22:].any())
    q = torch.randn(2, 16, d, generator=gen).half()
    got = fa.decode_paged(q.cuda(), kc, vc, table.cuda(), n)
    rows = [[new[s][:150], new[s][150:]] for s in range(2)]
    check_decode(got, None, q, rows, lens, d ** -0.5, heads=[0, 15])


def test_decode_output_workspace_and_strides(fa):
    lens, d = [300, 1000], 128
    kc, vc, table, rows = filled(lens, 16, 2, d, BF16, seed=26)
    both = torch.randn(2, 10, d, generator=torch.Generator().manual_seed(1)).to(BF16)
    q = both[:, 1:9]
    wide = torch.full((2, 1 + 80), -1, dtype=torch.int32)      # a table that is a slice of a wider one
    wide[:, 1:1 + table.shape[1]] = table
    tab = wide.cuda()[:, 1:1 + table.shape[1]]
    qd, n = both.cuda()[:, 1:9], torch.tensor(lens, dtype=torch.int32).cuda()
    caches = kc.cuda(), vc.cuda()
    want = fa.decode_paged(qd, *caches, tab, n)
    check_decode(want, None, q, rows, lens, d ** -0.5)
    need = fa.decode_workspace_bytes(qd, caches[0], tab)
    ws = fa.decode_workspace(qd, caches[0], tab)
    assert ws.numel() == need > 0
    for _ in range(3):                                        # one workspace for any number of calls
        room = torch.full((2, 9, d), 3.0, dtype=BF16, device="cuda")
        got = fa.decode_paged(qd, *caches, tab, n, out=room[:, :8], workspace=ws)
        assert torch.equal(got, want) and bool((room[:, 8] == 3.0).all())
    with pytest.raises(ValueError, match="workspace"):
        fa.decode_paged(qd, *caches, tab, n, workspace=ws[:need // 2])


def test_one_workspace_for_calls_of_different_shapes(fa):
    """Shapes, head dims and cut lengths by turns on one workspace and on the stream's own."""
    ws = None
    calls = []
    for lens, page, hq, hk, d, dtype in (([5000], 16, 8, 2, 128, F16), ([300] * 40, 32, 4, 4, 64, BF16), ([900, 2, 4000], 64, 16, 1, 96, F16),
                                         ([1300] * 9, 16, 20, 2, 128, BF16)):
        kc, vc, table, rows = filled(lens, page, hk, d, dtype, seed=sum(lens))
        q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(1)).to(dtype)
        args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
        mine = fa.decode_workspace(args[0], args[1], args[3])
        if ws is None or mine.numel() > ws.numel():
            ws = mine
        calls.append((args, q, rows, lens, d))
    for _ in range(2):
        for args, q, rows, lens, d in calls + calls[::-1]:
            got = fa.decode_paged(*args, workspace=ws)
            assert torch.equal(got, fa.decode_paged(*args))
    for args, q, rows, lens, d in calls:
        check_decode(fa.decode_paged(*args), None, q, rows, lens, d ** -0.5, heads=[0, q.shape[1] - 1])


def test_streams_decode_side_by_side(fa):
    """The same call on several streams at once: scratch is kept for each of them."""
    lens = [3000, 1200, 40]
    kc, vc, table, _ = filled(lens, 16, 2, 128, F16, seed=33)
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    args = (q, kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    want = fa.decode_paged(*args)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(fa.decode_paged(*args, sync=False))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_parts_join_through_lse(fa):
    """Two halves of a context decoded apart and joined by their lse give the whole."""
    d, n = 128, 1500
    kc, vc, table, rows = filled([n], 32, 2, d, F16, seed=27)
    q = torch.randn(1, 4, d, generator=torch.Generator().manual_seed(1)).half()
    caches = kc.cuda(), vc.cuda()
    cut = 640
    a, la = fa.decode_paged(q.cuda(), *caches, table[:, :cut // 32].contiguous().cuda(), torch.tensor([cut], dtype=torch.int32).cuda(), return_lse=True)
    b, lb = fa.decode_paged(q.cuda(), *caches, table[:, cut // 32:].contiguous().cuda(), torch.tensor([n - cut], dtype=torch.int32).cuda(), return_lse=True)
    lse = torch.logaddexp(la, lb)
    got = a.float() * (la - lse).exp()[..., None] + b.float() * (lb - lse).exp()[..., None]
    for h in range(4):
        out, want, spread, rise = ref.attention(q[:, h], rows[0][0][:, h // 2], rows[1][0][:, h // 2], torch.ones(1, n, dtype=torch.bool), d ** -0.5)
        # both halves are rounded to fp16; the join itself is exact next to that
        limit = 2 * ref.bound(out, spread, rise, n, d, F16, False) + 2.0 ** -11 * spread
        ref.assert_within(got[:, h], out, limit, f"joined head {h}")
        ref.assert_within(lse[:, h], want, 2 * ref.lse_bound(want, rise, n, d), f"joined lse {h}")


def test_two_graphs_and_an_eager_call_share_nothing(fa):
    """Two captured decoding steps, each with scratch from its own pool, replayed by turns and at the same time with
    growing lengths and an eager call between them."""
    lens, page, d = [900, 300, 2000], 16, 128
    kc, vc, table, _ = filled([1024, 512, 2048], page, 2, d, BF16, seed=28)
    caches = kc.cuda(), vc.cuda()
    tab = table.cuda()
    gen = torch.Generator().manual_seed(5)
    calls = []
    for _ in range(2):
        q = torch.randn(3, 8, d, generator=gen).to(BF16).cuda()
        n = torch.tensor(lens, dtype=torch.int32).cuda()
        out = torch.empty_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fa.decode_paged(q, *caches, tab, n, out=out, sync=False)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                fa.decode_paged(q, *caches, tab, n, out=out, sync=False)
        calls.append((q, n, out, graph, side))
    for step in range(4):
        for q, n, out, graph, side in calls:
            n.add_(step * 7).clamp_(max=512)
            out.zero_()
        torch.cuda.synchronize()
        for q, n, out, graph, side in calls:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for q, n, out, graph, side in calls:
            assert torch.equal(out, fa.decode_paged(q, *caches, tab, n)), step


def test_decode_same_bits_every_time(fa):
    lens = [5000, 64, 333]
    kc, vc, table, _ = filled(lens, 16, 2, 128, F16, seed=29)
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    args = (q, kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    first = fa.decode_paged(*args)
    for _ in range(5):
        assert torch.equal(fa.decode_paged(*args), first)


# ---- writes into the cache ------------------------------------------------------------------------------------------
APPEND = [
    # new, before, page, Hkv, d, dtype, cache, token-major
    ([1], [0], 16, 1, 64, F16, F16, False),
    ([5, 0, 17, 1, 64], [0, 9, 15, 33, 0], 16, 2, 128, BF16, BF16, False),
    ([300, 77], [3, 0], 64, 8, 128, F16, F16, True),
    ([40, 2], [7, 250], 1, 3, 72, BF16, BF16, False),
    ([33], [100], 256, 2, 8, F16, F16, False),
    ([1, 1, 1], [0, 15, 16], 16, 4, 64, BF16, E4M3, False),
    ([70, 0, 129], [3, 4, 0], 32, 2, 128, F16, E4M3, True),
    ([9], [2], 4, 5, 40, BF16, E4M3, False),
    ([n % 3 for n in range(150)], [n % 20 for n in range(150)], 8, 1, 64, F16, F16, False),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{len(c[0])}seq_{sum(c[0])}tok_p{c[2]}_{c[3]}h_d{c[4]}_{str(c[5])[6:]}_{str(c[6])[6:]}")
def test_append_bit_for_bit(fa, case):
    """New rows in their places, everything else as it was."""
    new, before, page, hk, d, dtype, cache_dtype, token_major = case
    lens = [a + b for a, b in zip(new, before)]
    kc, vc, table, rows = filled(lens, page, hk, d, cache_dtype, seed=sum(lens), token_major=token_major)
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(2, sum(new), hk + 1, d, generator=gen) * 3).to(dtype)       # rows of a wider tensor
    scales = [torch.rand(hk, generator=gen) * 0.03 + 0.004 for _ in range(2)] if cache_dtype == E4M3 else [None, None]
    want = [kc.clone(), vc.clone()]
    for c, src, s in zip(want, x, scales):
        at = 0
        vals = src[:, :hk].double() if s is None else ref.nearest_e4m3(src[:, :hk].float() / s[:, None])
        for b, (n, m) in enumerate(zip(new, before)):
            for i in range(n):
                bits(c)[int(table[b, (m + i) // page]), :, (m + i) % page] = bits(vals[at + i].to(cache_dtype).contiguous())
            at += n
    dev = on_gpu(kc), on_gpu(vc)
    xd = x.cuda()
    fa.cache_append(xd[0][:, :hk], xd[1][:, :hk], *dev, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ref.offsets(new).cuda(),
                    k_scale=None if scales[0] is None else scales[0].cuda(), v_scale=None if scales[1] is None else scales[1].cuda())
    for got, w in zip(dev, want):
        assert torch.equal(bits(got.cpu().contiguous()), bits(w.contiguous()))


def test_append_e4m3_rounds_every_value_right(fa):
    """Every finite fp16 value, a scale that makes ties and one that does not; NaN stays NaN, what lies beyond 448 and
    the infinities give +-448, signs of zero are kept."""
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(F16)
    hk, d, page = 1, 128, 64
    rows = every.reshape(-1, hk, d)
    pages = rows.shape[0] // page
    table = torch.arange(pages, dtype=torch.int32)[None]
    for scale in (1.0, 0.25, 0.3):
        kc = torch.zeros(pages, hk, page, d, dtype=torch.uint8).view(E4M3).cuda()
        vc = torch.zeros_like(kc)
        s = torch.tensor([scale], dtype=torch.float32).cuda()
        fa.cache_append(rows.cuda(), rows.cuda(), kc, vc, table.cuda(), torch.tensor([rows.shape[0]], dtype=torch.int32).cuda(),
                        ref.offsets([rows.shape[0]]).cuda(), k_scale=s, v_scale=s)
        got = kc.cpu().transpose(1, 2).reshape(-1).view(torch.uint8)
        assert torch.equal(got, vc.cpu().transpose(1, 2).reshape(-1).view(torch.uint8))
        x = every.float() / torch.tensor(scale, dtype=torch.float32)
        nan = torch.isnan(x)
        want = ref.nearest_e4m3(torch.where(nan, 0.0, x).clamp(-448, 448)).to(torch.float32).to(E4M3).view(torch.uint8)
        assert bool((got[nan] & 0x7f == 0x7f).all())
        assert torch.equal(got[~nan], want[~nan]), scale


def test_append_leaves_out_what_has_no_place(fa):
    page, hk, d = 16, 1, 64
    kc, vc, table, _ = filled([40, 40], page, hk, d, F16, seed=31)
    x = torch.randn(30, hk, d, generator=torch.Generator().manual_seed(1)).half()
    bad = table.clone()
    bad[1, 1] = kc.shape[0] + 5
    want = [kc.clone(), vc.clone()]
    # sequence 0: rows 2..10 -> positions 32..40; sequence 1: rows 10..25 -> positions 25..40, of which 25..32 lie in the
    # page that is not there; rows 0, 1 and 25.. belong to no sequence
    for c in want:
        for i in range(8):
            c[int(bad[0, (32 + i) // page]), :, (32 + i) % page] = x[2 + i]
        for i in range(7, 15):
            c[int(bad[1, (25 + i) // page]), :, (25 + i) % page] = x[10 + i]
    dev = kc.cuda(), vc.cuda()
    fa.cache_append(x.cuda(), x.cuda(), *dev, bad.cuda(), torch.tensor([40, 40], dtype=torch.int32).cuda(), torch.tensor([2, 10, 25], dtype=torch.int32).cuda())
    for got, w in zip(dev, want):
        assert torch.equal(bits(got.cpu()), bits(w))
    # lengths that put the new tokens before position 0 or behind the table
    dev = kc.cuda(), vc.cuda()
    fa.cache_append(x[:2].cuda(), x[:2].cuda(), *dev, table.cuda(), torch.tensor([0, 2 ** 31 - 1], dtype=torch.int32).cuda())
    assert torch.equal(bits(dev[0].cpu()), bits(kc)) and torch.equal(bits(dev[1].cpu()), bits(vc))


@pytest.mark.parametrize("dtype,cache_dtype,hq,hk,d", [(BF16, BF16, 8, 2, 128), (F16, E4M3, 4, 4, 64)])
def test_a_server_run(fa, dtype, cache_dtype, hq, hk, d):
    """Prompts of different lengths enter the cache and are attended to, then the batch decodes token by token, one
    sequence ending on the way; the last steps by a captured graph of both calls."""
    page, steps = 16, 20
    prompts = [37, 1, 130, 64]
    gen = torch.Generator().manual_seed(41)
    kc, vc, table = ref.page_pool([n + steps + 1 for n in prompts], page, hk, d, cache_dtype, seed=41)
    kc, vc, tab = kc.cuda(), vc.cuda(), table.cuda()
    ks = vs = None
    if cache_dtype == E4M3:
        ks, vs = (torch.full((hk,), s, dtype=torch.float32).cuda() for s in (0.011, 0.009))
    kept = [[[], []] for _ in prompts]       # rows as the cache holds them, by sequence

    def keep(b, k, v):
        for s, (x, sc) in enumerate(((k, ks), (v, vs))):
            kept[b][s].append(x if sc is None else ref.nearest_e4m3(x.float() / sc.cpu()[:, None]) * float(sc[0]))

    q, k, v = (torch.randn(sum(prompts), h, d, generator=gen).to(dtype) for h in (hq, hk, hk))
    cu, lens = ref.offsets(prompts), torch.tensor(prompts, dtype=torch.int32).cuda()
    fa.cache_append(k.cuda(), v.cuda(), kc, vc, tab, lens, cu.cuda(), k_scale=ks, v_scale=vs, sync=False)
    out = fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), sync=False)
    ref.check_packed(out, q, k, v, prompts, prompts, True, d ** -0.5, heads=[0, hq - 1])
    for b in range(len(prompts)):
        keep(b, k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]])
    x = torch.zeros(len(prompts), hq + 2 * hk, d, dtype=dtype, device="cuda")
    o = torch.empty(len(prompts), hq, d, dtype=dtype, device="cuda")

    def step():
        lens.add_((lens > 0).int())          # a sequence that has ended has length 0
        fa.cache_append(x[:, hq:hq + hk], x[:, hq + hk:], kc, vc, tab, lens, k_scale=ks, v_scale=vs, sync=False)
        fa.decode_paged(x[:, :hq], kc, vc, tab, lens, k_scale=ks, v_scale=vs, out=o, sync=False)

    graph = torch.cuda.CUDAGraph()
    alive = [True] * len(prompts)
    for t in range(steps):
        if t == 8:
            alive[2] = False
            lens[2] = 0
        host = torch.randn(x.shape, generator=gen).to(dtype)
        x.copy_(host.cuda())
        if t < 12:
            step()
        elif t == 12:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
            graph.replay()
        else:
            graph.replay()
        torch.cuda.synchronize()
        for b in range(len(prompts)):
            if alive[b]:
                keep(b, host[b:b + 1, hq:hq + hk], host[b:b + 1, hq + hk:])
        if t in (0, 7, 8, 11, 12, 13, steps - 1):
            rows = [[torch.cat([z.double() for z in kept[b][s]]) if alive[b] else torch.zeros(0, hk, d) for b in range(len(prompts))] for s in range(2)]
            check_decode(o, None, host[:, :hq], rows, [r.shape[0] for r in rows[0]], d ** -0.5, heads=[0, hq - 1], what=f"step {t}")
