"""GPU: the serving operators at the ends of what they take, against the float64 forms of serving_reference."""
import pytest
import torch

import serving_bounds as bounds
import serving_reference as ref
from test_paged_gpu import check_decode, filled, on_gpu

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("page,token_major", [(16, False), (4, True)])
@pytest.mark.parametrize("d", [8, 24, 40, 56, 72, 88, 104, 120, 16, 48, 112])
def test_rows_at_the_end_of_an_8_bit_cache(fa, d, page, token_major):
    """Rows that are no whole number of 16-byte loads, the last one of them the cache's last bytes."""
    lens = [page * 21, page * 3, 5 * page + 1]
    kc, vc, table, rows = filled(lens, page, 2, d, E4M3, seed=d, token_major=token_major)
    last = int(table.max())
    kc, vc = kc[: last + 1], vc[: last + 1]
    q = torch.randn(3, 6, d, generator=torch.Generator().manual_seed(1)).to(BF16)
    got, lse = fa.decode_paged(q.cuda(), on_gpu(kc), on_gpu(vc), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softmax_scale=0.003,
                               return_lse=True)
    check_decode(got, lse, q, rows, lens, 0.003)


def test_last_row_of_a_cache_of_whole_allocation_pages(fa):
    """80 MiB exactly, of which the last row is read."""
    page, hk, d, pages = 16, 8, 40, 16384
    gen = torch.Generator().manual_seed(2)
    rows = [[torch.randn(48, hk, d, generator=gen).mul(20).to(E4M3)] for _ in range(2)]
    table = torch.tensor([[pages - 2, 0, pages - 1]], dtype=torch.int32)
    caches = []
    for r in rows:
        c = torch.zeros((pages, hk, page, d), dtype=torch.uint8, device="cuda")
        assert c.numel() % (2 << 20) == 0
        for j in range(3):
            c[int(table[0, j])] = r[0][16 * j:16 * j + 16].view(torch.uint8).transpose(0, 1).cuda()
        caches.append(c.view(E4M3))
    q = torch.randn(1, 16, d, generator=gen).to(F16)
    got = fa.decode_paged(q.cuda(), *caches, table.cuda(), torch.tensor([48], dtype=torch.int32).cuda(), softmax_scale=0.004)
    check_decode(got, None, q, rows, [48], 0.004)


@pytest.mark.parametrize("heads,lens", [(8, [1700]), (8, [1000, 2000]), (2, [2048]), (16, [1536])])
def test_as_many_keys_as_queries_with_offsets_of_their_own(fa, heads, lens):
    """Key offsets in a tensor of their own, with the same totals: the same result as without, and other places too."""
    gen = torch.Generator().manual_seed(heads)
    total, d = sum(lens), 64
    q, k, v = (torch.randn(total, h, d, generator=gen).to(F16) for h in (heads, 1, 1))
    cu = ref.offsets(lens).cuda()
    args = [x.cuda() for x in (q, k, v)]
    got = fa.forward_packed(*args, cu, cu.clone())
    ref.check_packed(got, q, k, v, lens, lens, True, d ** -0.5, heads=[0, heads - 1])
    k_lens = [lens[0] + 0] if len(lens) == 1 else [lens[0] + 300, lens[1] - 300]
    got = fa.forward_packed(*args, cu, ref.offsets(k_lens).cuda())
    ref.check_packed(got, q, k, v, lens, k_lens, True, d ** -0.5, heads=[0, heads - 1])


@pytest.mark.parametrize("sequences,own_offsets", [(1 << 19, False), (400000, False), (400000, True)])
def test_more_short_prompts_than_one_dimension_of_a_grid_holds(fa, sequences, own_offsets):
    """Prompts of a row or two, 32 heads: over 2^24 (prompt, head) pairs, or, with two places for each prompt, twice as many
    as are there, on either side of that."""
    heads, d = 32, 8
    lens = torch.ones(sequences, dtype=torch.int64)
    lens[5::1000] = 0
    lens[7::997] = 2
    lens[:4] = torch.tensor([70, 3, 0, 130])
    total = int(lens.sum())
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(total, heads, d, generator=gen, device="cuda").to(BF16)
    k, v = (torch.randn(total, 1, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    cu_q = cu.to(torch.int32).cuda()
    got = fa.forward_packed(q, k, v, cu_q, cu_q.clone() if own_offsets else None)
    ref.check_packed(got[:203], q[:203], k[:203], v[:203], [70, 3, 0, 130], [70, 3, 0, 130], True, d ** -0.5, heads=[0, 31])
    first = cu[:-1][lens > 0].cuda()            # a prompt's first row sees itself alone
    assert torch.equal(got[first], v[first].expand(-1, heads, -1))
    last = total - int(lens[-600:].sum())
    tail = [int(n) for n in lens[-600:]]
    ref.check_packed(got[last:], q[last:], k[last:], v[last:], tail, tail, True, d ** -0.5, heads=[17])


def leading_key(n, heads, d, at, ahead, dtype, seed, tail=1.0):
    """(k, v): scores of about 0 against a query of ones at scale 1 / d, but for key `at`, which leads by `ahead` powers of
    two and has the value 0 (a key that takes what attention is not needed elsewhere); the others' values have mean `tail`."""
    gen = torch.Generator().manual_seed(seed)
    k = torch.randn(n, heads, d, generator=gen) * 0.05
    k[at] = ahead * 0.6931
    v = tail + 0.25 * torch.randn(n, heads, d, generator=gen)
    v[at] = 0.0
    return k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("ahead", [4, 14, 20, 24, 27, 31, 36])
@pytest.mark.parametrize("n,page,d,dtype,cache", [(20011, 16, 128, F16, F16), (300, 16, 64, F16, F16), (4000, 8, 72, F16, F16), (20011, 16, 64, BF16, BF16),
                                                  (5000, 32, 128, F16, E4M3)])
def test_decoding_with_one_leading_key(fa, n, page, d, dtype, cache, ahead):
    """The tail's weights, far below the leading one's, are what the result consists of."""
    ks, vs = (torch.tensor([0.0625]), torch.tensor([0.25])) if cache == E4M3 else (None, None)
    k, v = leading_key(n, 1, d, n // 3, ahead, torch.float32, 7)
    rows = [[(x if s is None else x / s).to(cache)] for x, s in ((k, ks), (v, vs))]
    kc, vc, table = ref.page_pool([n], page, 1, d, cache, seed=3)
    for c, r in zip((kc, vc), rows):
        ref.fill(c, table, r, page)
    q = torch.ones(1, 2, d, dtype=dtype)
    dev = [None if s is None else s.cuda() for s in (ks, vs)]
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), softmax_scale=1.0 / d,
                          k_scale=dev[0], v_scale=dev[1])
    bounds.check_decoding(got, q, rows, [n], 1.0 / d, ks, vs, what=f"{ahead} ahead")


@pytest.mark.parametrize("cut", [0, 1])
@pytest.mark.parametrize("d,dtype,cache", [(128, F16, F16), (64, BF16, BF16), (112, BF16, E4M3)])
def test_decoding_within_the_bounds_of_its_weights(fa, d, dtype, cache, cut):
    lens = [[700, 33, 1], [9000]][cut]
    kc, vc, table, rows = filled(lens, 16, 2, d, cache, seed=d)
    q = torch.randn(len(lens), 4, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    scale = 0.01 if cache == E4M3 else d ** -0.5
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softmax_scale=scale)
    bounds.check_decoding(got, q, rows, lens, scale)


PROMPTS = [
    # q_lens, k_lens, query heads, d, type, causal, K rows apart (0: adjacent)
    ([400, 90], [400, 90], 2, 128, F16, True, 0),           # 128-row items
    ([300], [700], 2, 64, F16, False, 0),
    ([4200], [4200], 32, 64, F16, True, 0),                 # 256-row items
    ([70], [6000], 2, 128, F16, True, 0),                   # the keys of a row dealt to several workgroups
    ([33, 150], [2500, 3100], 2, 72, F16, False, 0),
    ([60], [300], 2, 64, F16, True, (1 << 21) + 64),        # row by row
    ([400], [400], 2, 64, BF16, True, 0),
    ([70], [6000], 2, 128, BF16, True, 0),
]


@pytest.mark.parametrize("at,ahead", [(0, 4), (0, 20), (0, 25), (0, 29), (0.4, 14), (0.4, 20), (0.4, 25), (0.9, 25), ("two", 14), ("two", 18)])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"q{'-'.join(map(str, c[0]))}_k{'-'.join(map(str, c[1]))}_{c[2]}h_d{c[3]}_{str(c[4])[6:]}_{'causal' if c[5] else 'all'}_{c[6]}")
def test_prompts_with_one_leading_key(fa, case, at, ahead):
    """As for decoding.  "two": the first key leads and one in the middle leads by 7.5 powers of two more, which moves no
    reference."""
    q_lens, k_lens, heads, d, dtype, causal, apart = case
    parts = []
    for b, n in enumerate(k_lens):
        k, v = leading_key(n, 1, d, 0 if at == "two" else int(at * n), ahead, dtype, b)
        if at == "two":
            k[n // 2], v[n // 2] = ((ahead + 7.5) * 0.6931), 0.0
        parts.append((k, v))
    k, v = (torch.cat(x) for x in zip(*parts))
    q = torch.ones(sum(q_lens), heads, d, dtype=dtype)
    kd = k.cuda()
    if apart:
        kd = torch.zeros(k.shape[0], apart, dtype=dtype, device="cuda")[:, :d].unflatten(1, (1, d))
        kd.copy_(k)
    got = fa.forward_packed(q.cuda(), kd, v.cuda(), ref.offsets(q_lens).cuda(), ref.offsets(k_lens).cuda(), causal=causal, softmax_scale=1.0 / d)
    bounds.check_prompts(got, q, k, v, q_lens, k_lens, causal, 1.0 / d, heads=[0])


@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"q{'-'.join(map(str, c[0]))}_k{'-'.join(map(str, c[1]))}_{c[2]}h_d{c[3]}_{str(c[4])[6:]}_{'causal' if c[5] else 'all'}_{c[6]}")
@pytest.mark.parametrize("scale", [0.125, 2.0, 1e-30, 2e-38])
def test_prompts_within_the_bounds_of_their_weights(fa, case, scale):
    """Ordinary values, at ordinary scales and where the softmax has one key or all of them."""
    q_lens, k_lens, heads, d, dtype, causal, apart = case
    gen = torch.Generator().manual_seed(sum(k_lens))
    q = torch.randn(sum(q_lens), heads, d, generator=gen).to(dtype)
    k, v = (torch.randn(sum(k_lens), 1, d, generator=gen).to(dtype) for _ in range(2))
    kd = k.cuda()
    if apart:
        kd = torch.zeros(k.shape[0], apart, dtype=dtype, device="cuda")[:, :d].unflatten(1, (1, d))
        kd.copy_(k)
    got = fa.forward_packed(q.cuda(), kd, v.cuda(), ref.offsets(q_lens).cuda(), ref.offsets(k_lens).cuda(), causal=causal, softmax_scale=scale)
    bounds.check_prompts(got, q, k, v, q_lens, k_lens, causal, scale, heads=[0])


@pytest.mark.parametrize("page,lens", [(16, [2, 700, 3000]), (2, [40]), (16, [20000])])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 40), (F16, 64)])
def test_decoding_values_at_the_end_of_the_range(fa, page, lens, dtype, d):
    """Means of the type's largest values are finite, whatever their sum would be."""
    kc, vc, table, rows = filled(lens, page, 1, d, dtype, seed=5)
    gen = torch.Generator().manual_seed(4)
    rows[1] = [(torch.finfo(dtype).max * (0.5 + 0.49 * torch.rand(n, 1, d, generator=gen))).to(dtype) for n in lens]
    for b in range(len(lens)):
        rows[1][b][:, :, ::3] *= -1
        rows[1][b][1::2, :, 1::3] *= -1
    ref.fill(vc, table, rows[1], page)
    q = torch.randn(len(lens), 2, d, generator=gen).to(dtype)
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    bounds.check_decoding(got, q, rows, lens, d ** -0.5)


@pytest.mark.parametrize("nq,nk,d,dtype,causal", [(333, 333, 128, BF16, True), (290, 290, 64, F16, True), (150, 2300, 128, BF16, True), (90, 400, 72, BF16, False),
                                                 (60, 300, 64, F16, False)])
def test_prompts_with_the_lowest_values(fa, nq, nk, d, dtype, causal):
    """The type's lowest value in some values, seen by some rows and not by others: within the ordinary bound, or, where the
    sum of the products may pass the range of fp32, an infinity of the right sign; never another number, never NaN."""
    gen = torch.Generator().manual_seed(nk)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype) for n, h in ((nq, 2), (nk, 1), (nk, 1)))
    for row in (40, nk - 149, nk - 70, nk - 3):
        v[max(row, 0), 0, 3::7] = torch.finfo(dtype).min
    got = fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), ref.offsets([nq]).cuda(), ref.offsets([nk]).cuda(), causal=causal)
    bounds.check_prompts(got, q, k, v, [nq], [nk], causal, d ** -0.5)
    near = v.clone()
    near[near < -1e30] = -2.0 ** 90 if dtype == BF16 else -6e4      # far from the end: no infinity
    got = fa.forward_packed(q.cuda(), k.cuda(), near.cuda(), ref.offsets([nq]).cuda(), ref.offsets([nk]).cuda(), causal=causal)
    bounds.check_prompts(got, q, k, near, [nq], [nk], causal, d ** -0.5)
    assert bool(torch.isfinite(got).all())


def test_decoding_with_the_lowest_values(fa):
    lens, d = [700, 50, 3000], 128
    kc, vc, table, rows = filled(lens, 16, 1, d, BF16, seed=8)
    for r in rows[1]:
        r[::9, 0, 3::7] = torch.finfo(BF16).min
    ref.fill(vc, table, rows[1], 16)
    q = torch.randn(3, 4, d, generator=torch.Generator().manual_seed(1)).to(BF16)
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    bounds.check_decoding(got, q, rows, lens, d ** -0.5)
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("d,dtype,causal", [(128, BF16, True), (64, F16, True), (64, F16, False)])
@pytest.mark.parametrize("bad", [float("nan"), -float("nan"), float("inf")])
def test_a_query_that_is_no_number_stays_by_itself(fa, d, dtype, causal, bad):
    """Rows that share a wave with one whose scores are NaN or infinite, while their own references have to move."""
    n = 700
    gen = torch.Generator().manual_seed(d)
    q, k, v = (torch.randn(n, h, d, generator=gen).to(dtype) for h in (2, 1, 1))
    for j, gain in ((70, 0.3), (200, 1.0), (401, 2.0), (650, 3.5)):
        k[j] = q[j, 0] * gain
    cu = ref.offsets([n]).cuda()
    want = fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), cu, causal=causal)
    bounds.check_prompts(want, q, k, v, [n], [n], causal, d ** -0.5, heads=[0])
    rows = torch.tensor([3, 77, 300, 301, 540])
    q[rows] = bad
    got = fa.forward_packed(q.cuda(), k.cuda(), v.cuda(), cu, causal=causal)
    others = torch.ones(n, dtype=torch.bool)
    others[rows] = False
    assert torch.equal(got.cpu()[others].view(torch.int16), want.cpu()[others].view(torch.int16))
    assert bool(torch.isnan(got.cpu()[rows]).all())


def test_writes_are_seen_by_autograd(fa):
    """An output, a cache or scratch that was saved for a backward pass and is then written counts as modified in place;
    tensors of inference mode, which have no version, are taken."""
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    one = torch.tensor([3], dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 200, dtype=torch.int32, device="cuda")
    q = torch.ones(6, 2, 64, dtype=F16, device="cuda")

    def tensors():
        return (torch.zeros(6, 2, 64, dtype=F16, device="cuda"), torch.zeros(1, 2, 64, dtype=F16, device="cuda"),
                torch.zeros(2, 2, 16, 64, dtype=F16, device="cuda"), torch.zeros(2, 2, 16, 64, dtype=F16, device="cuda"),
                torch.zeros(1 << 24, dtype=torch.uint8, device="cuda"))

    def calls(out, step, kc, vc, scratch):
        return ((lambda: fa.forward_packed(q, q, q, cu, out=out), [out]), (lambda: fa.cache_append(q[:1], q[:1], kc, vc, table, one), [kc, vc]),
                (lambda: fa.decode_paged(q[:1], kc, vc, table, one, out=step, workspace=scratch), [step, scratch]))

    for call, written in calls(*tensors()):
        before = [t._version for t in written]
        saved = written[0]
        w = torch.ones_like(saved, requires_grad=True)
        product = (w * saved).sum()
        call()
        assert all(t._version > v for t, v in zip(written, before))
        assert [t._version for t in (q, cu, table, one)] == [0, 0, 0, 0]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
    with torch.inference_mode():
        made = tensors()
    for call, written in calls(*made):
        call()
        assert bool(torch.isfinite(written[0].float()).all())


def test_scratch_of_streams_is_given_back(fa):
    """What calls keep for their streams returns to the allocator; calls that run meanwhile and a captured one are not disturbed."""
    fa.release_workspaces()
    lens = [3000, 1200]
    kc, vc, table, _ = filled(lens, 16, 2, 128, F16, seed=33)
    gen = torch.Generator().manual_seed(1)
    args = (torch.randn(2, 4, 128, generator=gen).half().cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    q, k, v = (torch.randn(n, h, 128, generator=gen).half().cuda() for n, h in ((130, 2), (4200, 1), (4200, 1)))
    cus = ref.offsets([130]).cuda(), ref.offsets([4200]).cuda()
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    want = fa.decode_paged(*args), fa.forward_packed(q, k, v, *cus)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured = fa.decode_paged(*args, sync=False), fa.forward_packed(q, k, v, *cus, sync=False)
    fa.release_workspaces()
    before = torch.cuda.memory_allocated()
    got = []
    for turn in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((fa.decode_paged(*args, sync=False), fa.forward_packed(q, k, v, *cus, sync=False)))
        graph.replay()
        if turn % 2 == 1:
            fa.release_workspaces()
            other = [torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]     # takes freed memory
            del other
    torch.cuda.synchronize()
    for x in got + [captured]:
        assert all(torch.equal(a, b) for a, b in zip(x, want))
    outputs = sum(t.untyped_storage().nbytes() for x in got for t in x)
    assert torch.cuda.memory_allocated() - before < outputs + (1 << 20)
    fa.decode_paged(*args)
    assert torch.cuda.memory_allocated() - before > 10 << 20
    fa.release_workspaces()
    assert torch.cuda.memory_allocated() - before < outputs + (1 << 20)


@pytest.mark.parametrize("page", [16, 2])
@pytest.mark.parametrize("d,dtype", [(40, BF16), (72, F16), (120, BF16), (128, F16), (64, BF16), (8, F16)])
@pytest.mark.parametrize("column", [0, -1, -8])
def test_an_infinite_element_of_a_key(fa, page, d, dtype, column):
    """A score of minus infinity is a weight of nothing, at head dims that leave lanes without columns too."""
    n = 77
    kc, vc, table, rows = filled([n], page, 1, d, dtype, seed=d)
    q = torch.randn(1, 2, d, generator=torch.Generator().manual_seed(1)).abs().to(dtype)
    rows[0][0][[5, 40, 76], 0, column] = -float("inf")
    ref.fill(kc, table, rows[0], page)
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda())
    keep = [j for j in range(n) if j not in (5, 40, 76)]
    bounds.check_decoding(got, q, [[r[0][keep]] for r in rows], [len(keep)], d ** -0.5)


@pytest.mark.parametrize("dtype,scale", [(BF16, 1e33), (BF16, 3e-38), (F16, 100.0), (F16, 1e-7)])
@pytest.mark.parametrize("lens", [[40, 0], [5000, 1]])
def test_scales_of_values_of_any_size(fa, dtype, scale, lens):
    """What a stored 1 stands for enters the result as it is, whatever the weights are held as."""
    kc, vc, table, rows = filled(lens, 16, 1, 64, E4M3, seed=4)
    q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    vs = torch.tensor([scale])
    got = fa.decode_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), softmax_scale=0.005, v_scale=vs.cuda())
    bounds.check_decoding(got, q, rows, lens, 0.005, None, vs)


def test_waiting_inside_a_capture_is_refused(fa):
    """Each operator with its default sync=True: an error in front of the launch, and the capture goes on."""
    lens = [300, 2000]
    kc, vc, table, _ = filled(lens, 16, 2, 64, F16, seed=3)
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 64, generator=gen).half().cuda() for n, h in ((2, 4), (2, 2), (2, 2)))
    rest = (kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    want = fa.decode_paged(q, *rest), fa.forward_packed(q, k, v, cu)
    out = torch.empty_like(q), torch.empty_like(q)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        fa.decode_paged(q, *rest, out=out[0], sync=False)
        for call in (lambda: fa.decode_paged(q, *rest, out=out[0]), lambda: fa.forward_packed(q, k, v, cu, out=out[1]),
                     lambda: fa.cache_append(k, v, *rest)):
            with pytest.raises(ValueError, match="sync=False"):
                call()
        fa.forward_packed(q, k, v, cu, out=out[1], sync=False)
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
