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


def test_more_short_prompts_than_one_dimension_of_a_grid_holds(fa):
    """2^19 prompts of a row or two, 32 heads: over 2^24 (prompt, head) pairs."""
    heads, d, sequences = 32, 8, 1 << 19
    lens = torch.ones(sequences, dtype=torch.int64)
    lens[5::1000] = 0
    lens[7::997] = 2
    lens[:4] = torch.tensor([70, 3, 0, 130])
    total = int(lens.sum())
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(total, heads, d, generator=gen, device="cuda").to(BF16)
    k, v = (torch.randn(total, 1, d, generator=gen, device="cuda").to(BF16) for _ in range(2))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    got = fa.forward_packed(q, k, v, cu.to(torch.int32).cuda())
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
