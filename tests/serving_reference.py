"""Plain float64 forms of the serving operators, with the error bounds their results are tested against."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # largest relative rounding error of the type


def attention(q, k, v, visible, scale):
    """One head in float64: q [n, d], k and v [m, d], visible [n, m].  Returns (out, lse, spread, rise): spread is the
    weighted mean of |v|, what an error of the weights is multiplied with; rise a bound of the size of the sums
    behind a score, what an fp32 score's error is proportional to."""
    q, k, v = q.double(), k.double(), v.double()
    n, m = visible.shape
    if m == 0:
        zero = torch.zeros(n, v.shape[1], dtype=torch.float64)
        return zero, torch.full((n,), -math.inf, dtype=torch.float64), zero, torch.zeros(n, 1, dtype=torch.float64)
    # (masked keys and values may hold anything: they take no part, not even multiplied by zero)
    s = torch.full((n, m), -math.inf, dtype=torch.float64)
    used = visible.any(0)
    idx = used.nonzero()[:, 0]
    finite_q = q
    s[:, idx] = finite_q @ k[idx].T * scale
    s[~visible] = -math.inf
    lse = torch.logsumexp(s, 1)
    none = ~visible.any(1)
    p = torch.exp(s - torch.where(none, 0.0, lse)[:, None])
    p[none] = 0.0
    out = torch.zeros(n, v.shape[1], dtype=torch.float64)
    spread = torch.zeros_like(out)
    clean = torch.isfinite(v).all(1) & used
    ci = clean.nonzero()[:, 0]
    out += p[:, ci] @ v[ci]
    spread += p[:, ci] @ v[ci].abs()
    for j in (used & ~clean).nonzero()[:, 0].tolist():       # a non-finite value reaches the rows that see it only
        rows = visible[:, j]
        out[rows] += p[rows, j][:, None] * v[j]
        spread[rows] += p[rows, j][:, None] * v[j].abs()
    rise = torch.zeros(n, 1, dtype=torch.float64)
    ki = (torch.isfinite(k).all(1) & used).nonzero()[:, 0]
    if len(ki):
        rise[:, 0] = (q.abs() @ k[ki].abs().T * scale).amax(1)
    return out, lse, spread, rise


def bound(out, spread, rise, keys, d, dtype, weight_bits_rounded):
    """Largest error of a result of these kernels, from their arithmetic.

    * the result is rounded once: HALF_STEP * |out|;
    * the weights p enter the second product in 16 bits (`weight_bits_rounded`: each off by HALF_STEP of itself; fp16
      loses what is below 2^-25 of the largest as well) or as a sum of two 16-bit values (off by its square);
    * scores are sums of d products in fp32 (d * 2^-24 of the sums' size `rise`, both in p and in the sum of the
      p: twice), scaled (2^-23 of a score), and go through a base-2 exponential of one unit in the last place
      (2^-23, twice), p's sum and the second product through `keys` fp32 additions."""
    u = HALF_STEP[dtype]
    p = u if weight_bits_rounded else u * u
    relative = 2 * ((d + 8) * 2.0 ** -24 * (rise + 1) + 2 * 2.0 ** -23) + 2 * keys * 2.0 ** -24
    largest_value = max(8.0, float(spread.amax())) if spread.numel() else 8.0     # standard normal values, or planted ones
    lost = keys * 2.0 ** -25 * largest_value if dtype == torch.float16 else 0.0
    limit = u * out.abs() + (1 + u) * (p + relative) * spread + lost + 1e-30
    # The products are summed before they are divided by the sum of the weights, which is below keys * 2^16 (weights are
    # taken against a score at most 16 powers of two below the largest).  Where that sum passes the range of fp32
    # (bfloat16 values near the type's end; 2^128), an infinity is what arithmetic in 32 bits gives.
    return torch.where(spread * (keys * 2.0 ** 16) >= 2.0 ** 128, float("inf"), limit)


def lse_bound(lse, rise, keys, d):
    """lse: the score error once, the sum's relative error, and two fp32 roundings of the result."""
    return (d + 8) * 2.0 ** -24 * (rise[:, 0] + 1) + 2 * 2.0 ** -23 + keys * 2.0 ** -24 + 4 * 2.0 ** -24 * lse.abs()


def assert_within(got, want, limit, what):
    got, want = got.detach().double().cpu(), want.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    bad = finite & ((got - want).abs() > limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bound, first at "
                           f"{bad.nonzero()[:3].tolist()}: {got[bad][:3].tolist()} for {want[bad][:3].tolist()}, "
                           f"bound {limit.expand_as(want)[bad][:3].tolist()}")


def offsets(lens):
    total = [0]
    for n in lens:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32)


def visible_keys(nq, nk, causal):
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None]
    return (j <= i + (nk - nq)) if causal else torch.ones(nq, nk, dtype=torch.bool)


def check_packed(got, q, k, v, q_lens, k_lens, causal, scale, heads=None, what=""):
    """Every sequence's rows of `got` against the float64 form, for all heads or the listed ones."""
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    aq = ak = 0
    for b, (nq, nk) in enumerate(zip(q_lens, k_lens)):
        for h in range(q.shape[1]) if heads is None else heads:
            out, _, spread, rise = attention(q[aq:aq + nq, h], k[ak:ak + nk, h // group], v[ak:ak + nk, h // group],
                                             visible_keys(nq, nk, causal), scale)
            assert_within(got[aq:aq + nq, h], out, bound(out, spread, rise, nk, d, q.dtype, True),
                          f"{what} sequence {b} ({nq} x {nk}), head {h}")
        aq, ak = aq + nq, ak + nk


def page_pool(lens, page, heads, d, dtype, spare=2, token_major=False, seed=0, width=None):
    """(k_cache, v_cache, table, pages of every sequence): a shuffled pool filled with NaN (e4m3: with its NaN)."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen).tolist()
    table = torch.full((len(lens), max(max(need, default=0), 1) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    shape = (total, page, heads, d) if token_major else (total, heads, page, d)
    caches = []
    for _ in range(2):
        c = torch.full(shape, float("nan"), dtype=torch.float32).to(dtype)
        caches.append(c.transpose(1, 2) if token_major else c)
    return caches[0], caches[1], table


def fill(cache, table, rows, page):
    """rows[b] ([n, heads, d]) into the positions 0 .. n - 1 of sequence b, in place."""
    bits = {1: torch.uint8, 2: torch.int16}[cache.element_size()]
    raw = cache.view(bits)
    for b, x in enumerate(rows):
        for j in range(0, x.shape[0], page):
            piece = x[j:j + page]
            raw[int(table[b, j // page]), :, : piece.shape[0]] = piece.to(cache.dtype).view(bits).transpose(0, 1)


def nearest_e4m3(x):
    """float64 form of the e4m3 rounding: nearest, ties to even, at most 448 in size."""
    x = x.double()
    size = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.round(size / step) * step, x)
