"""Error bounds of the serving operators that hold key by key: what a weight loses in 16 bits is counted from the weight
itself, and sums of products from how many additions follow one another."""
import math

import torch

from serving_reference import HALF_STEP

# Half a step of the smallest values of a type (fp16 has no more bits below 2^-14; bfloat16 reaches as far as fp32)
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
# What the largest weight of a row is held as, at least, where weights go through 16 bits once (prompts) ...
PROMPT_TOP = {torch.float16: 2.0 ** 7, torch.bfloat16: 1.0}
# ... and as the sum of two values (decoding)
DECODE_TOP = {torch.float16: 2.0 ** 15, torch.bfloat16: 1.0}
# A prompt's weights stand up to 2^8 above that, and their products with the values are summed in fp32 before they are
# divided: bfloat16 values near the type's end may pass its range there
PROMPT_RISE = 2.0 ** 8


class Head:
    """One head in float64: q [n, d], k and v [m, d], visible [n, m].  Masked keys and values may hold anything."""

    def __init__(self, q, k, v, visible, scale):
        q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
        n, m = visible.shape
        s = torch.full((n, m), -math.inf, dtype=torch.float64)
        self.rise = torch.zeros(n, 1, dtype=torch.float64)          # size of the sums behind a score
        used = visible.any(0).nonzero()[:, 0]
        if len(used):
            s[:, used] = q @ k[used].T * scale
            size = torch.where(visible[:, used], q.abs() @ k[used].abs().T * scale, 0.0)
            self.rise[:, 0] = size.amax(1)
        s[~visible] = -math.inf
        self.lse = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64)
        none = ~visible.any(1) if m else torch.ones(n, dtype=torch.bool)
        self.p = torch.exp(s - torch.where(none, 0.0, self.lse)[:, None])
        self.p[none] = 0.0
        self.top = self.p.amax(1, keepdim=True) if m else torch.zeros(n, 1, dtype=torch.float64)
        self.v = torch.where(visible.any(0)[:, None], v, 0.0) if m else v
        self.out, self.spread = self.p @ self.v, self.p @ self.v.abs()
        self.keys, self.d, self.none = m, q.shape[1], none

    def limit(self, dtype, top, single):
        """Largest error of a result of `dtype`:

        * its own rounding: u |out|, half a step of the type's smallest values;
        * weights in 16 bits: each off by u of itself (one value; the sum of the weights is taken from them or from the
          exact ones, so that u (spread + |out|) covers both) or by u^2 (two values), and by at most SMALLEST where the
          largest is held as `top`, never by more than itself;
        * scores: d products in fp32 and a few operations on a score, an exponential of one unit, in the weights and in
          their sum (twice);
        * sums: at most keys / 8 + 40 additions in fp32 follow one another (8 keys of a lane a step, 32 products inside a
          matrix instruction, joins), in the products and in the weights."""
        u = HALF_STEP[dtype]
        relative = 2 * ((self.d + 8) * 2.0 ** -24 * (self.rise + 1) + 2 * 2.0 ** -23) + 2 * (self.keys / 8 + 40) * 2.0 ** -24
        weights = u * (self.spread + self.out.abs()) if single else 2 * u * u * self.spread
        floor = SMALLEST[dtype] / top * self.top
        least = torch.minimum(self.p, floor)
        lost = least @ self.v.abs() + least.sum(1, keepdim=True) * self.out.abs()
        return u * self.out.abs() + SMALLEST[dtype] + (1 + u) * (weights + relative * self.spread + lost) + 1e-38

    def may_overflow(self):
        """Where a prompt's sum of products, before it is divided, may pass the range of fp32 (half of it: the sum's own
        errors are far below that)."""
        total = self.spread / torch.where(self.top > 0, self.top, 1.0) * PROMPT_RISE
        return total >= 2.0 ** 127

    def check(self, got, dtype, what, decoding):
        got = got.detach().double().cpu()
        assert got.shape == self.out.shape, what
        assert bool((got[self.none] == 0).all()), f"{what}: rows that see no key"
        limit = self.limit(dtype, (DECODE_TOP if decoding else PROMPT_TOP)[dtype], not decoding)
        bad = ~((got - self.out).abs() <= limit)
        if not decoding:
            bad &= ~(self.may_overflow() & torch.isinf(got) & (got.sign() == self.out.sign()))
        assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bound, first at {bad.nonzero()[:3].tolist()}: "
                               f"{got[bad][:3].tolist()} for {self.out[bad][:3].tolist()}, bound {limit[bad][:3].tolist()}")


def check_prompts(got, q, k, v, q_lens, k_lens, causal, scale, heads=None, what=""):
    from serving_reference import visible_keys
    group = q.shape[1] // k.shape[1]
    aq = ak = 0
    for b, (nq, nk) in enumerate(zip(q_lens, k_lens)):
        for h in range(q.shape[1]) if heads is None else heads:
            head = Head(q[aq:aq + nq, h], k[ak:ak + nk, h // group], v[ak:ak + nk, h // group], visible_keys(nq, nk, causal), scale)
            head.check(got[aq:aq + nq, h], q.dtype, f"{what} sequence {b} ({nq} x {nk}), head {h}", False)
        aq, ak = aq + nq, ak + nk


def check_decoding(got, q, rows, lens, scale, ks=None, vs=None, heads=None, what=""):
    """rows: [K, V][sequence] of [n, kv_heads, d], as the cache holds them; ks, vs: what a stored 1 stands for."""
    hk = rows[0][0].shape[1]
    for b, n in enumerate(lens):
        for h in range(q.shape[1]) if heads is None else heads:
            g = h // (q.shape[1] // hk)
            k, v = (r[b][:, g].double() * (1.0 if s is None else float(s[g])) for r, s in zip(rows, (ks, vs)))
            head = Head(q[b:b + 1, h], k, v, torch.ones(1, n, dtype=torch.bool), scale)
            head.check(got[b:b + 1, h], q.dtype, f"{what} sequence {b} (length {n}), head {h}", True)
