"""CPU only: the bounds of serving_bounds tell a right result from a wrong one (the wrong ones are planted in the oracle)."""
import pytest
import torch

import serving_bounds as bounds

F16, BF16 = torch.float16, torch.bfloat16


def head(n, dtype, ahead, seed=0):
    gen = torch.Generator().manual_seed(seed)
    d = 64
    k, v = torch.randn(n, d, generator=gen) * 0.05, 1.0 + 0.25 * torch.randn(n, d, generator=gen)
    if ahead:
        k[n // 3], v[n // 3] = ahead * 0.6931, 0.0
    return bounds.Head(torch.ones(1, d, dtype=dtype), k.to(dtype), v.to(dtype), torch.ones(1, n, dtype=torch.bool), 1.0 / d)


@pytest.mark.parametrize("decoding", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,ahead", [(40, 0), (20000, 0), (20000, 20), (20000, 26)])
def test_right_results_pass_and_wrong_ones_do_not(dtype, n, ahead, decoding):
    h = head(n, dtype, ahead)
    h.check(h.out.to(dtype), dtype, "rounded once", decoding)
    for wrong in (torch.zeros_like(h.out), 1.02 * h.out, torch.full_like(h.out, float("nan")), torch.full_like(h.out, float("inf")), -h.out):
        with pytest.raises(AssertionError):
            h.check(wrong.to(dtype), dtype, "wrong", decoding)


def test_tails_lost_in_16_bits_are_found():
    """Weights against the row's largest, rounded to fp16 as they are: 2^26 behind the leading key nothing is left of them."""
    h = head(20000, F16, 26)
    p = (h.p / h.top).to(F16).double()
    got = p @ h.v / p.sum()
    assert float(got.abs().max()) == 0.0
    for decoding in (False, True):
        with pytest.raises(AssertionError):
            h.check(got, F16, "lost", decoding)
    raised = ((h.p / h.top * 128).to(F16).double()) / 128
    h.check((raised @ h.v / raised.sum()).to(F16), F16, "raised", False)
    twice = h.p / h.top * 32768
    high = twice.to(F16).double()
    both = (high + (twice - high).to(F16).double()) / 32768
    h.check((both @ h.v / (h.p / h.top).sum()).to(F16), F16, "in two parts", True)


def test_infinities_only_where_sums_may_pass_fp32():
    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn(n, 64, generator=gen).to(BF16) for n in (3, 200))
    visible = torch.ones(3, 200, dtype=torch.bool)
    for value, may in ((3e38, True), (1e20, False)):
        v = torch.full((200, 64), -value).to(BF16)
        h = bounds.Head(q, k, v, visible, 0.125)
        assert bool(h.may_overflow().all()) == may
        infinite = torch.full_like(h.out, -float("inf"))
        if may:
            h.check(infinite, BF16, "an infinity of the right sign", False)
        for wrong, decoding in ((-infinite, False), (infinite, True), (infinite * 0, False), (0.9 * h.out, False)) + (() if may else ((infinite, False),)):
            with pytest.raises(AssertionError):
                h.check(wrong, BF16, "wrong", decoding)
