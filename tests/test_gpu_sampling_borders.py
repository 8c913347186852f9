"""Sampling by row where its arithmetic is nearest to going wrong, against the definition (_sample_ref.py)."""
import math
from fractions import Fraction

import pytest
import torch

import _sample_ref as ref
from test_gpu_sampling import check, run

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def test_a_largest_logit_whose_bin_lies_next_to_a_half():
    """At temperature 1e-12 a logit is worth thousands of millions of bins: of some, the product rounded to a double has another
    nearest integer than the product itself.  Both filters' launches and the plain ones; whatever lies beside has no weight."""
    heat = float(torch.tensor(1e-12, dtype=F32))
    c4 = 4.0 * 1.4426950408889634 / heat
    g = torch.Generator().manual_seed(1)
    tops = [v for v in torch.rand(400000, generator=g).tolist() if round(v * c4) != round(Fraction(v) * Fraction(c4))]
    assert len(tops) >= 32
    x = torch.zeros(32, 9000)
    x[:, 4321] = torch.tensor(tops[:32])
    for s in (dict(heat=1e-12), dict(heat=1e-12, k=5), dict(heat=1e-12, p=0.9), dict(heat=1e-12, m=0.1)):
        got, lp = run(x, [0.0, 0.5, 1.0, 0.999] * 8, [s] * 32)
        assert got == [4321] * 32 and max(abs(v) for v in lp) <= 2.0 ** -33, s
    assert [ref.row(x[0], u, heat=heat)[0] for u in (0.0, 0.999)] == [4321] * 2


def last_kept(n, w, k, p):
    """Of a largest logit of weight 1 and n equal ones of weight w: how many of those top-k and then top-p leave, and
    what all that is kept weighs (exact fractions)."""
    n = min(n, k - 1)
    share = p * (1 + n * w) - 1
    kept = max(0, min(n, math.ceil(share / w)))
    assert kept in (0, n) or abs(share / w - round(share / w)) > 0.01, "the case itself is on a border"
    return kept, 1 + kept * w


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [9000, 60000, 248320])
@pytest.mark.parametrize("down,ps", [(12.125, (0.99, 0.999)), (17.28125, (0.99, 0.999, 0.9999)), (17.328125, (0.99999,)),
                                     (26.0, (1 - 2.0 ** -21, 1 - 2.0 ** -22, 1 - 2.0 ** -23))])
def test_an_equal_tail_far_below_one_peak(down, ps, V, dtype):
    """Top-k of most of the tail, then top-p within it, 70, 100 and 150 bins below the largest: how many of them are kept,
    and each drawn where its weight lies, at the ends of the chunks too.

    Weights are 2^-35.75 of themselves off at most and sums in doubles 2^-50 of the whole: of 250000 logits a border moves by
    2^-17 of a logit, and where each is 2^-37.5 of the whole by 2^-12 more.  u, a float, is off by 2^-24 of u, 2^-6 of a
    logit, and lies half a logit from its borders."""
    w = Fraction(math.exp(-down))      # 2^-52 of itself off
    x = torch.full((1, V), 20.0 - down, dtype=dtype)
    assert float(x[0, 0]) == 20.0 - down
    x[0, -1] = 20.0                    # behind the others, so that small u find them
    for p in ps:
        p32 = Fraction(float(torch.tensor(p, dtype=F32)))
        for k in (V // 5 * 4, V - 1, 5000):
            kept, whole = last_kept(V - 1, w, k, p32)
            places = sorted({0, 1, 100, 8191, 8192, 16383, 16384, kept // 2, 57343, kept - 2, kept - 1})
            places = [t for t in places if 0 <= t < kept]
            u = [float((t + Fraction(1, 2)) * w / whole) for t in places]
            want = list(places)
            if kept:
                u.append(float((kept + Fraction(1, 2)) * w / whole))
                want.append(V - 1)
            half = whole / 2 / w        # u = 1/2 may fall into the tail
            assert half > kept or abs(half - round(half)) > 0.01
            u += [0.5, 1.0]
            want += [V - 1 if half > kept else int(half), V - 1]
            got, lp = run(x.expand(len(u), V), u, [dict(k=k, p=p)] * len(u))
            assert got == want, (p, k, kept)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [30000, 100001, 248320])
@pytest.mark.parametrize("spread", [0.0, 0.02, 0.5, 2.0])
def test_a_tail_far_below_a_few_peaks(spread, V, dtype):
    """The same with tails of different logits and a min-p among them, against the definition in 64 bits."""
    g = torch.Generator().manual_seed(int(100 * spread) + V)
    x = torch.randn(1, V, generator=g) * spread + 2.0
    x[0, torch.randint(0, V, (5,), generator=g)] = torch.tensor([14.0, 16.5, 17.0, 19.0, 19.5])
    x = x.to(dtype)
    s, u = [], []
    for k in (V // 2, V // 5 * 4, 20000):
        for p in (0.9, 0.95, 0.99, 0.999, 0.9999):
            for m in (0.0, 1e-8, 2.0 ** -25):
                s.append(dict(k=k, p=p, m=m))
                u.append(float(torch.rand(1, generator=g)) ** 4)
    check(x.expand(len(s), V), u, s, leave=6)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("spread", [0.0, 0.01, 1.0])
def test_the_largest_vocabulary(spread, dtype):
    """2^20 logits, most of them in the range of the cuts: more than a row's list has places for."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, 2**20, generator=g) * spread - 3.0
    x[0, 2**20 - 7], x[0, 12] = 9.0, 5.5
    s = [dict(k=k, p=p, m=m) for k in (0, 1000, 700001, 2**20 - 1) for p in (1.0, 0.9375, 0.5) for m in (0.0, 1e-7)]
    u = torch.rand(len(s), generator=g).tolist()
    check(x.to(dtype).expand(len(s), -1), u, s, leave=8)
