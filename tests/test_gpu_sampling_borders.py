"""Sampling by row where its arithmetic is nearest to going wrong, against the definition (_sample_ref.py)."""
import math
from fractions import Fraction

import pytest
import torch

import _sample_ref as ref
from test_gpu_sampling import run

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
