"""Adapters of many requests: outputs that have to be finite numbers, and where infinities have to come out."""
import math

import pytest
import torch

from qwen35_amd import adapters

from test_gpu_adapters import BF, DEV, INT, case, pool, reference

pytestmark = pytest.mark.gpu
# few tokens, few columns of many, and the wide form, whose pieces of 64 tokens and 512 columns are 160 or more
SHAPES = [(1, 136), (40, 1000), (300, 264), (300, 16392), (701, 7176)]


def add(c, out=None):
    x, ids, y, a, b, scale = c
    ws = adapters.adapters_workspace(len(x), a.shape[1], device=DEV).fill_(0xFF)    # NaN, until it is written
    return pool(a, b, scale).add(x.to(DEV), ids.to(DEV), y.to(DEV), ws, out=out).cpu()


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("R", [8, 16, 24, 32, 56, 64, 72, 128])
@pytest.mark.parametrize("K", [72, 2560])
def test_every_output_is_a_number_within_its_bound(T, N, R, K):
    """Against 64 bits (the bound is derived in `reference`): an output that is no number is not within it, as it would be where nothing
    had been written to the workspace in front of it."""
    if K == 2560 and N > 8192:
        K = 136
    g = torch.Generator().manual_seed(T + N + R)
    ids = torch.randint(-1, 5, (-(-T // 7),), generator=g).repeat_interleave(7)[:T]
    c = case(T, R, K, N, 5, T + N + R + K, ids)
    got = add(c).double()
    want, err = reference(*c)
    assert bool(got.isfinite().all())
    assert bool(((got - want).abs() <= err).all()), float(((got - want).abs() / err.clamp(min=1e-30)).max())


@pytest.mark.parametrize("T,N", SHAPES)
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 128])
def test_an_infinity_in_b_comes_back_as_one(T, N, R):
    """In rows of B that hold one, with a finite A, x and scale: the infinity of the sign of its product, and no other column or
    token is touched.  Every other token's h is a power of two, of which two bf16 numbers have nothing left for the second."""
    ids = [t // 5 % 4 for t in range(T)]
    c = x, ids, y, a, b, scale = case(T, R, 64, N, 4, R + T, ids)
    x[::2] = 0.0
    x[::2, 3] = torch.tensor([0.5, -2.0, 1.0, -0.25]).repeat(T)[:len(x[::2])].to(BF)
    a[:, :, 3] = torch.where(torch.arange(R) % 3 == 0, -1.0, 0.5).to(BF)
    scale[:] = torch.tensor([1.0, 2.0, 0.5, 0.25])
    clean = add(c)
    assert bool(clean.isfinite().all())
    g = torch.Generator().manual_seed(R)
    for i in range(4):
        cols = torch.randperm(N, generator=g)[:N // 9]
        b[i, cols, torch.randint(0, R, (len(cols),), generator=g)] = torch.tensor([math.inf, -math.inf])[
            torch.randint(0, 2, (len(cols),), generator=g)].to(BF)
    got = add(c)
    want = reference(*c)[0].to(BF)
    odd = ~want.isfinite()
    assert bool(odd.any()) and not bool(want.isnan().any())
    assert torch.equal(got[odd], want[odd]) and torch.equal(got[~odd], clean[~odd])


@pytest.mark.parametrize("R", [16, 32, 128])
def test_an_infinity_in_b_beside_small_and_infinite_h(R):
    x = torch.zeros(6, 64, dtype=BF)
    x[:, 0] = torch.tensor([2.0 ** -60, -(2.0 ** -60), 2.0 ** -100, 1.0, -math.inf, math.inf]).to(BF)
    a = torch.zeros(1, R, 64, dtype=BF)
    a[:, :, 0] = torch.tensor([1.0, 1.0 + 2.0 ** -7, -1.0, -1.0 - 2.0 ** -7]).repeat(R)[:R].to(BF)
    b = torch.zeros(1, 32, R, dtype=BF) + 0.5
    b[0, 0, 0], b[0, 1, 1], b[0, 2, 2], b[0, 3, 3], b[0, 4, 5] = (math.inf,) * 4 + (-math.inf,)
    y = torch.ones(6, 32, dtype=BF)
    got = add((x, torch.zeros(6, dtype=INT), y, a, b, torch.ones(1)))
    for t, s in ((0, 1), (1, -1), (2, 1), (3, 1)):
        assert got[t, :5].tolist() == [s * math.inf] * 2 + [-s * math.inf] * 2 + [-s * math.inf], t
        assert bool(got[t, 5:].isfinite().all())
    b[:, 5:] = torch.where(a[0, :, 0] > 0, 0.5, -0.5).to(BF)     # every product of one sign
    got = add((x, torch.zeros(6, dtype=INT), y, a, b, torch.ones(1)))
    assert bool((got[4, 5:] == -math.inf).all()) and bool((got[5, 5:] == math.inf).all())


@pytest.mark.parametrize("T,N", [(3, 40), (300, 16392)])
@pytest.mark.parametrize("R", [16, 64])
def test_h_above_the_largest_bf16_number(T, N, R):
    """2^128 - 2^118 is finite in fp32 and rounds to infinity in bf16; the output is 2^28 of it."""
    x = torch.ones(T, 64, dtype=BF)
    a = torch.zeros(2, R, 64, dtype=BF)
    a[0, 0, :10] = (2.0 ** torch.arange(118, 128).double()).to(BF)      # their sum: 2^128 - 2^118
    a[1, 0, :10] = -a[0, 0, :10]
    b = torch.full((2, N, R), 2.0 ** -100, dtype=BF)
    ids = torch.arange(T, dtype=INT) % 2
    got = add((x, ids, torch.zeros(T, N, dtype=BF), a, b, torch.ones(2)))
    assert bool((got[::2] == 2.0 ** 28).all()) and bool((got[1::2] == -(2.0 ** 28)).all())
