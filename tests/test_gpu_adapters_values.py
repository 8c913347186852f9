"""Adapters of many requests: outputs that have to be finite numbers."""
import pytest
import torch

from qwen35_amd import adapters

from test_gpu_adapters import DEV, case, pool, reference

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
