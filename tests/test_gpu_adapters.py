"""Adapters of many requests on the GPU, each token against the same in 64 bits."""
import math

import pytest
import torch

from qwen35_amd import abi, adapters, ops

from _util import bf, gen, quant, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, INT = torch.bfloat16, torch.int32
HALF_BF16 = 2.0 ** -8      # torch.finfo(bfloat16).eps / 2


def reference(x, ids, y, a, b, scale):
    """(out, what its error may be) [T, N] in 64 bits.

    The error, per output: A x is a sum of K exact products in fp32.  A matrix instruction adds 32 of them to a
    running sum, and each partial sum passes through at most K / 32 such steps and 32 roundings within one, none
    of which is above 2^-24 of the sum of magnitudes: (K / 32 + 32) 2^-24 sum |x A|, and two more for joining
    slices and waves (below 16 sums).  h, scaled (one rounding), loses 2^-16 as two bf16 numbers; the second
    product adds R terms, high and low, below 2 R + 32 roundings; y is added (one), and the result rounded."""
    x, y, a, b, scale = (t.double() for t in (x, y, a, b, scale))
    out, err = y.clone(), torch.zeros_like(y)
    K, R, n = x.shape[1], a.shape[1], len(a)
    for t, i in enumerate(ids.tolist()):
        if not 0 <= i < n:
            continue
        h = a[i] @ x[t]
        dh = (K / 32 + 32 + 16) * 2.0 ** -24 * (a[i].abs() @ x[t].abs()) * scale[i].abs()
        h = h * scale[i]
        dh = dh + (2.0 ** -23 + 2.0 ** -16) * h.abs()
        out[t] += b[i] @ h
        size = b[i].abs() @ h.abs()
        e = b[i].abs() @ dh + (2 * R + 32) * 2.0 ** -24 * size + 2.0 ** -24 * (y[t].abs() + size)
        err[t] = e + HALF_BF16 * (out[t].abs() + e) + 1e-38
    return out, err


def case(T, R, K, N, n, seed, ids=None, gain=1.0):
    g = gen(seed)
    x, y = bf(randn(g, T, K)), bf(randn(g, T, N))
    a, b = bf(randn(g, n, R, K, std=gain / math.sqrt(K))), bf(randn(g, n, N, R, std=0.5))
    scale = torch.rand(n, generator=g) * 2 + 0.25
    if ids is None:
        ids = torch.randint(-1, n, (T,), generator=g)
    return x, torch.as_tensor(ids, dtype=INT), y, a, b, scale


def pool(a, b, scale):
    return adapters.Adapters(a.to(DEV), b.to(DEV), scale.to(DEV))


def check(c, what=""):
    x, ids, y, a, b, scale = c
    p, T = pool(a, b, scale), len(x)
    ws = adapters.adapters_workspace(T, a.shape[1], device=DEV)
    ws.fill_(0xFF)              # NaN: nothing of it is read before it is written
    xd, idd, yd = x.to(DEV), ids.to(DEV), y.to(DEV)
    out = p.add(xd, idd, yd, ws)
    assert torch.equal(yd.cpu(), y)
    want, err = reference(*c)
    off = (out.cpu().double() - want).abs()
    bad = off > err
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} off, {float((off / err.clamp(min=1e-30)).max()):.2f} of the bound"
    none = (ids < 0) | (ids >= len(a))
    assert torch.equal(out.cpu()[none].view(torch.int16), y[none].view(torch.int16)), f"{what}: rows without an adapter"
    return out


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 255, 256, 257, 300, 701])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 128])
def test_tokens_and_ranks(T, R):
    check(case(T, R, 256 + 8 * (T % 5), 136 + 8 * (R % 7), 5, 100 * T + R), f"T={T} R={R}")


@pytest.mark.parametrize("K,N", [(8, 8), (64, 8), (72, 32), (512, 40), (520, 1000), (1000, 264), (2560, 9216), (9216, 2560),
                                 (2560, 12352), (4096, 2560)])
@pytest.mark.parametrize("T,R", [(3, 16), (40, 64), (300, 32)])
def test_sizes(K, N, T, R):
    check(case(T, R, K, N, 4, K + N + T), f"K={K} N={N}")


@pytest.mark.parametrize("R", [8, 16, 24, 32, 56, 64, 72, 128])
@pytest.mark.parametrize("T,N", [(256, 20488), (257, 15872), (257, 16392), (320, 16384), (701, 7176), (1290, 3592)])
def test_wide_outputs(T, N, R):
    """Pieces of 64 tokens and 512 columns, the last of each ragged, and calls that just do not have enough of them."""
    g = gen(T + N + R)
    ids = torch.randint(-1, 5, (9,), generator=g).repeat_interleave(-(-T // 9))[:T]
    check(case(T, R, 72, N, 5, T + N + R, ids), f"T={T} N={N} R={R}")


@pytest.mark.parametrize("R", [16, 32, 64, 128])
def test_wide_outputs_of_an_adapter_a_token(R):
    check(case(300, R, 64, 16392, 300, R, list(range(300))[::-1]), f"R={R}")


@pytest.mark.parametrize("R", [16, 32, 64, 128])
def test_wide_outputs_in_place_beside_a_broken_adapter(R):
    T, N = 300, 16392
    x, ids, y, a, b, scale = case(T, R, 64, N, 5, R, [t // 7 % 6 - 1 for t in range(T)])
    want = check((x, ids, y, a, b, scale))
    bad = (ids == 2).to(DEV)
    a, b = a.clone(), b.clone()
    a[2], b[2] = math.nan, math.inf
    wide = torch.full((T, N + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, 8:8 + N]
    out.copy_(y)
    pool(a, b, scale).add(x.to(DEV), ids.to(DEV), out, adapters.adapters_workspace(T, R, device=DEV), out=out)
    assert torch.equal(out[~bad], want[~bad]) and bool(out[bad].isnan().all())
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + N:] == 7).all())


@pytest.mark.parametrize("T,runs", [(5000, 3), (9001, 40)])
def test_long_prompts(T, runs):
    g = gen(T)
    ids = torch.randint(-1, 6, (runs,), generator=g).repeat_interleave(-(-T // runs))[:T]
    check(case(T, 16, 264, 136, 6, T, ids), f"T={T}")


@pytest.mark.parametrize("T", [16, 48, 64, 300])
@pytest.mark.parametrize("kind", ["all one", "all different", "in turn", "none", "last"])
def test_who_shares_an_adapter(T, kind):
    n = max(T, 4)
    ids = {"all one": [2] * T, "all different": list(range(T))[::-1], "in turn": [t % 3 for t in range(T)], "none": [-1] * T,
           "last": [-1] * (T - 1) + [n - 1]}[kind]
    check(case(T, 16, 264, 136, n, T, ids), kind)


def test_ids_outside_the_pool_are_none():
    ids = [0, 3, 4, -1, -2**31, 2**31 - 1, 1000, 2]
    check(case(8, 16, 128, 64, 4, 7, ids))


@pytest.mark.parametrize("T", [24, 300])
@pytest.mark.parametrize("R", [16, 32, 64])
def test_a_broken_adapter_stays_with_its_request(T, R):
    """NaN and infinities in one adapter, its scale, and in one request's x: everybody else's rows are what they
    are without them."""
    x, ids, y, a, b, scale = case(T, R, 264, 136, 5, 3 * T + R, [t * 7 % 5 - (t % 11 == 0) for t in range(T)])
    clean = check((x, ids, y, a, b, scale))
    bad = ids == 2
    broken = [t.clone() for t in (x, y, a, b, scale)]
    broken[0][bad] = math.inf
    broken[2][2, ::3] = math.nan
    broken[3][2] = math.inf
    broken[4][2] = math.nan
    p = pool(*broken[2:])
    out = p.add(broken[0].to(DEV), ids.to(DEV), broken[1].to(DEV), adapters.adapters_workspace(T, R, device=DEV))
    assert torch.equal(out[~bad.to(DEV)], clean[~bad.to(DEV)])
    assert bool(out[bad.to(DEV)].isnan().all())


def test_an_infinity_in_x_comes_back_as_one():
    x, ids, y, a, b, scale = case(3, 16, 64, 32, 1, 5, [0, 0, 0])
    a[:] = a.abs() + 0.125
    b[:] = -(b.abs() + 0.125)
    x[1, 5] = math.inf
    out = pool(a, b, scale).add(x.to(DEV), ids.to(DEV), y.to(DEV), adapters.adapters_workspace(3, 16, device=DEV)).cpu()
    assert bool((out[1] == -math.inf).all()) and bool(out[::2].isfinite().all())


@pytest.mark.parametrize("T", [5, 70, 300])
def test_strided_and_in_place(T):
    """Columns of wider tensors, in place and not; what lies beside them keeps its values."""
    x, ids, y, a, b, scale = case(T, 32, 128, 72, 5, T)
    want = check((x, ids, y, a, b, scale))
    p, ws = pool(a, b, scale), adapters.adapters_workspace(T + 100, 32, device=DEV)
    wide = torch.full((T, 200), 3.0, dtype=BF, device=DEV)
    wide[:, 16:16 + 72] = y.to(DEV)
    xw = torch.full((T, 304), math.nan, dtype=BF, device=DEV)
    xw[:, 40:40 + 128] = x.to(DEV)
    view = wide[:, 16:16 + 72]
    out = torch.full((T + 1, 88), 5.0, dtype=BF, device=DEV)
    p.add(xw[:, 40:168], ids.to(DEV), view, ws, out=out[:T, 8:80])
    assert torch.equal(out[:T, 8:80], want) and bool((out[:, :8] == 5).all()) and bool((out[:, 80:] == 5).all())
    assert bool((out[T] == 5).all())
    got = p.add(xw[:, 40:168], ids.to(DEV), view, ws, out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
    assert bool((wide[:, :16] == 3).all()) and bool((wide[:, 88:] == 3).all())
    same = x[:1].expand(T, 128).to(DEV)             # one row of x for every token (and a stride of 0)
    got = p.add(x[:1].to(DEV).expand(T, 128), ids.to(DEV), y.to(DEV), ws)
    assert torch.equal(got, p.add(same.contiguous(), ids.to(DEV), y.to(DEV), ws))


@pytest.mark.parametrize("T", [3, 520])
def test_offsets_past_32_bits(T):
    """Tokens so far apart that the last ones lie behind element 2^31 of x, y and out."""
    c = case(T, 16, 128, 9216 if T > 3 else 72, 3, T)
    want = check(c)
    x, ids, y, a, b, scale = c
    stride = 2**32 // T // 8 * 8

    def apart(t):
        far = torch.empty((T - 1) * stride + t.shape[1], dtype=BF, device=DEV).as_strided(t.shape, (stride, 1))
        return far.copy_(t.to(DEV))
    out = apart(torch.zeros_like(y))
    pool(a, b, scale).add(apart(x), ids.to(DEV), apart(y), adapters.adapters_workspace(T, 16, device=DEV), out=out)
    assert torch.equal(out, want)


def test_adapters_past_32_bits():
    """A pool of more than 2^31 elements, of which the last adapters are named."""
    n, R, K, N = 8200, 128, 2056, 8
    g = gen(2)
    a = torch.zeros(n, R, K, dtype=BF, device=DEV)
    b = torch.zeros(n, N, R, dtype=BF, device=DEV)
    last = [n - 1, n - 2, 0]
    x, _, y, la, lb, scale = case(3, R, K, N, 3, 5)
    a[last], b[last] = la.to(DEV), lb.to(DEV)
    out = adapters.Adapters(a, b, scale[:1].expand(n).contiguous().to(DEV)).add(
        x.to(DEV), torch.tensor(last, dtype=INT, device=DEV), y.to(DEV), adapters.adapters_workspace(3, R, device=DEV))
    want, err = reference(x, torch.arange(3), y, la, lb, scale[:1].expand(3))
    assert bool(((out.cpu().double() - want).abs() <= err).all())
    del g


def test_repeats_are_equal_and_streams_apart():
    """The same call again, two calls at once on two streams with workspaces of their own, and a captured one
    replayed with other ids between eager calls: all give the same bits."""
    c = case(130, 64, 1000, 520, 9, 11)
    x, ids, y, a, b, scale = (t.to(DEV) for t in c)
    p = adapters.Adapters(a, b, scale)
    want = check(c)
    other = (ids + 1).remainder(9).to(INT)
    ws = [adapters.adapters_workspace(130, 64, device=DEV) for _ in range(3)]
    want_other = p.add(x, other, y, ws[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(y) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, w, o, i in zip(streams, ws, outs, (ids, other)):
            with torch.cuda.stream(s):
                p.add(x, i, y, w, out=o)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want_other)
    live, out = ids.clone(), torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.add(x, live, y, ws[2], out=out)
    for i in range(4):
        live.copy_(other if i % 2 else ids)
        graph.replay()
        eager = p.add(x, other, y, ws[0])
        torch.cuda.synchronize()
        assert torch.equal(out, want_other if i % 2 else want) and torch.equal(eager, want_other)


@pytest.mark.parametrize("M", [1, 20])
def test_beside_a_shared_projection(M):
    """fp8_linear's output with adapters added: what both give together."""
    g = gen(M)
    q, s = quant(g, 384, 256)
    x, ids, _, a, b, scale = case(M, 16, 256, 384, 4, M, [t % 4 for t in range(M)])
    y = ops.fp8_linear(x.to(DEV), q.view(torch.uint8).to(DEV), s.float().to(DEV))
    out = pool(a, b, scale).add(x.to(DEV), ids.to(DEV), y, adapters.adapters_workspace(M, 16, device=DEV))
    want, err = reference(x, ids, y.cpu(), a, b, scale)
    assert bool(((out.cpu().double() - want).abs() <= err).all())


def test_refusals_name_the_argument():
    x, ids, y, a, b, scale = (t.to(DEV) for t in case(4, 16, 64, 32, 2, 1))
    p, ws = adapters.Adapters(a, b, scale), adapters.adapters_workspace(4, 16, device=DEV)
    for bad, error in ((dict(x=x.float()), "x"), (dict(x=x[:, :32]), "x"), (dict(ids=ids.long()), "ids"), (dict(y=y[:3]), "y"),
                       (dict(y=y.cpu()), "y"), (dict(out=torch.empty(4, 64, dtype=BF, device=DEV)[:, ::2]), "out"),
                       (dict(ws=ws.view(torch.float32)), "ws")):
        with pytest.raises((ValueError, TypeError), match=error):
            p.add(**dict(dict(x=x, ids=ids, y=y, ws=ws), **bad))
    with pytest.raises(abi.QhError, match="workspace"):
        p.add(x, ids, y, ws[:256])
    with pytest.raises(ValueError, match="b"):
        adapters.Adapters(a, b[:1].contiguous(), scale)
    assert p.add(x[:0], ids[:0], y[:0], ws).shape == (0, 32)
