"""Sampling by row on the GPU against the definition in 64 bits (_sample_ref.py).

The kernels' weights are 2^-36 off, their sums 2^-35 at most: a decision whose distance to its border is above
2^-33 of the weight that it is taken in has to be the same.  Cases are chosen so that all are, which the oracle
asserts; where equal logits put a decision on its border exactly, the weights are equal in the kernels too and
their sums exact, so that it has to be the same there as well."""
import math
import random

import pytest
import torch

import _sample_ref as ref
from qwen35_amd import abi, sampling

from _util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32, INT = torch.bfloat16, torch.float32, torch.int32
OFF = 2.0 ** -33
SETTINGS = [dict(), dict(heat=0.7, k=20, p=0.8), dict(heat=0.0), dict(heat=0.6, p=0.95), dict(k=50), dict(heat=1.3, m=0.05),
            dict(heat=0.9, k=400, p=0.97, m=0.02), dict(k=1), dict(heat=2.0, p=0.9), dict(k=3, m=0.5), dict(heat=5.0, p=0.5, m=0.001),
            dict(p=0.001), dict(m=1.0), dict(k=10**9, p=2.0, m=-1.0), dict(heat=0.1, p=0.999), dict(k=7, p=0.3)]


def cols(settings):
    """The four tensors of the rows' settings."""
    get = lambda name, off, t: torch.tensor([s.get(name, off) for s in settings], dtype=t, device=DEV)   # noqa: E731
    return dict(temperature=get("heat", 1.0, F32), top_k=get("k", 0, INT), top_p=get("p", 1.0, F32), min_p=get("m", 0.0, F32))


def run(x, u, settings, ws=None, **kw):
    """(tokens, logprobs) of rows x (CPU, or a GPU view) with a list of settings."""
    x = x.to(DEV) if x.device.type == "cpu" else x
    B, V = x.shape
    if ws is None:
        ws = sampling.sample_workspace(B, V, device=DEV).fill_(0xFF)     # nothing of it is read before it is written
    lp = torch.full((B,), 7.0, device=DEV)
    tok = sampling.sample(x, torch.tensor(u, dtype=F32, device=DEV), ws, logprob=lp, **(cols(settings) if settings else {}), **kw)
    return tok.tolist(), lp.tolist()


def check(x, u, settings, exact=False, ws=None, leave=0):
    """Rows against the definition; exact: decisions may lie on their borders; leave: how many rows may be left out
    because one does."""
    got, lp = run(x, u, settings, ws)
    left = 0
    for b in range(len(x)):
        s = settings[b] if settings else {}
        tok, logp, margin = ref.row(x[b].cpu(), u[b], **s)
        if not exact and margin <= OFF and left < leave:
            left += 1
            continue
        assert exact or margin > OFF, f"row {b}: the case itself is on a border ({margin:.2e}, {s})"
        assert got[b] == tok, f"row {b}: {got[b]}, not {tok} ({s}, u={u[b]}, margin {margin:.2e})"
        # one rounding to fp32, the weights' and sums' 2^-34 before the logarithm
        assert lp[b] == logp or abs(lp[b] - logp) <= 2.0 ** -24 * abs(logp) + 2.0 ** -33, f"row {b}: logprob {lp[b]}, {logp}"
    return got


def logits(g, B, V, dtype, spread=2.5, peaks=12):
    x = torch.randn(B, V, generator=g) * spread
    if peaks and V > 4:
        at = torch.randint(0, V, (B, peaks), generator=g)
        x.scatter_(1, at, 4 + 8 * torch.rand(B, peaks, generator=g))
    return x.to(dtype)


def draws(rng, n):
    return [float(torch.tensor(rng.random(), dtype=F32)) for _ in range(n)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [1, 2, 5, 7, 8, 9, 63, 100, 1000, 8191, 8192, 8193, 16384, 50257, 100001])
def test_vocabularies(V, dtype):
    g, rng = gen(V), random.Random(V)
    B = len(SETTINGS)
    check(logits(g, B, V, dtype), draws(rng, B), SETTINGS)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["broad", "peaked", "narrow", "flat tail", "wide", "tiny", "shifted", "huge"])
def test_shapes_of_distributions(kind, dtype):
    """Logits whose cuts fall into bins of one logit and of most of them (a list longer than its place)."""
    V, B = 70000, len(SETTINGS)
    g, rng = gen(31), random.Random(kind)
    x = {"broad": lambda: logits(g, B, V, F32, 4.0, 0), "peaked": lambda: logits(g, B, V, F32, 1.0, 3) * 2,
         "narrow": lambda: logits(g, B, V, F32, 0.03, 0), "flat tail": lambda: logits(g, B, V, F32, 0.01, 5),
         "wide": lambda: logits(g, B, V, F32, 60.0, 0), "tiny": lambda: logits(g, B, V, F32, 1e-20, 0),
         "shifted": lambda: logits(g, B, V, F32, 2.0, 5) - 900, "huge": lambda: logits(g, B, V, F32, 1e36, 0)}[kind]().to(dtype)
    check(x, draws(rng, B), SETTINGS, leave=4)


def test_full_vocabulary_batch():
    """The vocabulary of the model that the framework serves, a batch of users."""
    g, rng = gen(5), random.Random(5)
    n = 24
    s = [rng.choice(SETTINGS) for _ in range(n)]
    x = logits(g, n, 248320, BF)
    check(x, draws(rng, n), s)
    check(x[:1], [0.37], [s[0]])


@pytest.mark.parametrize("n", [2, 3, 64, 1000, 8192, 20000, 65536, 248320])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_equal_logits(n, dtype):
    """All alike: sums are whole multiples of one weight, and draws and cuts on a border fall as they are defined."""
    x = torch.full((1, n), -3.25, dtype=dtype)
    u, s = [], []
    for p in (1.0, 0.5, 0.25, 0.75, 0.3):
        for at in (0.0, 0.5, 0.25, 0.125, 1 - 2.0 ** -24, 0.7):
            u.append(at)
            s.append(dict(p=p))
    for k in (1, 2, n // 2, n - 1, n, 777):
        u += [0.5, 0.9]
        s += [dict(k=k), dict(k=k, p=0.5)]
    u += [0.5, 0.5, 0.5]
    s += [dict(m=1.0), dict(m=0.5), dict(heat=0)]
    check(x.expand(len(u), n), u, s, exact=True)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_at_the_cut(dtype):
    """Few distinct values: of the equal ones at a cut the first indexes are kept."""
    g, rng = gen(9), random.Random(9)
    x = torch.randint(-3, 4, (40, 30011), generator=g).to(dtype)
    s = [dict(k=rng.choice([5, 4000, 4300, 12345]), p=rng.choice([1.0, 0.9, 0.5])) if i % 2 else dict(p=rng.choice([0.1, 0.6, 0.95]))
         for i in range(40)]
    check(x, draws(rng, 40), s, exact=True)      # half of 4000 equal ones, for instance


def test_zeros_of_both_signs_are_equal():
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0]])
    assert run(x.expand(4, 4), [0.0] * 4, [dict(heat=0), dict(k=1), dict(k=2), dict(p=0.1)])[0] == [0, 0, 0, 0]
    assert run(x.expand(2, 4), [0.9, 0.4], [dict(k=2), dict(k=2)])[0] == [1, 0]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("low", ["-inf", "lowest", "nan"])
def test_masked_logits(dtype, low):
    """Most logits masked, all but one, and all of them."""
    fill = {"-inf": -math.inf, "lowest": torch.finfo(dtype).min, "nan": math.nan}[low]
    g, rng = gen(3), random.Random(3)
    V, B = 20000, len(SETTINGS)
    x = logits(g, 3 * B, V, dtype)
    x[torch.rand(3 * B, V, generator=g) < 0.99] = fill
    x[B:2 * B] = fill
    x[B:2 * B, 9000] = -50.0
    x[2 * B:] = fill
    got = check(x, draws(rng, 3 * B), SETTINGS * 3, exact=low == "lowest")
    assert got[B:2 * B] == [9000] * B
    if low != "lowest":
        assert got[2 * B:] == [-1] * B
    else:       # nothing but the lowest value: equal logits
        assert all(t >= 0 for t in got[2 * B:])


def test_masked_logits_hold_nothing_back():
    """NaN and -infinity around a row's logits change neither its token nor its log-probability."""
    g = gen(8)
    x = logits(g, 1, 5000, BF)
    wide = torch.full((1, 30000), math.nan, dtype=BF)
    wide[:, 10000:20000] = -math.inf
    wide[:, 20001:25001] = x
    for s in SETTINGS:
        t, lp = run(x, [0.61], [s])
        tw, lpw = run(wide, [0.61], [s])
        assert tw == [t[0] + 20001] and lpw == lp


@pytest.mark.parametrize("dtype", [BF, F32])
def test_every_nan_is_masked(dtype):
    """NaN of either sign and any payload, quiet and signaling."""
    x = logits(gen(18), 16, 9000, dtype)
    u, s = draws(random.Random(18), 16), SETTINGS
    inner = x[:, 1000:].contiguous()
    codes = torch.arange(0x7F81, 0x7F81 + 127).repeat(8)[:1000] | torch.where(torch.arange(1000) % 3 == 0, 0x8000, 0)
    if dtype == BF:
        x.view(torch.int16)[:, :1000] = codes.to(torch.int32).to(torch.int16)
    else:
        x.view(torch.int32)[:, :1000] = ((codes << 16) - torch.where(codes >= 0x8000, 1 << 32, 0) + torch.arange(1000)).to(torch.int32)
    assert bool(x[:, :1000].isnan().all())
    t, lp = run(x, u, s)
    tw, lpw = run(inner, u, s)
    assert t == [v + 1000 for v in tw] and lp == lpw


def test_infinite_logits():
    """+infinity takes all the weight, shared by those that have it."""
    x = torch.randn(6, 9000, generator=gen(1))
    x[:, [17, 4000, 8500]] = math.inf
    u = [0.1, 0.5, 0.9, 0.5, 0.99, 0.5]
    got, lp = run(x, u, [dict(), dict(), dict(), dict(k=2), dict(p=0.5), dict(heat=0, m=0.5)])
    assert got == [17, 4000, 8500, 4000, 4000, 17]
    assert lp == pytest.approx([-math.log(3)] * 6)


@pytest.mark.parametrize("heat,like", [(1e-30, 0.0), (1e-45, 0.0), (-1.0, 0.0), (math.nan, 0.0), (-math.inf, 0.0)])
def test_cold(heat, like):
    x = logits(gen(2), 3, 9001, F32, peaks=0)
    assert run(x, [0.3, 0.6, 0.9], [dict(heat=heat)] * 3)[0] == run(x, [0.3, 0.6, 0.9], [dict(heat=like)] * 3)[0] == \
        x.argmax(-1).tolist()


@pytest.mark.parametrize("heat", [1e30, math.inf])
def test_hot(heat):
    """Every weight is 1, masked logits apart: 8192.5 of 16384, 4096.25 of 8192."""
    x = logits(gen(2), 2, 1 << 14, F32)
    x[1, ::2] = -math.inf
    assert run(x, [8192.5 / 2**14] * 2, [dict(heat=heat)] * 2)[0] == [1 << 13, (1 << 13) + 1]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_random_numbers_at_the_ends(dtype):
    x = logits(gen(4), 1, 20000, dtype, 1.0, 0)
    x[0, :5] = x[0, -3:] = -math.inf
    u = [0.0, -1.0, math.nan, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 5.0, math.inf]
    for s in (dict(), dict(p=0.9), dict(k=100), dict(m=0.01)):
        got = run(x.expand(8, -1), u, [s] * 8)[0]
        want = [ref.row(x[0], v, **s)[0] for v in u]
        assert got == want, s


def test_settings_that_are_no_numbers_keep_the_first():
    x = logits(gen(6), 1, 9000, BF)
    first = int(x[0].float().argmax())
    s = [dict(p=math.nan), dict(m=math.nan), dict(p=0.0), dict(p=-1.0), dict(m=1.5), dict(p=-math.inf), dict(m=math.inf)]
    assert run(x.expand(7, -1), [0.99] * 7, s)[0] == [first] * 7
    s = [dict(k=-5), dict(p=math.inf), dict(m=-math.inf), dict(k=-2**31), dict(k=2**31 - 1)]
    assert run(x.expand(5, -1), [0.8] * 5, s)[0] == [ref.row(x[0], 0.8)[0]] * 5


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("s", [dict(), dict(heat=0.8, p=0.9), dict(k=30), dict(m=0.02)])
def test_every_token_gets_its_share(dtype, s):
    """4096 random numbers one step apart: each token is drawn as often as its kept weight says, within one."""
    x = logits(gen(12), 1, 9000, dtype, 2.0, 6)
    n = 4096
    got = torch.tensor(run(x.expand(n, -1), [(i + 0.5) / n for i in range(n)], [s] * n)[0])
    w = (x[0].double() / s.get("heat", 1.0)).softmax(0)
    order = w.argsort(descending=True, stable=True)[:s.get("k") or None]
    c = w[order].cumsum(0)
    order = order[(c - w[order] < s.get("p", 2.0) * c[-1]) & (w[order] >= s.get("m", 0.0) * w.max())]
    share = torch.zeros_like(w)
    share[order] = w[order] / w[order].sum()
    assert bool(((torch.bincount(got, minlength=9000) - n * share).abs() <= 1.0 + 1e-9 * n).all())
    assert bool((got.diff() >= 0).all())        # in index order


def test_without_settings_and_with_some():
    g, rng = gen(14), random.Random(14)
    x, u = logits(g, 9, 12345, BF), draws(rng, 9)
    check(x, u, None)
    ws = sampling.sample_workspace(9, 12345, device=DEV)
    xd, ud = x.to(DEV), torch.tensor(u, device=DEV)
    heat = torch.full((9,), 0.7, device=DEV)
    want = [ref.row(x[b], u[b], heat=0.7)[0] for b in range(9)]
    out = torch.zeros(9, dtype=torch.int64, device=DEV)
    assert sampling.sample(xd, ud, ws, temperature=heat, out=out) is out and out.tolist() == want
    want = [ref.row(x[b], u[b], k=9)[0] for b in range(9)]
    assert sampling.sample(xd, ud, ws, top_k=torch.full((9,), 9, dtype=INT, device=DEV)).tolist() == want
    want = [ref.row(x[b], u[b], m=0.1)[0] for b in range(9)]
    assert sampling.sample(xd, ud, ws, min_p=torch.full((9,), 0.1, device=DEV)).tolist() == want


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_any_alignment_and_stride(dtype):
    g, rng = gen(15), random.Random(15)
    B, V = len(SETTINGS), 9999
    x, u = logits(g, B, V, dtype), draws(rng, B)
    want = check(x, u, SETTINGS)
    for off, width in ((1, V + 1), (3, V + 5), (8, V + 100)):
        wide = torch.full((B, width + off), math.inf, dtype=dtype, device=DEV)   # +infinity beside a row would take it over
        wide[:, off:off + V] = x.to(DEV)
        assert run(wide[:, off:off + V], u, SETTINGS)[0] == want
    flipped = x.flip(0).to(DEV)
    assert run(flipped, u[::-1], SETTINGS[::-1])[0] == want[::-1]


def test_one_workspace_for_calls_of_many_sizes():
    """A workspace serves smaller calls, in any order; what an earlier call left in it does not matter."""
    g, rng = gen(16), random.Random(16)
    ws = sampling.sample_workspace(40, 60000, device=DEV)
    for B, V in ((3, 60000), (40, 100), (40, 60000), (1, 9000), (17, 33333), (40, 60000)):
        s = [rng.choice(SETTINGS) for _ in range(B)]
        check(logits(g, B, V, BF), draws(rng, B), s, ws=ws)


def test_repeats_streams_and_replays():
    """The same call again gives the same tokens, two at once on two streams too, and a captured one replayed with
    other random numbers and settings between eager calls."""
    g, rng = gen(17), random.Random(17)
    B, V = 33, 50257
    s, other = ([rng.choice(SETTINGS) for _ in range(B)] for _ in range(2))
    x, u, v = logits(g, B, V, BF).to(DEV), draws(rng, B), draws(rng, B)
    want, want_lp = run(x, u, s)
    then, then_lp = run(x, v, other)
    ws = [sampling.sample_workspace(B, V, device=DEV) for _ in range(3)]
    dev = [dict(cols(c), u=torch.tensor(w, device=DEV)) for c, w in ((s, u), (other, v))]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros(B, dtype=torch.int64, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(6):
        for st, w, o, d in zip(streams, ws, outs, dev):
            with torch.cuda.stream(st):
                sampling.sample(x, ws=w, out=o, **d)
    torch.cuda.synchronize()
    assert outs[0].tolist() == want and outs[1].tolist() == then
    live = {k: t.clone() for k, t in dev[0].items()}
    out, lp = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.sample(x, ws=ws[2], out=out, logprob=lp, **live)
    for i in range(5):
        for k, t in live.items():
            t.copy_(dev[i % 2][k])
        graph.replay()
        assert sampling.sample(x, ws=ws[0], **dev[1]).tolist() == then
        torch.cuda.synchronize()
        assert out.tolist() == (then if i % 2 else want) and lp.tolist() == (then_lp if i % 2 else want_lp), i


@pytest.mark.parametrize("dtype", [BF, F32])
def test_offsets_past_32_bits(dtype):
    """Rows 2^31 + 24 elements apart."""
    g, rng = gen(21), random.Random(21)
    B, V, stride = 3, 20000, 2**31 + 24
    x, u = logits(g, B, V, dtype), draws(rng, B)
    s = [SETTINGS[3], SETTINGS[0], SETTINGS[1]]
    want = check(x, u, s)
    far = torch.empty((B - 1) * stride + V, dtype=dtype, device=DEV).as_strided((B, V), (stride, 1))
    far.copy_(x.to(DEV))
    assert run(far, u, s)[0] == want


def test_many_rows():
    """As many rows as the grid's axis is long, two logits each."""
    n = 65535
    x = torch.tensor([[0.0, math.log(3.0)]]).expand(n, 2).to(DEV)
    u = torch.arange(n, device=DEV) / n
    ws = sampling.sample_workspace(n, 2, device=DEV)
    got = sampling.sample(x, u.float(), ws, top_p=torch.full((n,), 0.9, device=DEV))
    assert int((got == 0).sum()) == pytest.approx(n / 4, abs=2) and bool((got.diff() >= 0).all())


def test_refusals_name_the_argument():
    x, u = torch.zeros(4, 100, dtype=BF, device=DEV), torch.zeros(4, device=DEV)
    ws = sampling.sample_workspace(4, 100, device=DEV)
    for bad, error in ((dict(logits=x.half()), "logits"), (dict(logits=x.t()), "logits|contiguous"), (dict(u=u[:3]), "u"),
                       (dict(u=u.double()), "u"), (dict(top_k=u), "top_k"), (dict(top_p=u.to(BF)), "top_p"),
                       (dict(min_p=u.cpu()), "min_p"), (dict(temperature=u[:2]), "temperature"), (dict(logprob=u.double()), "logprob"),
                       (dict(out=torch.zeros(4, dtype=INT, device=DEV)), "out"), (dict(ws=ws.float()), "ws")):
        with pytest.raises((ValueError, TypeError), match=error):
            sampling.sample(**dict(dict(logits=x, u=u, ws=ws), **bad))
    with pytest.raises(abi.QhError, match="workspace"):
        sampling.sample(torch.zeros(4, 9000, dtype=BF, device=DEV), u, ws)
    assert sampling.sample(x[:0], u[:0], ws).shape == (0,)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("s", [dict(), dict(m=1e-25), dict(p=0.999), dict(k=5), dict(heat=0.0)])
def test_a_draw_of_nothing_passes_over_far_chunks(dtype, s):
    """u at (or next to) zero: the first logit that has a weight, not one of the logits in front of it whose weights
    (2^-144 of the largest, or 2^-65) are none, though they are weights beside each other."""
    V, at = 20000, 9003
    for far in (-100.0, -45.5):
        x = torch.full((4, V), far, dtype=dtype)
        x[:, at] = 0.0
        x[:, 8192:at] = -200.0
        got, lp = run(x, [0.0, 1e-44, 0.5, 1.0], [s] * 4)
        assert got == [at] * 4, (far, got)
        assert all(abs(v) <= 2.0 ** -33 for v in lp), (far, lp)
