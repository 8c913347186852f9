"""Paged KV cache on the GPU: tokens written (head norm, rotary axes, quantisation), rows read
back, decode attention, and a prompt with its next tokens run through all of them, each against
the same in 64 bits."""
import itertools
import math

import pytest
import torch

import _paged_ref as ref
from oracle import qwen35_oracle as orc
from qwen35_amd import abi, paged

from _util import bf, gen, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
HALF_BF16 = 2.0 ** -8      # torch.finfo(bfloat16).eps / 2
HALF_E4M3 = 2.0 ** -4
# fp32 head norm and rotation: the mean of D squares (64 lanes' chains and their tree, below 16
# roundings), rsqrt (1 ulp), two products, then two products and a sum: below 32 roundings of 2^-24
ARITH = 32 * 2.0 ** -24


def pool(g, n_pages, n_kv, page, D, fp8, std=1.0):
    """(k, v, k_scale, v_scale) on the CPU, filled."""
    out, sc = [], []
    for _ in range(2):
        x = randn(g, n_pages, n_kv, page, D, std=std)
        if fp8:
            s = (x.abs().amax(-1) / 448).clamp(min=ref.MIN_SCALE)
            out.append((x / s[..., None]).to(F8))
            sc.append(s)
        else:
            out.append(bf(x))
            sc.append(None)
    return (*out, *sc)


def on_gpu(parts):
    return paged.PagedKVCache(*(None if t is None else t.to(DEV) for t in parts))


def tables(g, lens, page, extra=2):
    """Page tables [B, most] in random order (-1 behind a sequence's last page) and the number of pages."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    ids = torch.randperm(total, generator=g).to(torch.int32)
    t = torch.full((len(lens), max(1, max(need, default=1))), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = ids[at:at + k]
        at += k
    return t, max(1, total)


# ------------------------------------------------------------------ prep
def check_row(got, scale, y, tol, what):
    """A cached row against y (64 bits, off by at most tol before its rounding)."""
    if scale is None:
        err, lim = (got.double() - y).abs(), HALF_BF16 * (y.abs() + tol) + tol + 1e-38
    else:
        s = scale.double()[..., None]
        want = (y.abs().amax(-1) / 448).clamp(min=ref.MIN_SCALE)
        stol = tol.amax(-1) / 448 + 2.0 ** -23 * want
        assert bool(((scale.double() - want).abs() <= stol).all()), f"{what}: scale"
        # half a step of the code, relative above 2^-6 and 2^-10 below; the quotient's own rounding
        err = (got.double() * s - y).abs()
        lim = HALF_E4M3 * (y.abs() + tol) + 2.0 ** -10 * s + tol + 2.0 ** -22 * y.abs()
    assert bool((err <= lim).all()), f"{what}: {float((err / lim).max()):.3f} of the bound"


@pytest.mark.parametrize("T,H,kv,D,page,fp8,rot,sections,inter,f32,norm", [
    (1, 16, 4, 256, 16, True, 64, (11, 11, 10), True, False, True),
    (1, 16, 4, 256, 16, False, 64, (32,), False, True, True),
    (37, 16, 4, 256, 24, True, 64, (12, 10, 10), False, True, True),
    (64, 32, 8, 128, 32, False, 128, (64,), False, False, True),
    (65, 6, 2, 128, 8, True, 32, (6, 5, 5), True, False, True),
    (5, 4, 1, 256, 40, True, 256, (64, 64), True, False, False),
    (19, 3, 3, 128, 8, False, 48, (8, 8, 8), False, True, True),
    (33, 16, 1, 256, 64, True, 16, (2, 2, 2, 2), True, False, True),
    (9, 10, 2, 256, 16, True, 0, (), False, True, True),
    (130, 12, 12, 128, 256, False, 64, (16, 16), True, False, False),
    (301, 16, 4, 256, 16, True, 64, (11, 11, 10), True, True, True),
    (2050, 5, 5, 128, 24, True, 128, (24, 20, 20), True, False, True),
])
def test_prep(T, H, kv, D, page, fp8, rot, sections, inter, f32, norm):
    g = gen(T * 7 + D + rot)
    S = 1 if T == 1 else 3
    past = [int(x) for x in torch.randint(0, 70, (S,), generator=g)]
    cut = [T] if S == 1 else [T // 2, T // 3, T - T // 2 - T // 3]
    lens = [p + c for p, c in zip(past, cut)]
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    cache = on_gpu(parts)
    max_pos = 4096
    cos, sin = orc.rope_tables(max_pos, max(rot, 16), 1e7)
    pos = torch.randint(0, max_pos, (max(1, len(sections)), T), generator=g).to(torch.int32)
    qg = bf(randn(g, T, H, 2 * D))
    kvp = bf(randn(g, T, 2 * kv + 1, D))               # k and v heads of one fused projection
    k, v = kvp[:, :kv], kvp[:, kv:2 * kv]
    qn = randn(g, D, std=0.3) if norm else None
    kn = randn(g, D, std=0.3) if norm else None
    seq = torch.cat([torch.full((c,), b) for b, c in enumerate(cut)]).to(torch.int32)
    at = torch.cat([torch.arange(p, p + c) for p, c in zip(past, cut)]).to(torch.int32)
    perm = torch.randperm(T, generator=g)              # tokens in any order
    seq, at = seq[perm].contiguous(), at[perm].contiguous()

    cu = lambda t: None if t is None else t.to(DEV)    # noqa: E731
    qd, kvd = cu(qg), cu(kvp)
    q_out = torch.empty(T, H, D, dtype=torch.float32 if f32 else torch.bfloat16, device=DEV)
    rp = paged.RopeAxes(cu(cos), cu(sin), sections, interleaved=inter) if rot else None
    cache.prep(kvd[:, :kv], kvd[:, kv:2 * kv], cu(table), cu(at), seq=cu(seq), q=qd[..., :D], q_out=q_out, rope=rp,
               pos=cu(pos) if rot else None, q_norm=cu(qn), k_norm=cu(kn))
    torch.cuda.synchronize()

    axes = ref.axes_of(rot // 2, list(sections), inter) if rot else []
    qx, kx = ref.head_norm(qg[..., :D], qn), ref.head_norm(k, kn)
    qy, ky = ref.rotate(qx, cos, sin, pos, axes), ref.rotate(kx, cos, sin, pos, axes)
    qt, kt = ARITH * ref.pair_size(qx, rot // 2), ARITH * ref.pair_size(kx, rot // 2)
    err = (q_out.cpu().double() - qy).abs()
    lim = qt + (0 if f32 else HALF_BF16 * (qy.abs() + qt)) + 1e-38
    assert bool((err <= lim).all()), f"q: {float((err / lim).max()):.3f} of the bound"

    page_id, off = table[seq.long(), at.long() // page].long(), at.long() % page
    for got, sc, y, tol, was, name in ((cache.k, cache.k_scale, ky, kt, parts[0], "k"),
                                       (cache.v, cache.v_scale, v.double(), torch.zeros_like(v.double()), parts[1], "v")):
        got = got.cpu()
        rows = got.view(torch.uint8 if fp8 else torch.bfloat16)[page_id, :, off]
        check_row(rows.view(F8) if fp8 else rows, None if sc is None else sc.cpu()[page_id, :, off], y, tol, name)
        # every other row is what it was
        here = torch.zeros(n_pages, page, dtype=torch.bool)
        here[page_id, off] = True
        keep = ~here[:, None, :, None].expand_as(was)
        raw = torch.uint8 if fp8 else torch.int16
        assert torch.equal(got.view(raw)[keep], was.view(raw)[keep]), f"{name}: a row that no token names"


@pytest.mark.parametrize("fp8", [False, True])
def test_prep_without_seq_and_without_q_writes_v_as_it_is(fp8):
    """One token a sequence, no q, no norm, no rotation: bf16 rows are copies."""
    g = gen(5)
    B, kv, D, page = 6, 2, 128, 8
    table, n_pages = tables(g, [20] * B, page)
    cache = on_gpu(pool(g, n_pages, kv, page, D, fp8))
    k, v = bf(randn(g, B, kv, D)), bf(randn(g, B, kv, D))
    at = torch.tensor([0, 7, 8, 15, 16, 19], dtype=torch.int32)
    assert cache.prep(k.to(DEV), v.to(DEV), table.to(DEV), at.to(DEV)) is None
    b = torch.arange(B)
    pid, off = table[b, at.long() // page].long(), at.long() % page
    for got, sc, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        rows = got.cpu().view(torch.uint8 if fp8 else torch.bfloat16)[pid, :, off]
        if fp8:
            check_row(rows.view(F8), sc.cpu()[pid, :, off], x.double(), torch.zeros(B, kv, D, dtype=torch.float64), "row")
        else:
            assert torch.equal(rows, x)


@pytest.mark.parametrize("fp8", [False, True])
def test_prep_leaves_out_what_its_indexes_do_not_name(fp8):
    """Padding and indexes outside their ranges: neither the cache nor q_out is touched."""
    g = gen(6)
    T, H, kv, D, page = 11, 4, 2, 256, 8
    table, n_pages = tables(g, [24, 24], page)
    table[1, 1], table[1, 2] = n_pages, -7
    parts = pool(g, n_pages, kv, page, D, fp8)
    cache = on_gpu(parts)
    cos, sin = orc.rope_tables(32, 64, 1e4)
    seq = torch.tensor([-1, 2, 1 << 30, 0, 0, 0, 1, 1, 0, 0, 1], dtype=torch.int32)
    at = torch.tensor([0, 0, 0, -1, 24, 2**31 - 1, 8, 16, 3, 4, 5], dtype=torch.int32)
    pos = torch.full((3, T), 5, dtype=torch.int32)
    pos[1, 8], pos[2, 9] = 32, -1                      # only the last token is whole
    q_was = randn(g, T, H, D)
    q_out = q_was.to(DEV)
    k, v = bf(randn(g, T, kv, D)), bf(randn(g, T, kv, D))
    cache.prep(k.to(DEV), v.to(DEV), table.to(DEV), at.to(DEV), seq=seq.to(DEV), q=bf(randn(g, T, H, D)).to(DEV),
               q_out=q_out, rope=paged.RopeAxes(cos.to(DEV), sin.to(DEV), (12, 10, 10)), pos=pos.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(q_out.cpu()[:-1], q_was[:-1])
    assert not torch.equal(q_out.cpu()[-1], q_was[-1])
    raw = torch.uint8 if fp8 else torch.int16
    for got, was in ((cache.k, parts[0]), (cache.v, parts[1])):
        diff = (got.cpu().view(raw) != was.view(raw)).any(-1).any(1)     # [pages, page]
        assert diff.nonzero().tolist() == [[int(table[1, 0]), 5]]


def test_prep_e4m3_zeros_tiny_and_values_that_are_not_finite():
    g = gen(7)
    kv, D, page = 1, 128, 8
    x = bf(randn(g, 6, kv, D))
    x[0] = 0
    x[1] = bf(torch.full((kv, D), 1e-37))              # below what the smallest scale resolves: zeros
    x[2, 0, 3], x[2, 0, 9], x[2, 0, 77] = math.nan, math.inf, -math.inf
    x[3] = math.nan
    x[4] = bf(torch.tensor(3.3e38)) * torch.sign(x[4])  # amax near the type's largest
    table, n_pages = tables(g, [8], page)
    cache = on_gpu(pool(g, n_pages, kv, page, D, True))
    seq, at = torch.zeros(6, dtype=torch.int32), torch.arange(6, dtype=torch.int32)
    cache.prep(x.to(DEV), x.to(DEV), table.to(DEV), at.to(DEV), seq=seq.to(DEV))
    pid = int(table[0, 0])
    codes, s = cache.v.cpu()[pid, 0].float()[:6], cache.v_scale.cpu()[pid, 0][:6]
    assert s[0] == ref.MIN_SCALE and s[1] == ref.MIN_SCALE and s[3] == ref.MIN_SCALE
    assert bool((codes[:2] == 0).all()) and bool(torch.isnan(codes[3]).all())
    bad = ~torch.isfinite(x[2, 0].float())
    assert torch.equal(torch.isnan(codes[2]), bad)
    fine = ~bad
    y = x[2, 0].double()[fine]
    assert s[2].double() == pytest.approx(float(y.abs().max()) / 448, rel=2.0 ** -23)
    assert bool(((codes[2][fine].double() * s[2].double() - y).abs() <= HALF_E4M3 * y.abs() + 2.0 ** -10 * s[2] + 1e-30).all())
    y = x[4, 0].double()
    assert bool(((codes[4].double() * s[4].double() - y).abs() <= HALF_E4M3 * y.abs()).all())


def test_prep_e4m3_normalised_rows_that_are_not_finite():
    """Through the head norm: a NaN makes the whole row NaN; an infinity itself, the rest zeros (the
    norm of the row is infinite); a row of zeros stays zeros."""
    g = gen(17)
    kv, D, page = 2, 256, 8
    x = bf(randn(g, 4, kv, D))
    x[0, 0, 5] = math.nan
    x[1, 0, 200] = math.inf
    x[2, 0] = 0
    cache = paged.PagedKVCache.alloc(1, page, kv, D, dtype=F8)
    z = torch.zeros(4, dtype=torch.int32, device=DEV)
    cos, sin = (t.to(DEV) for t in orc.rope_tables(16, 64, 1e4))
    at = torch.arange(4, dtype=torch.int32, device=DEV)
    cache.prep(x.to(DEV), x.to(DEV), z[:1].view(1, 1), at, seq=z, rope=paged.RopeAxes(cos, sin), pos=at,
               k_norm=torch.zeros(D, device=DEV))
    k, s = cache.k.cpu()[0].float(), cache.k_scale.cpu()[0]
    assert bool(torch.isnan(k[0, 0]).all()) and s[0, 0] == ref.MIN_SCALE
    # the infinity's pair (200 is not turned) alone is NaN
    assert torch.isnan(k[0, 1]).nonzero().flatten().tolist() == [200] and s[0, 1] == ref.MIN_SCALE
    assert bool((k[0, 1][~torch.isnan(k[0, 1])] == 0).all())
    assert bool((k[0, 2] == 0).all()) and s[0, 2] == ref.MIN_SCALE
    for t in range(4):                                 # the other head's rows are rows of their own
        y = ref.rotate(ref.head_norm(x[t:t + 1, 1:], torch.zeros(D)), cos.cpu(), sin.cpu(), torch.tensor([[t]]), [0] * 32)
        check_row(cache.k.cpu()[0, 1, t][None, None], s[1, t][None, None], y, ARITH * ref.pair_size(y, 32) * 2, "row")


def test_prep_e4m3_codes_are_those_of_64_bits():
    """K through norm and rotation: no code differs from the exact quotient's but where this lies within
    fp32's own rounding of a border between two codes; V: none."""
    g = gen(18)
    T, kv, D, page, rot = 300, 4, 256, 16, 64
    k, v = bf(randn(g, T, kv, D)), bf(randn(g, T, kv, D))
    kn = randn(g, D, std=0.3)
    cos, sin = orc.rope_tables(512, rot, 1e7)
    n_pages = -(-T // page)
    cache = paged.PagedKVCache.alloc(n_pages, page, kv, D, dtype=F8)
    at = torch.arange(T, dtype=torch.int32, device=DEV)
    cache.prep(k.to(DEV), v.to(DEV), torch.arange(n_pages, dtype=torch.int32, device=DEV).view(1, -1), at,
               seq=torch.zeros_like(at), rope=paged.RopeAxes(cos.to(DEV), sin.to(DEV)), pos=at, k_norm=kn.to(DEV))
    y = ref.rotate(ref.head_norm(k, kn), cos, sin, at.cpu()[None], [0] * (rot // 2))
    for got, x in ((cache.k, y), (cache.v, v.double())):
        z = x * 448 / x.abs().amax(-1, keepdim=True)      # of V's bf16 numbers exact where a tie
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
        want = torch.round(z / step) * step
        codes = got.cpu().view(torch.uint8).view(n_pages, kv, page, D).transpose(1, 2).reshape(-1, kv, D)[:T].view(F8).double()
        border = ((z / step - torch.floor(z / step)) - 0.5).abs() * step <= 2.0 ** -23 * z.abs()
        if x is y:
            assert bool(((codes == want) | border).all())
        else:
            assert torch.equal(codes, want)


def test_prep_e4m3_code_of_every_rounding():
    """Rows whose scale is 1 (an element of 448): every bf16 value up to 448 takes the code that
    torch's own conversion gives."""
    D, page = 128, 8
    vals = torch.arange(0, 0x8000, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    vals = vals[vals.float() <= 448]
    vals = torch.cat([vals, -vals])
    n = -(-vals.numel() // (D - 1))
    x = torch.zeros(n * (D - 1), dtype=torch.bfloat16)
    x[:vals.numel()] = vals
    x = torch.cat([torch.full((n, 1), 448.0, dtype=torch.bfloat16), x.view(n, D - 1)], 1).view(n, 1, D)
    n_pages = -(-n // page)
    cache = paged.PagedKVCache.alloc(n_pages, page, 1, D, dtype=F8)
    table = torch.arange(n_pages, dtype=torch.int32, device=DEV).view(1, -1)
    xd = x.to(DEV)
    cache.prep(xd, xd, table, torch.arange(n, dtype=torch.int32, device=DEV),
               seq=torch.zeros(n, dtype=torch.int32, device=DEV))
    got = cache.k.view(torch.uint8).view(-1, D)[:n].cpu()
    assert bool((cache.k_scale.view(-1)[:n] == 1).all())
    assert torch.equal(got, x[:, 0].float().to(F8).view(torch.uint8))
    assert torch.equal(cache.v.view(torch.uint8).view(-1, D)[:n].cpu(), got)


def test_prep_one_axis_is_the_dense_paths_rotation():
    """With one axis and a page as long as the sequence, q and the bf16 cache agree with qh_attn_prep's
    (which rounds the norm to bf16 in between: one bf16 step of each)."""
    g = gen(8)
    M, H, kv, D, rot, page = 40, 16, 4, 256, 64, 64
    q, k, v = bf(randn(g, M, H, 2 * D)).to(DEV), bf(randn(g, M, kv, D)).to(DEV), bf(randn(g, M, kv, D)).to(DEV)
    qn, kn = (randn(g, D, std=0.1).to(DEV) for _ in range(2))
    cos, sin = (t.to(DEV) for t in orc.rope_tables(page, rot, 1e7))
    lib = abi.load()
    q32 = torch.empty(M, H, D, device=DEV)
    kc, vc = torch.zeros(2, kv, page, D, dtype=torch.bfloat16, device=DEV).unbind(0)
    abi.check(lib.qh_attn_prep(abi.ptr(q), abi.ptr(k), abi.ptr(v), abi.ptr(qn), abi.ptr(kn), abi.ptr(cos), abi.ptr(sin),
                               abi.ptr(q32), abi.ptr(kc), abi.ptr(vc), M, H, kv, D, rot, 0, page, 1e-6,
                               abi.stream_handle()))
    cache = paged.PagedKVCache.alloc(1, page, kv, D)
    at = torch.arange(M, dtype=torch.int32, device=DEV)
    q_out = torch.empty(M, H, D, device=DEV)
    cache.prep(k, v, torch.zeros(1, 1, dtype=torch.int32, device=DEV), at, seq=torch.zeros_like(at), q=q[..., :D],
               q_out=q_out, rope=paged.RopeAxes(cos, sin), pos=at, q_norm=qn, k_norm=kn)
    torch.cuda.synchronize()
    assert torch.equal(cache.v[0, :, :M], vc[:, :M])
    for a, b in ((q_out, q32), (cache.k[0, :, :M].transpose(0, 1).float(), kc[:, :M].transpose(0, 1).float())):
        lim = 2 * HALF_BF16 * ref.pair_size(b.cpu().double(), rot // 2) * 1.5 + 1e-6
        assert bool(((a - b).abs().cpu().double() <= lim).all())


def test_wrapper_refusals():
    cache = paged.PagedKVCache.alloc(4, 16, 2, 128)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)   # noqa: E731
    i32 = torch.int32
    k, pages, at = z(3, 2, 128), z(3, 2, dtype=i32), z(3, dtype=i32)
    rp = paged.RopeAxes(z(8, 32, dtype=torch.float32), z(8, 32, dtype=torch.float32))
    for exc, args, kw in [
        (TypeError, (k.float(), k, pages, at), {}),
        (ValueError, (k[:, :1], k, pages, at), {}),
        (ValueError, (k, z(3, 2, 256)[..., ::2], pages, at), {}),
        (ValueError, (z(3, 4, 128)[:, ::2], k, pages, at), {}),
        (TypeError, (k, k, pages.long(), at), {}),
        (ValueError, (k, k, pages, at[:2]), {}),
        (ValueError, (k, k, pages, z(6, dtype=i32)[::2]), {}),
        (ValueError, (k, k, pages.t(), at), {}),
        (ValueError, (k, k, pages.cpu(), at), {}),
        (ValueError, (k, k, pages, at), dict(rope=rp)),
        (ValueError, (k, k, pages, at), dict(rope=rp, pos=z(2, 3, dtype=i32))),
        (TypeError, (k, k, pages, at), dict(q_norm=z(128))),
        (TypeError, (k, k, pages, at), dict(q=k, q_out=z(3, 2, 128, dtype=torch.float16))),
        (ValueError, (k, k, pages, at), dict(q=k, q_out=z(3, 2, 256)[..., :128])),
        (ValueError, (k, k, pages, at), dict(q_out=z(3, 2, 128))),
        (abi.QhError, (k, k, pages[:2], at), {}),                 # three tokens, two sequences
        (abi.QhError, (k, k, pages, at), dict(q=k, q_out=k)),
    ]:
        with pytest.raises(exc):
            cache.prep(*args, **kw)
    with pytest.raises(abi.QhError, match="aligned"):
        cache.prep(z(3 * 2 * 128 + 4)[4:].view(3, 2, 128), k, pages, at)
    with pytest.raises(ValueError):
        paged.PagedKVCache(z(4, 2, 16, 128, dtype=torch.uint8).view(F8), z(4, 2, 16, 128, dtype=torch.uint8).view(F8))
    with pytest.raises(abi.QhError, match="page_size"):
        paged.PagedKVCache.alloc(4, 12, 2, 128).prep(k, k, pages, at)
    ws = paged.attn_workspace(4, 2, 128)
    q = z(3, 4, 128)
    for exc, args, kw in [
        (ValueError, (q, pages, at[:2], ws), {}),
        (ValueError, (q, pages[:2], at, ws), {}),
        (TypeError, (q, pages, at, ws.view(torch.int32)), {}),
        (abi.QhError, (q, pages, at, ws[:1024]), {}),
        (abi.QhError, (z(3, 5, 128), pages, at, ws), {}),
        (TypeError, (q, pages, at, ws), dict(gate=q.float())),
        (ValueError, (q, pages, at, ws), dict(out=z(3, 2, 128))),
        (abi.QhError, (q, pages, at, ws), dict(out=q)),
    ]:
        with pytest.raises(exc):
            cache.attend(*args, **kw)
    with pytest.raises(ValueError):
        cache.read(pages, at, z(3, 2, 32, 128), z(3, 2, 33, 128))
    with pytest.raises(ValueError):
        cache.read(pages, at, z(3, 3, 32, 128), z(3, 3, 32, 128))


def test_nothing_to_write_read_or_attend_to():
    cache = paged.PagedKVCache.alloc(4, 16, 2, 128)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)   # noqa: E731
    i32 = torch.int32
    out = cache.prep(z(0, 2, 128), z(0, 2, 128), z(2, 3, dtype=i32), z(0, dtype=i32), q=z(0, 4, 128))
    assert out.shape == (0, 4, 128) and out.dtype == torch.bfloat16
    cache.read(z(0, 3, dtype=i32), z(0, dtype=i32), z(0, 2, 8, 128), z(0, 2, 8, 128))
    assert cache.attend(z(0, 4, 128), z(0, 3, dtype=i32), z(0, dtype=i32), paged.attn_workspace(4, 2, 128)).shape == (0, 4, 128)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("lens,kv,D,page,fp8,max_seq", [
    ([1], 4, 256, 16, True, 1),
    ([130], 4, 256, 16, True, 135),
    ([0, 5, 300, 64, 63], 2, 128, 24, False, 301),
    ([77, 0, 8, 9, 2049], 3, 128, 8, True, 2049),
    ([500, 17], 1, 256, 40, False, 100),               # the dense cache ends before the sequence
    ([1000] * 20, 2, 256, 256, True, 1024),
])
def test_read(lens, kv, D, page, fp8, max_seq):
    g = gen(sum(lens) + D)
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8, std=3.0)
    cache = on_gpu(parts)
    last = torch.tensor(lens, dtype=torch.int32) - 1
    was = [bf(randn(g, len(lens), kv, max_seq, D)) for _ in range(2)]
    out = [t.to(DEV) for t in was]
    cache.read(table.to(DEV), last.to(DEV), *out)
    torch.cuda.synchronize()
    for x, sc, o, w in ((parts[0], parts[2], out[0], was[0]), (parts[1], parts[3], out[1], was[1])):
        want = w.clone()
        for b, n in enumerate(lens):
            n = min(n, max_seq)
            if n:
                j = torch.arange(n)
                y = x[table[b].long()[j // page], :, j % page].float()
                if sc is not None:
                    y = y * sc[table[b].long()[j // page], :, j % page][..., None]
                want[b, :, :n] = bf(y).transpose(0, 1)
        assert torch.equal(o.cpu(), want)


def test_read_leaves_out_pages_that_do_not_exist_and_ends_at_the_table():
    g = gen(9)
    kv, D, page = 2, 128, 8
    table = torch.tensor([[1, 99, 2], [-1, 0, 3]], dtype=torch.int32)
    parts = pool(g, 4, kv, page, D, False)
    cache = on_gpu(parts)
    was = bf(randn(g, 2, kv, 40, D))
    ko, vo = was.to(DEV), was.to(DEV)
    cache.read(table.to(DEV), torch.tensor([2**31 - 1, 30], dtype=torch.int32, device=DEV), ko, vo)
    for o, x in ((ko.cpu(), parts[0]), (vo.cpu(), parts[1])):
        want = was.clone()
        for b, i in itertools.product(range(2), range(3)):
            pid = int(table[b, i])
            if 0 <= pid < 4:
                want[b, :, 8 * i:8 * i + 8] = x[pid]
        assert torch.equal(o, want)


# ------------------------------------------------------------------ attention
def check_attend(parts, cache, q, table, last, gate=None, ws=None, what=""):
    H, kv, D = q.shape[1], cache.n_kv, q.shape[2]
    ws = paged.attn_workspace(H, kv, D) if ws is None else ws
    out = cache.attend(q.to(DEV), table.to(DEV), last.to(DEV), ws, gate=None if gate is None else gate.to(DEV))
    torch.cuda.synchronize()
    want, tol = ref.attend(q, *parts, table, last, gate)
    err, lim = (out.cpu().double() - want).abs(), HALF_BF16 * (want.abs() + tol) + tol
    assert bool(torch.isfinite(out).all()), what
    assert bool((err <= lim).all()), f"{what}: {float((err / lim.clamp(min=1e-30)).max()):.3f} of the bound"
    empty = want.abs().amax((1, 2)) == 0
    assert bool((out.cpu()[empty] == 0).all()), what
    return out


@pytest.mark.parametrize("H,kv,D,page,fp8,gated", [
    (16, 4, 256, 16, True, True),
    (16, 4, 256, 16, False, True),
    (4, 1, 256, 8, True, False),
    (64, 8, 128, 32, False, False),
    (64, 8, 128, 32, True, True),
    (16, 1, 128, 24, False, True),                     # 16 query heads to a KV head
    (16, 1, 256, 40, True, False),
    (3, 3, 128, 8, False, False),                      # one to one
    (10, 2, 256, 256, True, True),
    (14, 2, 128, 64, True, False),
])
def test_attend_over_ragged_lengths(H, kv, D, page, fp8, gated):
    g = gen(H * 13 + D + page)
    lens = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1000, 3]
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    cache = on_gpu(parts)
    B = len(lens)
    q = bf(randn(g, B, H, D))
    gate = bf(randn(g, B, H, D)) if gated else None
    check_attend(parts, cache, q, table, torch.tensor(lens, dtype=torch.int32) - 1, gate)


@pytest.mark.parametrize("n", [1, 31, 100, 1025, 4096, 9999])
@pytest.mark.parametrize("H,kv,D,page,fp8", [(16, 4, 256, 64, True), (8, 1, 128, 24, False)])
def test_attend_one_sequence(n, H, kv, D, page, fp8):
    g = gen(n)
    table, n_pages = tables(g, [n], page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    check_attend(parts, on_gpu(parts), bf(randn(g, 1, H, D, std=2.0)), table, torch.tensor([n - 1], dtype=torch.int32))


@pytest.mark.parametrize("B,H,kv,D", [(2048, 16, 1, 256), (513, 8, 8, 128), (700, 32, 32, 128)])
def test_attend_many_sequences(B, H, kv, D):
    """The most sequences that a call takes with the widest group, and counts that fit nothing: lengths of
    0 to 70 with a few long ones in between."""
    g = gen(B)
    page = 8
    lens = torch.randint(0, 70, (B,), generator=g).tolist()
    lens[0], lens[B // 2], lens[B - 1] = 0, 900, 1500
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, True)
    q, last = bf(randn(g, B, H, D)), torch.tensor(lens, dtype=torch.int32) - 1
    out = on_gpu(parts).attend(q.to(DEV), table.to(DEV), last.to(DEV), paged.attn_workspace(H, kv, D)).cpu()
    empty = last < 0
    assert bool((out[empty] == 0).all()) and bool(torch.isfinite(out).all())
    some = [0, 1, 2, B // 2 - 1, B // 2, B // 2 + 1, B - 2, B - 1] + torch.randint(0, B, (60,), generator=g).tolist()
    want, tol = ref.attend(q[some], *parts, table[some], last[some])
    assert bool(((out[some].double() - want).abs() <= HALF_BF16 * (want.abs() + tol) + tol).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_attend_strided_q_and_gate(fp8):
    """q and its gate interleaved per head, as the gated q projection leaves them."""
    g = gen(21)
    B, H, kv, D, page = 5, 16, 4, 256, 16
    lens = [40, 3, 200, 0, 77]
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    qg = bf(randn(g, B, H, 2 * D))
    d = qg.to(DEV)
    cache, last = on_gpu(parts), torch.tensor(lens, dtype=torch.int32) - 1
    ws = paged.attn_workspace(H, kv, D)
    out = cache.attend(d[..., :D], table.to(DEV), last.to(DEV), ws, gate=d[..., D:])
    same = cache.attend(d[..., :D].contiguous(), table.to(DEV), last.to(DEV), ws, gate=d[..., D:].contiguous())
    assert torch.equal(out, same)
    want, tol = ref.attend(qg[..., :D], *parts, table, last, qg[..., D:])
    assert bool(((out.cpu().double() - want).abs() <= HALF_BF16 * (want.abs() + tol) + tol).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_attend_never_uses_what_lies_behind_the_newest_position(fp8):
    """NaN, infinities and the largest values in slots behind a sequence's last position and on pages
    that no table names change nothing, bit for bit."""
    g = gen(22)
    H, kv, D, page = 8, 2, 256, 24
    lens = [1, 23, 25, 100, 700]
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    last = torch.tensor(lens, dtype=torch.int32) - 1
    q = bf(randn(g, len(lens), H, D))
    clean = check_attend(parts, on_gpu(parts), q, table, last)
    seen = torch.zeros(n_pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        seen[table[b].long()[j // page], j % page] = True
    for bad in (math.nan, math.inf, -3e38):
        dirty = [t.clone() if t is not None else None for t in parts]
        for t in dirty[:2]:
            if fp8:
                t.view(torch.uint8).transpose(1, 2)[~seen] = 0x7F      # NaN
            else:
                t.transpose(1, 2)[~seen] = bad
        for t in dirty[2:]:
            if t is not None:
                t.transpose(1, 2)[~seen] = bad
        got = on_gpu(dirty).attend(q.to(DEV), table.to(DEV), last.to(DEV), paged.attn_workspace(H, kv, D))
        assert torch.equal(got, clean)


@pytest.mark.parametrize("fp8", [False, True])
def test_attend_leaves_out_pages_that_do_not_exist_and_ends_at_the_table(fp8):
    g = gen(23)
    H, kv, D, page = 8, 2, 128, 8
    table, n_pages = tables(g, [64] * 5, page)
    table[0, 0] = -1
    table[1, 7] = n_pages
    table[2, 2], table[2, 3], table[2, 4] = -1, 2**31 - 1, -2**31
    table[3] = -1                                       # nothing left: zeros
    parts = pool(g, n_pages, kv, page, D, fp8)
    last = torch.tensor([63, 63, 50, 63, 2**31 - 1], dtype=torch.int32)
    out = check_attend(parts, on_gpu(parts), bf(randn(g, 5, H, D)), table, last, bf(randn(g, 5, H, D)))
    assert bool((out[3] == 0).all())


@pytest.mark.parametrize("lens", [(0, 40, 900), (0, 40, 40000)])   # in one workgroup, in pieces
def test_attend_to_nothing_is_zeros_whatever_the_gate_holds(lens):
    g = gen(30)
    H, kv, D, page = 8, 2, 256, 16
    table, n_pages = tables(g, lens, page)
    table[:] = -1
    out = on_gpu(pool(g, n_pages, kv, page, D, True)).attend(
        bf(randn(g, 3, H, D)).to(DEV), table.to(DEV), torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=DEV),
        paged.attn_workspace(H, kv, D), gate=torch.full((3, H, D), math.nan, dtype=torch.bfloat16, device=DEV))
    assert bool((out == 0).all())


def test_attend_propagates_a_visible_nan():
    g = gen(24)
    H, kv, D, page, n = 4, 2, 128, 8, 300
    for where in (0, 1):
        table, n_pages = tables(g, [n, n], page)
        parts = pool(g, n_pages, kv, page, D, False)
        parts[where][int(table[0, 12]), 1, 3, 5] = math.nan       # sequence 0, KV head 1
        out = on_gpu(parts).attend(bf(randn(g, 2, H, D)).to(DEV), table.to(DEV),
                                   torch.tensor([n - 1] * 2, dtype=torch.int32, device=DEV),
                                   paged.attn_workspace(H, kv, D)).cpu()
        nan = torch.isnan(out.float())
        assert not bool(nan[1].any()) and not bool(nan[0, :2].any())
        assert bool(nan[0, 2:].all()) if where == 0 else bool(nan[0, 2:, 5].all())


@pytest.mark.parametrize("peak", [0, 150, 299])
def test_attend_one_position_outweighs_all(peak):
    """A score far above the others, first, in between or last: its value comes back."""
    g = gen(25)
    H, kv, D, page, n = 4, 1, 256, 16, 300
    table, n_pages = tables(g, [n], page)
    parts = pool(g, n_pages, kv, page, D, False, std=0.1)
    pid, off = int(table[0, peak // page]), peak % page
    parts[0][pid, 0, off] = 20.0
    q = bf(torch.ones(1, H, D))
    out = check_attend(parts, on_gpu(parts), q, table, torch.tensor([n - 1], dtype=torch.int32))
    assert torch.equal(out.cpu()[0], parts[1][pid, 0, off].expand(H, D))


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_past_32_bits(fp8):
    """Pages at the end of a pool of more than 2^32 bytes a tensor (bf16: 2^31 elements)."""
    g = gen(26)
    H, kv, D, page = 8, 4, 256, 64
    n_pages = (1 << 32) // (kv * page * D) + 40
    raw = [torch.empty(n_pages, kv, page, D, dtype=torch.uint8 if fp8 else torch.bfloat16, device=DEV) for _ in range(2)]
    sc = [torch.empty(n_pages, kv, page, device=DEV) for _ in range(2)] if fp8 else [None, None]
    cache = paged.PagedKVCache(*([t.view(F8) for t in raw] if fp8 else raw), *sc)
    n = 330
    ids = (n_pages - 1 - torch.randperm(6, generator=g)).to(torch.int32)
    table = ids.view(1, -1).to(DEV)
    k, v = bf(randn(g, n, kv, D)), bf(randn(g, n, kv, D))
    at = torch.arange(n, dtype=torch.int32, device=DEV)
    cache.prep(k.to(DEV), v.to(DEV), table, at, seq=torch.zeros_like(at))
    last = torch.tensor([n - 1], dtype=torch.int32)
    ko, vo = (torch.zeros(1, kv, n, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache.read(table, last.to(DEV), ko, vo)
    for o, x in ((ko, k), (vo, v)):
        err = (o.cpu()[0].transpose(0, 1).double() - x.double()).abs()
        s = x.double().abs().amax(-1, keepdim=True) / 448
        lim = (HALF_E4M3 + HALF_BF16 * 1.1) * x.double().abs() + 2.0 ** -10 * 1.01 * s if fp8 else 0 * s
        assert bool((err <= lim).all())
    # the same rows at the front of a small pool give the same output
    small = [t[n_pages - 6:].contiguous() if t is not None else None for t in (cache.k.view(torch.uint8) if fp8 else cache.k,
                                                                             cache.v.view(torch.uint8) if fp8 else cache.v, *sc)]
    c2 = paged.PagedKVCache(*([t.view(F8) for t in small[:2]] if fp8 else small[:2]), *small[2:])
    q = bf(randn(g, 1, H, D)).to(DEV)
    ws = paged.attn_workspace(H, kv, D)
    a = cache.attend(q, table, last.to(DEV), ws)
    b = c2.attend(q, table - (n_pages - 6), last.to(DEV), ws)
    assert torch.equal(a, b)


def test_attend_is_the_same_each_time_and_in_any_batch():
    """Repeats are equal bit for bit, with other shapes on the same workspace in between; an output
    differs from the same sequence's alone only by how its length is split (fp32)."""
    g = gen(27)
    H, kv, D, page = 16, 4, 256, 16
    lens = [900, 4000, 10, 0, 333]
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, True)
    cache = on_gpu(parts)
    q, last = bf(randn(g, 5, H, D)).to(DEV), (torch.tensor(lens, dtype=torch.int32) - 1).to(DEV)
    ws = paged.attn_workspace(H, kv, D)
    first = cache.attend(q, table.to(DEV), last, ws)
    for b in range(5):
        one = cache.attend(q[b:b + 1], table[b:b + 1].to(DEV), last[b:b + 1], ws)
        assert bool(((one - first[b:b + 1]).abs().float() <= 2 * HALF_BF16 * first[b:b + 1].abs().float() + 1e-5).all())
    for _ in range(3):
        assert torch.equal(cache.attend(q, table.to(DEV), last, ws), first)


@pytest.mark.parametrize("seed", range(24))
def test_attend_takes_every_position_once(seed):
    """Batches of all kinds (empty, tiny, whole tiles, long) and head counts over the ways that the work
    is split: with K zero all weights are equal, so an output is the mean of its sequence's values."""
    g = gen(100 + seed)
    B = [1, 2, 3, 7, 15, 16, 31, 33, 64, 65, 200, 600][seed % 12]
    kv = [1, 2, 3, 4, 8][seed % 5]
    G, D, page, fp8 = 1 + seed % 3, 128 if seed % 2 else 256, [8, 24, 64][seed % 3], seed % 4 < 2
    hi = [30, 300, 4000, 40000][seed % 4] if B < 8 else [30, 300, 2000][seed % 3]
    u = torch.rand(B, generator=g)
    lens = torch.exp(u * math.log(hi)).long()
    lens = torch.where(u < 0.1, 0, torch.where(u > 0.8, (lens // 32 + 1) * 32, lens)).tolist()
    table, n_pages = tables(g, lens, page)
    v = torch.randn(n_pages, kv, page, D, generator=g, dtype=torch.float32)
    v = v.to(F8) if fp8 else bf(v)
    k = torch.zeros(n_pages, kv, page, D, dtype=torch.uint8).view(F8) if fp8 else torch.zeros_like(v)
    sc = [torch.ones(n_pages, kv, page)] * 2 if fp8 else [None, None]
    cache = on_gpu((k, v, *sc))
    q = bf(randn(g, B, kv * G, D))
    last = torch.tensor(lens, dtype=torch.int32) - 1
    out = cache.attend(q.to(DEV), table.to(DEV), last.to(DEV), paged.attn_workspace(kv * G, kv, D)).cpu().double()
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((out[b] == 0).all())
            continue
        j = torch.arange(n)
        rows = v[table[b].long()[j // page]] if not fp8 else v.view(torch.uint8)[table[b].long()[j // page]].view(F8)
        mean = rows.double()[j, :, j % page].mean(0).repeat_interleave(G, 0)    # [heads, D]
        # sums of n fp32 terms of weight 1 in some order, |v| below 6: well within n 2^-24 6 / n each
        lim = HALF_BF16 * mean.abs() + 6 * 2.0 ** -20
        assert bool(((out[b] - mean).abs() <= lim).all()), (b, n)


# ------------------------------------------------------------------ streams and graphs
def test_calls_at_once_on_two_streams_with_workspaces_of_their_own():
    g = gen(31)
    H, kv, D, page = 16, 4, 256, 16
    jobs = []
    for lens in ([3000, 50, 700], [9000]):
        table, n_pages = tables(g, lens, page)
        cache = on_gpu(pool(g, n_pages, kv, page, D, True))
        q, last = bf(randn(g, len(lens), H, D)).to(DEV), (torch.tensor(lens, dtype=torch.int32) - 1).to(DEV)
        ws = paged.attn_workspace(H, kv, D)
        jobs.append((cache, q, table.to(DEV), last, ws, cache.attend(q, table.to(DEV), last, ws), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for (cache, q, table, last, ws, _, st), outs in zip(jobs, got):
            with torch.cuda.stream(st):
                outs.append(cache.attend(q, table, last, ws))
    torch.cuda.synchronize()
    for job, outs in zip(jobs, got):
        assert all(torch.equal(o, job[5]) for o in outs)


def test_graphs_that_share_a_workspace_follow_lengths_tables_and_streams():
    """Two captured decode steps (other batches, one workspace) replayed in turn while lengths,
    tables and inputs change, against eager calls."""
    g = gen(28)
    H, kv, D, page = 16, 4, 256, 16
    cos, sin = (t.to(DEV) for t in orc.rope_tables(2048, 64, 1e7))
    rp = paged.RopeAxes(cos, sin, (11, 11, 10), interleaved=True)
    ws = paged.attn_workspace(H, kv, D)
    steps = []
    for B in (3, 7):
        table, n_pages = tables(g, [640] * B, page)
        parts = pool(g, n_pages, kv, page, D, True)
        s = dict(cache=on_gpu(parts), twin=on_gpu(parts), table=table.to(DEV),
                 q=bf(randn(g, B, H, 2 * D)).to(DEV), k=bf(randn(g, B, kv, D)).to(DEV), v=bf(randn(g, B, kv, D)).to(DEV),
                 at=torch.zeros(B, dtype=torch.int32, device=DEV), pos=torch.zeros(3, B, dtype=torch.int32, device=DEV),
                 qo=torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV),
                 out=torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV))

        def step(s, cache, qo, out, ws):
            cache.prep(s["k"], s["v"], s["table"], s["at"], q=s["q"][..., :D], q_out=qo, rope=rp, pos=s["pos"])
            cache.attend(qo, s["table"], s["at"], ws, gate=s["q"][..., D:], out=out)
        step(s, s["cache"], s["qo"], s["out"], ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(s, s["cache"], s["qo"], s["out"], ws)
        s["graph"] = graph
        # what capture's warm-up wrote is written in the twin as well
        step(s, s["twin"], torch.empty_like(s["qo"]), torch.empty_like(s["out"]), ws)
        steps.append(s)
    side, ws2 = torch.cuda.Stream(), paged.attn_workspace(H, kv, D)
    for i in range(6):
        for s in steps:
            B = s["at"].numel()
            s["at"].copy_(torch.randint(-1, 640, (B,), generator=g).to(torch.int32))
            s["pos"].copy_(torch.randint(0, 2048, (3, B), generator=g).to(torch.int32))
            s["q"].copy_(bf(randn(g, B, H, 2 * D)))
            s["table"].copy_(s["table"][torch.randperm(B, generator=g).to(DEV)])
        torch.cuda.synchronize()
        for s in steps:
            s["graph"].replay()
        eager = []
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for s in steps:
                qo, out = s["qo"].clone(), torch.empty_like(s["out"])
                step(s, s["twin"], qo, out, ws2)
                eager.append((qo, out))
        side.synchronize()
        for s, (qo, out) in zip(steps, eager):
            assert torch.equal(s["qo"], qo) and torch.equal(s["out"], out), f"replay {i}"
            for a, b in ((s["cache"].k, s["twin"].k), (s["cache"].v, s["twin"].v)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), f"replay {i}"
            assert torch.equal(s["cache"].k_scale, s["twin"].k_scale)


# ------------------------------------------------------------------ all of them together
@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_and_next_tokens_through_the_paged_cache(fp8):
    """Two sequences: prompts in chunks (prep, read back, the dense path's prompt attention), then
    decode steps of the batch (prep, attend), against attention in 64 bits over the rows that the
    cache holds."""
    g = gen(29)
    H, kv, D, page, rot = 16, 4, 256, 24, 64
    lib = abi.load()
    chunks, steps = [[50, 290], [7]], 4
    lens = [sum(c) + steps for c in chunks]
    table, n_pages = tables(g, lens, page)
    cache = paged.PagedKVCache.alloc(n_pages, page, kv, D, dtype=F8 if fp8 else torch.bfloat16)
    S = max(lens)
    cos, sin = orc.rope_tables(S, rot, 1e7)
    rp = paged.RopeAxes(cos.to(DEV), sin.to(DEV), (12, 10, 10), interleaved=True)
    axes = ref.axes_of(rot // 2, [12, 10, 10], True)
    qn, kn = randn(g, D, std=0.1), randn(g, D, std=0.1)
    td = table.to(DEV)
    cu = lambda t: t.to(DEV)   # noqa: E731

    def rows():
        k, v = cache.k.cpu(), cache.v.cpu()
        return k, v, *((cache.k_scale.cpu(), cache.v_scale.cpu()) if fp8 else (None, None))

    def want(qx, parts, b, at, gate):
        """Attention of one token (q in 64 bits) over what the cache holds up to it."""
        out, tol = ref.attend(qx[None], *parts, table[b:b + 1], torch.tensor([at]), gate[None])
        return out[0], tol[0]

    for b, cs in enumerate(chunks):
        past = 0
        for M in cs:
            qg, k, v = bf(randn(g, M, H, 2 * D)), bf(randn(g, M, kv, D)), bf(randn(g, M, kv, D))
            at = torch.arange(past, past + M, dtype=torch.int32)
            pos = torch.stack([at, at // 3, at % 5]).to(torch.int32)
            qd, q32 = cu(qg), torch.empty(M, H, D, device=DEV)
            cache.prep(cu(k), cu(v), td, cu(at), seq=torch.full((M,), b, dtype=torch.int32, device=DEV), q=qd[..., :D],
                       q_out=q32, rope=rp, pos=cu(pos), q_norm=cu(qn), k_norm=cu(kn))
            kd, vd = (torch.zeros(1, kv, S, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
            cache.read(td[b:b + 1], torch.tensor([past + M - 1], dtype=torch.int32, device=DEV), kd, vd)
            out = torch.empty(M, H * D, dtype=torch.bfloat16, device=DEV)
            abi.check(lib.qh_attn_prefill(abi.ptr(q32), abi.ptr(qd.view(-1)[D:]), H * 2 * D, 2 * D, abi.ptr(kd), abi.ptr(vd),
                                          abi.ptr(out), M, H, kv, D, past, S, abi.stream_handle()), "attn_prefill")
            torch.cuda.synchronize()
            parts = rows()
            qx = ref.rotate(ref.head_norm(qg[..., :D], qn), cos, sin, pos, axes)
            for i in {0, M // 2, M - 1}:
                y, tol = want(qx[i], parts, b, past + i, qg[i, :, D:])
                # the dense rows are bf16 (half a step of K moves a score by up to sum|q k| 2^-8 / 16, of V a value),
                # the prompt attention rounds its output before the gate and the gate itself
                kk, _ = ref.gather(parts[0], parts[2], table, b, past + i + 1, page)
                vv, _ = ref.gather(parts[1], parts[3], table, b, past + i + 1, page)
                kk, vv = kk.repeat_interleave(H // kv, 0), vv.repeat_interleave(H // kv, 0)
                ds = HALF_BF16 * (kk.abs() * qx[i].abs()[:, None]).sum(-1).amax(-1) / math.sqrt(D) if fp8 else torch.zeros(H)
                top = vv.abs().amax((1, 2))
                lim = (4 * HALF_BF16) * y.abs() + (2 * ds * top + (HALF_BF16 if fp8 else 0) * top)[:, None] + tol + 1e-6
                err = (out[i].cpu().double().view(H, D) - y).abs()
                assert bool((err <= lim).all()), (b, past, i, float((err / lim).max()))
            past += M
    ws = paged.attn_workspace(H, kv, D)
    pos0 = torch.tensor([sum(c) for c in chunks], dtype=torch.int32)
    for t in range(steps):
        at = pos0 + t
        qg, k, v = bf(randn(g, 2, H, 2 * D)), bf(randn(g, 2, kv, D)), bf(randn(g, 2, kv, D))
        pos = torch.stack([at, at // 3, at % 5]).to(torch.int32)
        qd = cu(qg)
        q = cache.prep(cu(k), cu(v), td, cu(at), q=qd[..., :D], rope=rp, pos=cu(pos), q_norm=cu(qn), k_norm=cu(kn))
        out = cache.attend(q, td, cu(at), ws, gate=qd[..., D:])
        torch.cuda.synchronize()
        parts = rows()
        qx = ref.rotate(ref.head_norm(qg[..., :D], qn), cos, sin, pos, axes)
        kx = ref.rotate(ref.head_norm(k, kn), cos, sin, pos, axes)
        for b in range(2):
            pid, off = int(table[b, int(at[b]) // page]), int(at[b]) % page
            check_row(parts[0][pid, :, off], parts[2][pid, :, off] if fp8 else None, kx[b],
                      ARITH * ref.pair_size(kx[b], rot // 2), "k")
            y, tol = ref.attend(q.cpu()[b:b + 1], *parts, table[b:b + 1], at[b:b + 1], qg[b:b + 1, :, D:])
            err = (out.cpu()[b:b + 1].double() - y).abs()
            assert bool((err <= HALF_BF16 * (y.abs() + tol) + tol).all())
            assert bool(((q.cpu()[b].double() - qx[b]).abs() <= HALF_BF16 * qx[b].abs() + 2 * ARITH * ref.pair_size(qx[b], 32)).all())


# ------------------------------------------------------------------ batches of which nothing is left
@pytest.mark.parametrize("fp8", [False, True])
def test_prep_of_padding_alone_without_a_sequence(fp8):
    """A batch whose sequences have all ended: a table without rows, tokens of padding.  Nothing is written."""
    g = gen(40)
    T, H, kv, D, page = 5, 4, 2, 128, 8
    parts = pool(g, 3, kv, page, D, fp8)
    cache = on_gpu(parts)
    none = torch.empty(0, 4, dtype=torch.int32, device=DEV)
    q_was = randn(g, T, H, D)
    q_out = q_was.to(DEV)
    k, v = bf(randn(g, T, kv, D)).to(DEV), bf(randn(g, T, kv, D)).to(DEV)
    at = torch.tensor([-1, 0, 7, 31, 2**31 - 1], dtype=torch.int32, device=DEV)
    seq = torch.tensor([-1, 0, 1, 2**31 - 1, -2**31], dtype=torch.int32, device=DEV)
    assert cache.prep(k, v, none, at, seq=seq, q=bf(randn(g, T, H, D)).to(DEV), q_out=q_out) is q_out
    torch.cuda.synchronize()
    assert torch.equal(q_out.cpu(), q_was)
    for got, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), parts):
        assert got is None or torch.equal(got.cpu().view(torch.uint8), was.view(torch.uint8))


# ------------------------------------------------------------------ infinities that are seen
@pytest.mark.parametrize("lens", [(1, 2, 40), (300, 33), (6000,)])     # in a wave, in a workgroup, in pieces
@pytest.mark.parametrize("H,kv,D", [(8, 2, 256), (16, 2, 128)])
def test_attend_hands_on_a_visible_infinity_of_v(H, kv, D, lens):
    """An infinity in a visible row of V is the output's in its dimension, of the heads of its KV head,
    with its sign; all else is as it was.  Scores stay within a few units, so no weight vanishes."""
    g = gen(41 + D + lens[0])
    page, B = 16, len(lens)
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, False)
    q, last = bf(randn(g, B, H, D)), torch.tensor(lens, dtype=torch.int32) - 1
    ws = paged.attn_workspace(H, kv, D)
    clean = check_attend(parts, on_gpu(parts), q, table, last, ws=ws).cpu()
    for b, n in enumerate(lens):
        for j, d, x in ((0, 5, math.inf), (n // 2, D // 2 + 1, -math.inf), (n - 1, D - 1, math.inf)):
            parts[1][int(table[b, j // page]), 1, j % page, d] = x
    out = on_gpu(parts).attend(q.to(DEV), table.to(DEV), last.to(DEV), ws).cpu()
    want = clean.clone()
    want[:, H // 2:, 5], want[:, H // 2:, D // 2 + 1], want[:, H // 2:, D - 1] = math.inf, -math.inf, math.inf
    assert torch.equal(out, want)


# ------------------------------------------------------------------ batches, every instance of the attention
def check_batch(g, lens, H, kv, D, page, fp8, gated, most=48):
    """A batch against 64 bits, K and V random: its longest and shortest sequences, the first and last ones
    and some in between (`most` of them), zeros and finite values in all."""
    B = len(lens)
    table, n_pages = tables(g, lens, page)
    parts = pool(g, n_pages, kv, page, D, fp8)
    q, last = bf(randn(g, B, H, D)), torch.tensor(lens, dtype=torch.int32) - 1
    gate = bf(randn(g, B, H, D)) if gated else None
    out = on_gpu(parts).attend(q.to(DEV), table.to(DEV), last.to(DEV), paged.attn_workspace(H, kv, D),
                               gate=None if gate is None else gate.to(DEV)).cpu()
    assert bool(torch.isfinite(out).all()) and bool((out[last < 0] == 0).all())
    order = sorted(range(B), key=lambda b: lens[b])
    some = list(dict.fromkeys([0, 1, B - 2, B - 1, *order[-4:], *order[:4], *torch.randperm(B, generator=g).tolist()]))
    some = [b for b in some if 0 <= b < B][:most]
    want, tol = ref.attend(q[some], *parts, table[some], last[some], None if gate is None else gate[some])
    err, lim = (out[some].double() - want).abs(), HALF_BF16 * (want.abs() + tol) + tol
    assert bool((err <= lim).all()), f"{float((err / lim.clamp(min=1e-30)).max()):.3f} of the bound"


def ragged(g, B, positions):
    """B lengths of about `positions` in all: some empty, some of whole tiles, one in sixteen many times the others."""
    u = torch.rand(B, 3, generator=g)
    n = (u[:, 0] * 2 * positions / B / (1 + 8 / 16)).long() + 1
    n = torch.where(u[:, 1] < 1 / 16, 8 * n, n)
    n = torch.where(u[:, 2] < 0.1, 0, torch.where(u[:, 2] > 0.8, (n // 32 + 1) * 32, n))
    return n.tolist()


@pytest.mark.parametrize("B,H,kv,D,page,fp8,gated", [
    (65, 16, 4, 256, 16, True, True),                  # E4M3 of 256 with eight waves
    (200, 16, 4, 256, 24, True, False),
    (600, 16, 4, 256, 8, True, True),
    (300, 10, 2, 256, 64, True, True),
    (129, 12, 1, 256, 40, True, True),                 # ... with four: more than 8 heads to a KV head
    (65, 16, 4, 256, 16, False, True),                 # bf16 of 256
    (130, 8, 8, 256, 40, False, True),
    (600, 4, 1, 256, 64, False, False),
    (65, 64, 8, 128, 32, False, True),                 # bf16 of 128
    (200, 32, 8, 128, 24, False, True),
    (2048, 6, 2, 128, 16, False, True),
    (65, 64, 8, 128, 32, True, True),                  # E4M3 of 128
    (333, 16, 1, 128, 8, True, False),
])
def test_attend_over_more_sequences_than_lanes(B, H, kv, D, page, fp8, gated):
    g = gen(B * 31 + H + D + page)
    check_batch(g, ragged(g, B, 50000 * 1024 // (kv * D) if kv * D > 512 else 100000), H, kv, D, page, fp8, gated)


@pytest.mark.parametrize("seed", range(40))
def test_attend_over_batches_of_all_kinds(seed):
    """Sequences, lengths, heads, width, page and type drawn each by itself."""
    g = gen(1000 + seed)
    pick = lambda *xs: xs[int(torch.randint(0, len(xs), (1,), generator=g))]    # noqa: E731
    B, D, page, fp8 = pick(1, 2, 5, 16, 31, 64, 65, 128, 200, 500), pick(128, 256), pick(8, 16, 24, 64, 256), pick(False, True)
    kv, G, gated = pick(1, 2, 3, 4, 8), pick(1, 2, 4, 5, 8, 9, 16), pick(False, True)
    check_batch(g, ragged(g, B, pick(1000, 8000, 40000) * 512 // (kv * D)), kv * G, kv, D, page, fp8, gated, most=16)


# ------------------------------------------------------------------ values near the type's largest
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,peak", [(64, 40), (40000, 20000), (40000, 20032), (40000, 20064)])   # tiles side by side
def test_attend_to_values_near_the_largest(fp8, n, peak):
    """One position of V near the largest bf16 value, the rest zeros, and its score e^5 times the others':
    a maximum that lags behind must not carry its weight past 1, or a finite output overflows."""
    H, kv, D, page = 8, 2, 256, 16
    g = gen(42 + n)
    table, n_pages = tables(g, [n], page)
    q = bf(torch.zeros(1, H, D))
    q[..., 0] = 16.0
    k, v = (torch.zeros(n_pages, kv, page, D) for _ in range(2))
    pid, off = int(table[0, peak // page]), peak % page
    k[pid, :, off, 0] = 5.0                            # a score of 16 * 5 / sqrt(256) = 5, the others' is 0
    v[pid, :, off] = 3.25e38 * torch.sign(torch.randn(kv, D, generator=g))
    sc = [None, None]
    if fp8:
        sc = [torch.ones(n_pages, kv, page), torch.full((n_pages, kv, page), ref.MIN_SCALE)]
        sc[1][pid, :, off] = 3.25e38 / 448
        k, v = k.to(F8), torch.sign(v).mul(448).to(F8)
    else:
        k, v = bf(k), bf(v)
    check_attend((k, v, *sc), on_gpu((k, v, *sc)), q, table, torch.tensor([n - 1], dtype=torch.int32))
