"""The paged cache's host module (csrc/paged_host.cpp) on CPU tensors, which it takes as those of
device -1, with entry points that only write down what they were given."""
import ctypes

import pytest
import torch

from qwen35_amd import _paged_host, abi

BF, F32, INT = torch.bfloat16, torch.float32, torch.int32
KV, D, PAGE, B, T, H = 2, 128, 8, 3, 5, 6
CACHE = abi.PagedCacheDesc(16, 32, None, None, 4, PAGE, KV, D, 0)


def entry(name, seen, status=0):
    """A C function of entry point `name`'s signature that puts its arguments into `seen`."""
    rest, args = abi.NATIVE_SIGNATURES[name]

    def record(*a):
        seen.append(a)
        return status
    return ctypes.CFUNCTYPE(rest, *args)(record)


def call(fn, name, args, status=0):
    """The host function's result and the arguments that the entry point saw (None: not called)."""
    seen = []
    f = entry(name, seen, status)
    got = fn(ctypes.cast(f, ctypes.c_void_p).value, ctypes.addressof(CACHE), -1, *args)
    return got, (seen[0] if seen else None)


def rope(axes):
    return abi.RopeAxesDesc(16, 32, 64, 32, axes, 0, (ctypes.c_int * 4)(*([16 // axes] * axes), *([0] * (4 - axes))))


def prep_args():
    qg = torch.zeros(T, H, 2 * D, dtype=BF)
    kv = torch.zeros(T, 2 * KV * D + 8, dtype=BF)
    r = rope(2)
    a = dict(rope=ctypes.addressof(r), k=kv[:, :KV * D].view(T, KV, D), v=kv[:, KV * D:2 * KV * D].view(T, KV, D),
             pages=torch.zeros(B, 4, dtype=INT), at=torch.zeros(T, dtype=INT), seq=torch.zeros(T, dtype=INT),
             q=qg[..., :D], q_out=torch.zeros(T, H, D), pos=torch.zeros(2, T, dtype=INT), q_norm=torch.zeros(D),
             k_norm=torch.zeros(D), eps=0.5, stream=77)
    return a, (r, qg, kv)


def ptr(t):
    return t.data_ptr()


def test_prep_hands_on_pointers_strides_and_sizes():
    a, keep = prep_args()
    got, s = call(_paged_host.prep, "qh_attn_prep_paged", a.values())
    assert got == 0
    assert s == (ctypes.addressof(CACHE), a["rope"], ptr(a["q"]), 2 * D * H, 2 * D, ptr(a["k"]), 2 * KV * D + 8,
                 ptr(a["v"]), 2 * KV * D + 8, ptr(a["q_norm"]), ptr(a["k_norm"]), 0.5, ptr(a["pos"]), ptr(a["seq"]),
                 ptr(a["at"]), T, ptr(a["pages"]), B, 4, ptr(a["q_out"]), 1, H, 77)
    del keep


def test_prep_without_what_may_be_left_out():
    a, keep = prep_args()
    a.update(rope=0, seq=None, q=None, q_out=None, pos=None, q_norm=None, k_norm=None)
    got, s = call(_paged_host.prep, "qh_attn_prep_paged", a.values(), status=-1)
    assert got == -1                                   # the entry point's status
    assert [s[i] for i in (1, 2, 3, 4, 9, 10, 12, 13, 19, 20, 21)] == [None, None, 0, 0, None, None, None, None, None, 0, 0]
    del keep


def test_prep_one_axis_takes_flat_positions():
    for pos in (torch.zeros(T, dtype=INT), torch.zeros(1, T, dtype=INT)):
        a, keep = prep_args()
        r = rope(1)
        a.update(rope=ctypes.addressof(r), pos=pos, q_out=a["q_out"].to(BF))
        got, s = call(_paged_host.prep, "qh_attn_prep_paged", a.values())
        assert got == 0 and s[12] == ptr(pos) and s[20] == 0
        del keep


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(k=torch.zeros(T, KV, D)), dict(k=torch.zeros(T, KV + 1, D, dtype=BF)),
    dict(k=torch.zeros(T, KV, 2 * D, dtype=BF)[..., ::2]), dict(k=torch.zeros(T, 2 * KV, D, dtype=BF)[:, ::2]),
    dict(v=torch.zeros(T + 1, KV, D, dtype=BF)), dict(v=torch.zeros(KV, T, D, dtype=BF).transpose(0, 1)),
    dict(pages=torch.zeros(B, 4, dtype=torch.int64)), dict(pages=torch.zeros(4, B, dtype=INT).t()),
    dict(pages=torch.zeros(4, dtype=INT)), dict(at=torch.zeros(T + 1, dtype=INT)), dict(at=torch.zeros(2 * T, dtype=INT)[::2]),
    dict(seq=torch.zeros(T - 1, dtype=INT)), dict(seq=torch.zeros(T)), dict(seq=[0] * T),
    dict(pos=None), dict(pos=torch.zeros(T, dtype=INT)), dict(pos=torch.zeros(T, 2, dtype=INT).t()),
    dict(q_norm=torch.zeros(D, dtype=BF)), dict(k_norm=torch.zeros(D + 1)), dict(k_norm=torch.zeros(1, D)),
    dict(q=torch.zeros(T, H, D)), dict(q=torch.zeros(T, H, D + 8, dtype=BF)), dict(q=torch.zeros(T, H, 2 * D, dtype=BF)[..., ::2]),
    dict(q=None), dict(q_out=None), dict(q_out=torch.zeros(T, H, D, dtype=torch.float16)),
    dict(q_out=torch.zeros(T, H + 1, D)), dict(q_out=torch.zeros(H, T, D).transpose(0, 1)),
    dict(k=torch.zeros(T, KV, D, dtype=BF, device="meta"))], ids=lambda b: next(iter(b)))
def test_prep_leaves_a_misfit_to_the_caller(bad):
    a, keep = prep_args()
    a.update(bad)
    assert call(_paged_host.prep, "qh_attn_prep_paged", a.values()) == (None, None)
    del keep


def read_args():
    return dict(pages=torch.zeros(B, 4, dtype=INT), last=torch.zeros(B, dtype=INT), k=torch.zeros(B, KV, 40, D, dtype=BF),
                v=torch.zeros(B, KV, 40, D, dtype=BF), stream=77)


def test_read_hands_on_pointers_and_sizes():
    a = read_args()
    got, s = call(_paged_host.read, "qh_kv_read_paged", a.values())
    assert got == 0
    assert s == (ctypes.addressof(CACHE), ptr(a["pages"]), B, 4, ptr(a["last"]), ptr(a["k"]), ptr(a["v"]), 40, 77)


@pytest.mark.parametrize("bad", [
    dict(pages=torch.zeros(B + 1, 4, dtype=INT)), dict(pages=None), dict(last=torch.zeros(B)), dict(last=torch.zeros(B, 1, dtype=INT)),
    dict(k=torch.zeros(B, KV, 40, D)), dict(k=torch.zeros(B, KV, 41, D, dtype=BF)), dict(k=torch.zeros(B, KV, 40, D + 8, dtype=BF)),
    dict(v=torch.zeros(B, 40, KV, D, dtype=BF).transpose(1, 2)), dict(v=None)], ids=lambda b: next(iter(b)))
def test_read_leaves_a_misfit_to_the_caller(bad):
    a = read_args()
    a.update(bad)
    assert call(_paged_host.read, "qh_kv_read_paged", a.values()) == (None, None)


def attend_args():
    qg = torch.zeros(B, H, 2 * D, dtype=BF)
    return dict(q=qg[..., :D], pages=torch.zeros(B, 4, dtype=INT), last=torch.zeros(B, dtype=INT),
                ws=torch.zeros(1000, dtype=torch.uint8), gate=qg[..., D:], out=torch.zeros(B, H, D, dtype=BF), stream=77)


def test_attend_hands_on_pointers_strides_and_sizes():
    a = attend_args()
    got, s = call(_paged_host.attend, "qh_attn_decode_paged", a.values())
    assert got == 0
    assert s == (ctypes.addressof(CACHE), ptr(a["q"]), 2 * D * H, 2 * D, ptr(a["gate"]), 2 * D * H, 2 * D, ptr(a["pages"]), B,
                 4, ptr(a["last"]), H, ptr(a["out"]), ptr(a["ws"]), 1000, 77)
    got, s = call(_paged_host.attend, "qh_attn_decode_paged", {**a, "gate": None}.values())
    assert got == 0 and s[4:7] == (None, 0, 0)


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(B, H, D)), dict(q=torch.zeros(B + 1, H, D, dtype=BF)), dict(q=torch.zeros(B, H * D, dtype=BF)),
    dict(pages=torch.zeros(B, 4)), dict(last=torch.zeros(B + 1, dtype=INT)), dict(ws=torch.zeros(1000)),
    dict(ws=torch.zeros(2000, dtype=torch.uint8)[::2]), dict(gate=torch.zeros(B, H + 1, D, dtype=BF)),
    dict(gate=torch.zeros(B, H, D)), dict(out=torch.zeros(B, H, D)), dict(out=torch.zeros(H, B, D, dtype=BF).transpose(0, 1)),
    dict(out=None)], ids=lambda b: next(iter(b)))
def test_attend_leaves_a_misfit_to_the_caller(bad):
    a = attend_args()
    a.update(bad)
    assert call(_paged_host.attend, "qh_attn_decode_paged", a.values()) == (None, None)


def test_a_call_with_other_arguments_raises():
    for fn in (_paged_host.prep, _paged_host.read, _paged_host.attend):
        with pytest.raises(TypeError, match="arguments"):
            fn(1, 2)
    a, keep = prep_args()
    with pytest.raises(TypeError):
        call(_paged_host.prep, "qh_attn_prep_paged", {**a, "eps": "small"}.values())
    del keep


def odd(*shape):
    """A bf16 tensor whose axes of size 1 have odd strides."""
    t = torch.zeros(shape, dtype=BF)
    return t.as_strided(shape, [s if n > 1 else 2 * s + 7 for n, s in zip(shape[:-1], t.stride()[:-1])] + [1])


@pytest.mark.parametrize("n,heads", [(1, H), (T, 1), (1, 1)])
def test_the_stride_of_an_axis_of_one_is_not_handed_on(n, heads):
    """One token or one head: nothing is read at that axis's stride, whatever it is."""
    a, keep = prep_args()
    zi = torch.zeros(n, dtype=INT)
    q, k, v = odd(n, heads, D), odd(n, KV, D), odd(n, KV, D)
    a.update(k=k, v=v, q=q, at=zi, seq=zi, pos=torch.zeros(2, n, dtype=INT), q_out=torch.zeros(n, heads, D))
    got, s = call(_paged_host.prep, "qh_attn_prep_paged", a.values())
    assert got == 0
    assert s[3:5] == (heads * D if n > 1 else 0, D if heads > 1 else 0)
    assert s[6] == s[8] == (KV * D if n > 1 else 0)
    assert s[2] == ptr(q) and s[5] == ptr(k) and s[7] == ptr(v)
    a = attend_args()
    a.update(q=q, gate=odd(n, heads, D), pages=torch.zeros(n, 4, dtype=INT), last=zi, out=torch.zeros(n, heads, D, dtype=BF))
    got, s = call(_paged_host.attend, "qh_attn_decode_paged", a.values())
    assert got == 0 and s[2:4] == s[5:7] == (heads * D if n > 1 else 0, D if heads > 1 else 0)
    del keep
