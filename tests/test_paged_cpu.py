"""Paged KV cache: what its entry points refuse, before anything touches a GPU, and the
arithmetic that they share with the kernels."""
import ctypes
import random

import pytest
import torch

import _paged_ref as ref
from qwen35_amd import abi, paged

P = [ctypes.c_void_p(1 << 20 | 4096 * k) for k in range(12)]


def cache(**kw):
    d = dict(k=P[0], v=P[1], k_scale=None, v_scale=None, n_pages=4, page_size=16, n_kv=4, head_dim=256, fp8=0)
    d.update(kw)
    return abi.PagedCacheDesc(**d)


def rope(sections=(32,), **kw):
    d = dict(cos_t=P[2], sin_t=P[3], max_pos=64, rot=64, n_axes=len(sections), interleaved=0)
    d.update(kw)
    return abi.RopeAxesDesc(section=(ctypes.c_int * 4)(*sections, *([0] * (4 - len(sections)))), **d)


def prep(c=None, r=None, **kw):
    a = dict(q=P[4], q_ts=8192, q_hs=512, k=P[5], k_ts=1024, v=P[6], v_ts=1024, qn=None, kn=None, eps=1e-6, pos=P[7],
             seq=P[8], at=P[9], T=3, pages=P[10], n_seqs=2, max_pages=4, q_out=P[11], f32=0, heads=16)
    a.update(kw)
    c = cache() if c is None else c
    return abi.load().qh_attn_prep_paged(ctypes.byref(c), None if r is None else ctypes.byref(r), *a.values(), None)


def read(c=None, **kw):
    a = dict(pages=P[10], n_seqs=2, max_pages=4, last=P[9], k=P[4], v=P[5], max_seq=64)
    a.update(kw)
    return abi.load().qh_kv_read_paged(ctypes.byref(c or cache()), *a.values(), None)


def attend(c=None, **kw):
    a = dict(q=P[4], q_bs=4096, q_hs=256, gate=None, g_bs=0, g_hs=0, pages=P[10], n_seqs=2, max_pages=4, last=P[9],
             heads=16, out=P[11], ws=P[8], ws_bytes=1 << 40)
    a.update(kw)
    return abi.load().qh_attn_decode_paged(ctypes.byref(c or cache()), *a.values(), None)


@pytest.mark.parametrize("call", [prep, read, attend])
@pytest.mark.parametrize("bad,said", [
    (dict(k=None), "null cache"),
    (dict(v=None), "null cache"),
    (dict(head_dim=64), "head_dim"),
    (dict(head_dim=0), "head_dim"),
    (dict(page_size=12), "page_size"),
    (dict(page_size=0), "page_size"),
    (dict(page_size=-8), "page_size"),
    (dict(n_pages=0), "n_pages"),
    (dict(n_kv=0), "n_kv"),
    (dict(fp8=1), "scales"),
    (dict(fp8=1, k_scale=P[2]), "scales"),
    (dict(k_scale=P[2], v_scale=P[3]), "scales"),
    (dict(k=ctypes.c_void_p(4104)), "aligned"),
    (dict(fp8=1, k_scale=P[2], v_scale=ctypes.c_void_p(4100)), "aligned"),
])
def test_a_cache_that_no_entry_point_takes(call, bad, said):
    assert call(cache(**bad)) == -1
    assert said in abi.last_error()


@pytest.mark.parametrize("call", [prep, read, attend])
@pytest.mark.parametrize("bad", [dict(n_seqs=-1), dict(max_pages=0), dict(pages=None), dict(n_seqs=65536),
                                 dict(max_pages=1 << 27)])
def test_a_page_table_that_no_entry_point_takes(call, bad):
    assert call(**bad) == -1
    assert "n_seqs" in abi.last_error()


def test_null_descriptor():
    lib = abi.load()
    assert lib.qh_kv_read_paged(None, P[10], 2, 4, P[9], P[4], P[5], 64, None) == -1
    assert "null cache" in abi.last_error()


@pytest.mark.parametrize("bad,said", [
    (dict(T=-1), "T=-1"),
    (dict(heads=0), "n_heads"),
    (dict(heads=4097), "4096 heads"),
    (dict(c=cache(n_kv=4097)), "4096 heads"),
    (dict(seq=None, T=3), "one per sequence"),
    (dict(k=None), "null pointer"),
    (dict(v=None), "null pointer"),
    (dict(at=None), "null pointer"),
    (dict(q_out=None), "null pointer"),
    (dict(q_out=P[4]), "alias"),
    (dict(q_ts=8190), "multiples of 8"),
    (dict(q_hs=260), "multiples of 8"),
    (dict(k_ts=1025), "multiples of 8"),
    (dict(v_ts=1028), "multiples of 8"),
    (dict(q=ctypes.c_void_p(4098)), "aligned"),
    (dict(q_out=ctypes.c_void_p(4104)), "aligned"),
    (dict(qn=ctypes.c_void_p(4100)), "aligned"),
])
def test_prep_refusals(bad, said):
    assert prep(**bad) == -1
    assert said in abi.last_error()


@pytest.mark.parametrize("r,said", [
    (rope(rot=24, sections=(12,)), "rot=24"),
    (rope(rot=272, sections=(136,)), "rot=272"),
    (rope(rot=-16), "rot=-16"),
    (rope(max_pos=0), "max_pos"),
    (rope(cos_t=None), "null table"),
    (rope(n_axes=0), "n_axes"),
    (rope(n_axes=5), "n_axes"),
    (rope(sections=(30,)), "add up"),
    (rope(sections=(16, 8, 4)), "add up"),
    (rope(sections=(40, -8)), "section"),
    (rope(sections=(4, 4, 24), interleaved=1), "section[2]"),
])
def test_rotary_axes_refusals(r, said):
    assert prep(r=r) == -1
    assert said in abi.last_error()


def test_rotation_needs_positions():
    assert prep(r=rope(), pos=None) == -1
    assert "null table" in abi.last_error()


@pytest.mark.parametrize("bad", [dict(max_seq=0), dict(last=None), dict(k=None), dict(v=None),
                                 dict(k=ctypes.c_void_p(4104))])
def test_read_refusals(bad):
    assert read(**bad) == -1
    assert "kv_read_paged" in abi.last_error()


@pytest.mark.parametrize("bad,said", [
    (dict(heads=18), "n_heads"),
    (dict(heads=0), "n_heads"),
    (dict(heads=68), "n_heads"),           # 17 query heads to a KV head
    (dict(n_seqs=2049), "at most 2048"),
    (dict(q=None), "null pointer"),
    (dict(last=None), "null pointer"),
    (dict(out=None), "null pointer"),
    (dict(ws=None), "null pointer"),
    (dict(out=P[4]), "alias"),
    (dict(gate=P[11]), "alias"),
    (dict(q_bs=4100), "multiples of 8"),
    (dict(gate=P[7], g_hs=4), "multiples of 8"),
    (dict(q=ctypes.c_void_p(4104)), "aligned"),
    (dict(ws=ctypes.c_void_p(4096 + 128)), "256-byte"),
    (dict(ws_bytes=1024), "workspace"),
])
def test_attention_refusals(bad, said):
    assert attend(**bad) == -1
    assert said in abi.last_error()


def test_read_pairs_limit():
    assert read(cache(n_kv=64), n_seqs=1024) == -1
    assert "pairs" in abi.last_error()


def test_attention_pairs_limit():
    assert attend(cache(n_kv=64), n_seqs=2048, heads=64) == -1
    assert "pairs" in abi.last_error()
    assert attend(cache(n_kv=32), n_seqs=2048, heads=32, max_pages=1 << 17) == -1
    assert "tiles" in abi.last_error()


def test_workspace_size():
    lib = abi.load()
    assert lib.qh_attn_decode_paged_workspace_size(16, 4, 256) > 0
    for bad in [(16, 3, 256), (0, 4, 256), (16, 0, 256), (68, 4, 256), (16, 4, 64)]:
        assert lib.qh_attn_decode_paged_workspace_size(*bad) == 0
    with pytest.raises(ValueError):
        paged.attn_workspace(16, 3, 256)


def test_nothing_to_do_launches_nothing():
    assert prep(T=0) == 0
    assert read(n_seqs=0) == 0
    assert attend(n_seqs=0) == 0


def test_wrappers_refuse_cpu_tensors():
    k = torch.zeros(2, 4, 16, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        paged.PagedKVCache(k, k.clone())
    with pytest.raises(ValueError, match="GPU"):
        paged.RopeAxes(torch.zeros(8, 64), torch.zeros(8, 64))


def test_division_by_the_page_size():
    """The multiplier and shift of qh_paged_view give the quotient for every position below 2^31."""
    rng = random.Random(3)
    for d in list(range(8, 600, 8)) + [8 * rng.randint(1, 1 << 27) for _ in range(400)] + [0x7FFF0000]:
        s = 3
        while (1 << s) < d:
            s += 1
        m = (1 << (31 + s)) // d + 1
        assert m < 1 << 32
        for x in [0, 1, d - 1, d, d + 1, 2**31 - 1] + [rng.randrange(2**31) for _ in range(40)] + \
                [d * rng.randrange(2**31 // d) + e for e in (-1, 0) for _ in range(20)]:
            if 0 <= x < 2**31:
                assert (x * m >> 32) >> (s - 1) == x // d, (x, d)


def test_axes_of_pairs():
    assert ref.axes_of(8, [4, 2, 2], False) == [0, 0, 0, 0, 1, 1, 2, 2]
    assert ref.axes_of(8, [4, 2, 2], True) == [0, 1, 2, 0, 1, 2, 0, 0]
    a = ref.axes_of(32, [11, 11, 10], True)
    assert [a.count(i) for i in range(3)] == [11, 11, 10]


@pytest.mark.parametrize("pages", [None, P[10]])
def test_prep_without_sequences_launches_nothing(pages):
    """Every token of a batch without sequences is left out: there is no table to look anything up in
    (an empty tensor's address is null)."""
    assert prep(n_seqs=0, pages=pages) == 0, abi.last_error()
    assert prep(c=cache(fp8=1, k_scale=P[2], v_scale=P[3]), r=rope(), n_seqs=0, pages=pages) == 0, abi.last_error()
    # what no call may bring is refused all the same
    for bad, said in ((dict(k=None), "null pointer"), (dict(seq=None), "one per sequence"), (dict(k_ts=1025), "multiples of 8"),
                      (dict(r=rope(rot=24, sections=(12,))), "rot=24")):
        assert prep(n_seqs=0, pages=pages, **bad) == -1
        assert said in abi.last_error()


@pytest.mark.parametrize("T", [2**26 - 63, 2**31 - 1])
def test_prep_token_limit(T):
    """More tokens than a launch can count: k and v may be expanded views, so such a call fits the memory."""
    assert prep(T=T, q=None, q_out=None) == -1
    assert f"T={T}" in abi.last_error()
