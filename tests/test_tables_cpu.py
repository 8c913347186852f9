"""Page tables of a step: what the entry point refuses before anything touches a GPU, what the host
module hands on, and the rules themselves."""
import ctypes
import random

import pytest
import torch

import _tables_ref as ref
from qwen35_amd import _serve_host, abi, tables

P = [ctypes.c_void_p(1 << 20 | 4096 * k) for k in range(12)]
INT = torch.int32


def call(**kw):
    a = dict(pages=P[0], n_rows=3, max_pages=4, page_size=16, length=P[1], new=P[2], done=P[3], free=P[4], n_pages=9,
             n_free=P[5], length_out=P[1], n_free_out=P[5], at=P[6], seq=P[7], T=5, start=P[8], last=P[9])
    a.update(kw)
    return abi.load().qh_page_tables_step(*a.values(), None)


@pytest.mark.parametrize("bad,said", [
    (dict(n_rows=-1), "n_rows=-1"), (dict(n_rows=2049), "at most 2048"), (dict(page_size=0), "page_size"),
    (dict(page_size=12), "page_size"), (dict(page_size=-8), "page_size"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 27), "2^31"), (dict(n_pages=-1), "n_pages"), (dict(T=-1), "T=-1"), (dict(T=2**26 - 63), "2^26"),
    (dict(seq=None), "start belongs"), (dict(start=None), "start belongs"), (dict(seq=None, start=None), "one token a row"),
    (dict(pages=None), "null"), (dict(length=None), "null"), (dict(new=None), "null"), (dict(free=None), "null"),
    (dict(n_free=None), "null"), (dict(length_out=None), "null"), (dict(n_free_out=None), "null"), (dict(at=None), "null")])
def test_refusals(bad, said):
    assert call(**bad) == -1
    assert "page_tables_step" in abi.last_error() and said in abi.last_error()


def entry(name, seen, status=0):
    rest, args = abi.NATIVE_SIGNATURES[name]

    def record(*a):
        seen.append(a)
        return status
    return ctypes.CFUNCTYPE(rest, *args)(record)


def host(args, status=0):
    seen = []
    f = entry("qh_page_tables_step", seen, status)
    got = _serve_host.step(ctypes.cast(f, ctypes.c_void_p).value, -1, *args)
    return got, (seen[0] if seen else None)


def args(**kw):
    z = lambda *s: torch.zeros(*s, dtype=INT)   # noqa: E731
    a = dict(pages=z(3, 4), page=16, length=z(3), new=z(3), done=z(3), free=z(9), n_free=z(1), length_out=z(3),
             n_free_out=z(1), at=z(5), seq=z(5), start=z(4), last=z(3), stream=77)
    a.update(kw)
    return a


def test_host_hands_on_pointers_and_sizes():
    a = args()
    got, s = host(a.values(), status=-1)
    p = {k: t.data_ptr() for k, t in a.items() if isinstance(t, torch.Tensor)}
    assert got == -1
    assert s == (p["pages"], 3, 4, 16, p["length"], p["new"], p["done"], p["free"], 9, p["n_free"], p["length_out"],
                 p["n_free_out"], p["at"], p["seq"], 5, p["start"], p["last"], 77)
    a = args(at=torch.zeros(3, dtype=INT), seq=None, start=None, done=None, last=None)
    got, s = host(a.values())
    assert got == 0 and s[6] is None and s[13:17] == (None, 3, None, None)


def test_host_keeps_a_step_without_room_a_ragged_one():
    z = torch.zeros(0, dtype=INT)
    a = args(at=z, seq=z)
    got, s = host(a.values())
    assert got == 0 and s[13] is not None and s[14] == 0 and s[15] == a["start"].data_ptr()


@pytest.mark.parametrize("bad", [
    dict(pages=None), dict(pages=torch.zeros(3, 4)), dict(pages=torch.zeros(4, 3, dtype=INT).t()),
    dict(pages=torch.zeros(12, dtype=INT)), dict(length=torch.zeros(4, dtype=INT)), dict(new=torch.zeros(3, dtype=torch.int64)),
    dict(new=[1, 1, 1]), dict(done=torch.zeros(3, dtype=torch.bool)), dict(free=torch.zeros(3, 3, dtype=INT)),
    dict(free=torch.zeros(18, dtype=INT)[::2]), dict(n_free=torch.zeros((), dtype=INT)), dict(n_free=torch.zeros(2, dtype=INT)),
    dict(length_out=torch.zeros(2, dtype=INT)), dict(n_free_out=None), dict(at=None), dict(at=torch.zeros(6, dtype=INT)),
    dict(seq=torch.zeros(4, dtype=INT)), dict(seq=None), dict(start=None), dict(start=torch.zeros(3, dtype=INT)),
    dict(last=torch.zeros(3)), dict(seq=None, start=None), dict(new=torch.zeros(3, dtype=INT, device="meta"))],
    ids=lambda b: next(iter(b)))
def test_host_leaves_a_misfit_to_the_caller(bad):
    assert host(args(**bad).values()) == (None, None)


def test_host_refuses_another_number_of_arguments():
    with pytest.raises(TypeError, match="arguments"):
        _serve_host.step(1, 2)


def test_wrapper_refuses_cpu_tensors():
    z = torch.zeros(1, dtype=INT)
    with pytest.raises(ValueError, match="GPU"):
        tables.PageTables(torch.zeros(1, 4, dtype=INT), z, z, z, 16)


@pytest.mark.parametrize("seed", range(40))
def test_rules_keep_every_page_in_one_place(seed):
    """The rules themselves: after any step each page is in one row or free, rows that were served have
    the pages of their length, and nobody has more tokens than asked for."""
    rng = random.Random(seed)
    page, max_pages, rows = rng.choice([8, 16, 24]), rng.randint(1, 9), rng.randint(1, 40)
    flat = rng.random() < 0.6
    state = ref.batch(rng, rows, page, max_pages, rng.randint(0, 30), 0.7, 3 * page, flat, rng.choice([0, 0.3]))
    T = rng.choice([1, rows, 4 * rows]) if flat else rows
    out = ref.step(*state[:2], state[2], state[3], state[4], page, T, flat)
    held = [p for row, n in zip(out["pages"], out["length"]) for p in row[:-(-n // page)]]
    everything = held + out["free"][:out["n_free"]]
    assert sorted(everything) == list(range(len(everything))) and len(everything) == len(state[2][1])
    assert out["start"][-1] <= T and len(out["at"]) == T
