"""Page tables of a step on the GPU against the rules row after row (_tables_ref.py)."""
import random

import pytest
import torch

import _tables_ref as ref
from qwen35_amd import tables

pytestmark = pytest.mark.gpu
DEV = "cuda"
INT = torch.int32


def out_of(t, T, flat, apart):
    """(keyword arguments of a step, the tensors it writes): apart, lengths and count go to tensors of their own."""
    e = lambda n: torch.full((n,), -77, dtype=INT, device=DEV)   # noqa: E731
    n = t.n_rows
    kw = dict(last=e(n))
    if flat:
        kw.update(seq=e(T), start=e(n + 1))
    if apart:
        kw.update(length_out=e(n), n_free_out=e(1))
    at = e(T)
    return at, kw


def check(state, page, T, flat, apart=False):
    want = ref.step(*state[:2], state[2], state[3], state[4], page, T, flat)
    d = ref.tensors(state, DEV)
    t = tables.PageTables(d["pages"], d["length"], d["free"], d["n_free"], page)
    before = t.length.clone(), t.n_free.clone()
    at, kw = out_of(t, T, flat, apart)
    t.step(d["new"], at, done=d["done"], **kw)
    got = dict(pages=t.pages, free=t.free, at=at, last=kw["last"], length=kw.get("length_out", t.length),
               n_free=kw.get("n_free_out", t.n_free))
    if flat:
        got.update(seq=kw["seq"], start=kw["start"])
    for name, x in got.items():
        w = want[name]
        assert x.flatten().tolist() == (sum(w, []) if name == "pages" else [w] if name == "n_free" else w), name
    if apart:
        assert torch.equal(t.length, before[0]) and torch.equal(t.n_free, before[1])


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 128, 129, 255, 511, 512, 513, 1500, 2047, 2048])
@pytest.mark.parametrize("flat", [False, True])
def test_rows(rows, flat):
    rng = random.Random(rows)
    for spare, over, T in ((0, 0.2, rows), (rows // 3 + 1, 0, 2 * rows), (4 * rows, 0.1, 8 * rows + 5)):
        state = ref.batch(rng, rows, 16, 6, spare, 0.8, 40, flat, over)
        check(state, 16, T if flat else rows, flat, apart=spare > 0)


@pytest.mark.parametrize("seed", range(30))
def test_random_batches(seed):
    rng = random.Random(100 + seed)
    page, rows, flat = rng.choice([8, 16, 24, 40, 128]), rng.choice([1, 5, 40, 300, 900]), rng.random() < 0.6
    state = ref.batch(rng, rows, page, rng.choice([1, 3, 20]), rng.choice([0, 1, 10, 500]), rng.choice([0, 0.5, 1]),
                      rng.choice([2, page, 5 * page]), flat, rng.choice([0, 0.1, 1]))
    check(state, page, rng.choice([1, rows, 3 * rows, 5000]) if flat else rows, flat, apart=rng.random() < 0.5)


@pytest.mark.parametrize("T", [1, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 20000])
def test_long_steps(T):
    """Prompts of thousands of tokens: flat rows at the border between one launch and two."""
    rng = random.Random(T)
    for rows in (1, 7, 600):
        state = ref.batch(rng, rows, 24, 300, 900, 0.2, 5000, True, 0.1)
        check(state, 24, T, True)


@pytest.mark.parametrize("new,spare,T,got", [
    ([5, 900, 5], 3, 100, [5, 0, 5]),           # one that no step could serve holds up nobody
    ([40, 1, 8], 5, 100, [40, 0, 0]),           # 5 + 1 + 1 pages
    ([40, 40, 8], 5, 100, [40, 0, 0]),          # ... one whose pages are gone holds up those that need pages
    ([8, 60, 60, 1], 99, 100, [8, 60, 0, 0]),   # ... one whose tokens have no room holds up all
    ([0, 0, -5], 0, 4, [0, 0, 0]),
    ([2**31 - 1, 3], 9, 10, [0, 3]),
])
def test_who_is_served(new, spare, T, got):
    n = len(new)
    state = ([[-7] * 100 for _ in range(n)], [0] * n, (spare, list(range(max(1, spare)))), new, None)
    want = ref.step(*state[:2], state[2], state[3], state[4], 8, T, True)
    assert [b - a for a, b in zip(want["start"], want["start"][1:])] == got
    check(state, 8, T, True)


def test_a_row_that_goes_on_without_a_page_is_served_behind_one_that_waits():
    state = ([[0, -7], [1, -7], [2, -7]], [8, 3, 8], (1, [3, -9, -9, -9]), [1, 1, 1], None)
    for flat in (False, True):
        want = ref.step(*state[:2], state[2], state[3], state[4], 8, 3, flat)
        assert want["length"] == [9, 4, 8]
        check(state, 8, 3, flat)


def test_a_finished_row_begins_again_on_its_own_pages():
    """Pages given back in a step are the first to be taken in it, into the tables they were read from."""
    state = ([[4, 1], [0, 3], [2, -7]], [16, 9, 5], (0, [-9] * 5), [12, 16, 4], [1, 1, 0])
    for flat in (False, True):
        check(state, 8, 32 if flat else 3, flat)


def test_no_rows():
    t = tables.PageTables(torch.zeros(0, 3, dtype=INT, device=DEV), *(torch.zeros(n, dtype=INT, device=DEV) for n in (0, 4, 1)), 16)
    at, kw = out_of(t, 5, True, False)
    t.step(torch.zeros(0, dtype=INT, device=DEV), at, **kw)
    assert at.tolist() == [-1] * 5 and kw["seq"].tolist() == [-1] * 5 and kw["start"].tolist() == [0]
    t.step(torch.zeros(0, dtype=INT, device=DEV), torch.empty(0, dtype=INT, device=DEV))


def test_no_room_for_any_token():
    state = ([[3, -7], [1, -7]], [5, 8], (2, [0, 2, -9, -9]), [1, 1], [0, 1])
    want = ref.step(*state[:2], state[2], state[3], state[4], 8, 0, True)
    assert want["start"] == [0, 0, 0] and want["length"] == [5, 0]
    check(state, 8, 0, True)


@pytest.mark.parametrize("page_size", [0, 12, -8, 2**32 + 16])
def test_a_page_size_that_is_none(page_size):
    with pytest.raises(ValueError, match="page_size"):
        tables.PageTables.alloc(2, 2, 4, page_size, device=DEV)


def test_state_out_of_range_stays_in_bounds():
    """Lengths and counts that no step leaves behind: nothing outside the tensors is touched."""
    e = lambda v: torch.tensor(v, dtype=INT, device=DEV)   # noqa: E731
    guard = torch.full((3, 6), -5, dtype=INT, device=DEV)
    pages, free = guard[1:2, :2].clone(), e([9, 8, 7])
    t = tables.PageTables(pages, e([2**31 - 1]), free, e([2**31 - 1]), 8)
    at, kw = out_of(t, 1, False, False)
    t.step(e([1]), at, done=e([0]), **kw)          # the row counts as full, the stack as full
    assert t.length.tolist() == [16] and t.n_free.tolist() == [3] and at.tolist() == [-1]
    t.step(e([1]), at, done=e([1]), **kw)          # nothing fits on a full stack: its pages are lost, not written
    assert t.length.tolist() == [1] and t.n_free.tolist() == [2] and at.tolist() == [0]
    assert t.pages.tolist() == [[7, -5]] and t.free.tolist() == [9, 8, 7]
    t2 = tables.PageTables(pages, e([-4]), free, e([-1]), 8)
    t2.step(e([1]), at, **kw)
    assert t2.length.tolist() == [0] and t2.n_free.tolist() == [0] and at.tolist() == [-1]


def test_many_steps_in_place_and_replayed():
    """A batch lives through 60 steps, every other one a replay of a captured step, on a stream of its own."""
    rng = random.Random(5)
    rows, page, max_pages, n_pages, T = 37, 8, 12, 150, 64
    t = tables.PageTables.alloc(rows, max_pages, n_pages, page, device=DEV)
    pages, length, free = [[0] * max_pages for _ in range(rows)], [0] * rows, (n_pages, list(range(n_pages - 1, -1, -1)))
    new, done = torch.zeros(rows, dtype=INT, device=DEV), torch.zeros(rows, dtype=INT, device=DEV)
    at, kw = out_of(t, T, True, False)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        t.step(new, at, done=done, **kw)
    for i in range(60):
        n = [rng.choice([0, 1, 1, rng.randint(0, 30)]) for _ in range(rows)]
        d = [int(rng.random() < 0.15) for _ in range(rows)]
        want = ref.step(pages, length, free, n, d, page, T, True)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            new.copy_(torch.tensor(n, dtype=INT))
            done.copy_(torch.tensor(d, dtype=INT))
            if i % 2:
                graph.replay()
            else:
                t.step(new, at, done=done, **kw)
        torch.cuda.synchronize()
        pages, length, free = want["pages"], want["length"], (want["n_free"], want["free"])
        assert t.pages.tolist() == pages and t.length.tolist() == length and t.n_free.tolist() == [free[0]], i
        assert at.tolist() == want["at"] and kw["seq"].tolist() == want["seq"] and kw["last"].tolist() == want["last"], i


@pytest.mark.parametrize("bad,error", [
    (dict(new=torch.zeros(3)), "new"), (dict(at=torch.zeros(4, dtype=INT)), "at"), (dict(last=torch.zeros(2, dtype=INT)), "last"),
    (dict(seq=torch.zeros(3, dtype=INT)), "seq"), (dict(start=torch.zeros(4, dtype=INT)), "start"),
    (dict(done=torch.zeros(4, dtype=INT)), "done"), (dict(n_free_out=torch.zeros(2, dtype=INT)), "n_free_out")])
def test_refusals_name_the_argument(bad, error):
    t = tables.PageTables.alloc(3, 2, 9, 16, device=DEV)
    kw = dict(new=torch.zeros(3, dtype=INT), at=torch.zeros(3, dtype=INT), **bad) if "new" not in bad and "at" not in bad else \
        dict(dict(new=torch.zeros(3, dtype=INT), at=torch.zeros(3, dtype=INT)), **bad)
    with pytest.raises((ValueError, TypeError), match=error):
        t.step(**{k: v.to(DEV) for k, v in kw.items()})
