"""The rules of PageTables.step, row after row."""
import torch


def step(pages, length, free, new, done, page, T, flat):
    """(pages, length, free stack, at, seq, start, last) after a step; pages a list of lists with any
    length, free the whole stack's list, whose entries above the free ones keep what they held."""
    pages, length = [list(r) for r in pages], list(length)
    n_free, free = free[0], list(free[1])
    S, room = len(pages), len(pages[0]) * page if pages else 0
    for b in range(S):
        if done is not None and done[b]:
            for j in range(-(-length[b] // page)):
                free[n_free] = pages[b][j]
                n_free += 1
            length[b] = 0
    want_pages = want_tokens = taken = 0
    got = []
    for b in range(S):
        t = max(new[b], 0) if flat else min(max(new[b], 0), 1)
        held = -(-length[b] // page)
        need = -(-(length[b] + t) // page) - held
        if length[b] + t > room or need > n_free or t > T:
            got.append(0)
            continue
        want_pages += need
        if need and want_pages > n_free:
            got.append(0)
            continue
        want_tokens += t
        if flat and t and want_tokens > T:
            got.append(0)
            continue
        for j in range(need):
            pages[b][held + j] = free[n_free - 1 - taken]
            taken += 1
        got.append(t)
    at, seq, start = [], [], [0]
    for b in range(S):
        row = [length[b] + i for i in range(got[b])]
        at += row if flat else (row or [-1])
        seq += [b] * got[b]
        start.append(start[-1] + got[b])
    if flat:
        seq += [-1] * (T - len(at))
        at += [-1] * (T - len(at))
    length = [n + g for n, g in zip(length, got)]
    return dict(pages=pages, length=length, n_free=n_free - taken, free=free, at=at, seq=seq, start=start,
                last=[n - 1 for n in length])


def batch(rng, rows, page, max_pages, spare, fill, most, flat, over):
    """A batch in the middle of its life: (pages, length, (n_free, stack), new, done)."""
    room = max_pages * page
    length = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, room), room]) if rng.random() < fill else 0
              for _ in range(rows)]
    length = [min(n, room) for n in length]
    held = [-(-n // page) for n in length]
    ids = rng.sample(range(sum(held) + spare), sum(held) + spare)
    pages, at = [], 0
    for h in held:
        pages.append(ids[at:at + h] + [-7] * (max_pages - h))
        at += h
    new = [rng.choice([0, -3, 1, 1, 1, rng.randint(0, most)]) for _ in range(rows)]
    done = [int(rng.random() < over) * rng.choice([1, -1, 5]) for _ in range(rows)] if over else None
    return pages, length, (spare, ids[at:] + [-9] * sum(held)), new, done


def tensors(state, device):
    pages, length, (n_free, free), new, done = state
    t = lambda v, *shape: torch.tensor(v, dtype=torch.int32, device=device).view(*shape)   # noqa: E731
    n = len(length)
    return dict(pages=t(pages, n, -1), length=t(length, n), free=t(free, -1), n_free=t([n_free], 1), new=t(new, n),
                done=None if done is None else t(done, n))
