"""Page tables of a batch whose sequences come and go, kept on the GPU.

The reference serves one sequence, whose position is a Python integer (main.py:1509-1604).  Here each
row of a batch holds the pages of one sequence in a paged cache (``paged.PagedKVCache``), and one call
a step does what would otherwise be the host's work between two steps:

  PageTables.step    pages of finished rows given back, pages taken for the new tokens, the
                     position (and the row) of every token of the step (qh_page_tables_step)

``at``, ``seq`` and ``last`` are what ``PagedKVCache.prep`` and ``attend`` take.  Nothing is read
back, so a step can be captured in a HIP graph: what changes between replays is on the device.
"""
import torch

from . import abi
from .paged import _INT, _need, _raw_stream, _serve_host, _with_device


class PageTables:
    """pages: int32 [n_rows, max_pages], the pages of each row's sequence in order (what lies
    behind a row's last page is not read); length: int32 [n_rows], the positions that it holds;
    free: int32 [n_pages] with the ids of the pages that no row holds, n_free: int32 [1], how many
    they are (the last of them is taken first).  No page is in two places: sequences that share
    pages are not for these tables.  A step takes at most 2048 rows of 1 to 2^31 - 65536 positions."""

    def __init__(self, pages, length, free, n_free, page_size):
        dev = pages.get_device()
        if dev < 0:
            raise ValueError("PageTables: tensors must be on the GPU (there is no CPU fallback)")
        _need(pages, "pages", _INT, (None, None), dev)
        _need(length, "length", _INT, (len(pages),), dev)
        _need(free, "free", _INT, (None,), dev)
        _need(n_free, "n_free", _INT, (1,), dev)
        if not 8 <= page_size < 1 << 31 or page_size % 8:
            raise ValueError(f"page_size: a positive multiple of 8, got {page_size}")
        self.pages, self.length, self.free, self.n_free = pages, length, free, n_free
        self.page_size, self.n_rows, self.dev, self.device = int(page_size), len(pages), dev, pages.device
        self._entry = abi.address("qh_page_tables_step")
        self._step = _serve_host().step

    @classmethod
    def alloc(cls, n_rows, max_pages, n_pages, page_size, device="cuda"):
        """Rows that hold nothing, all of `n_pages` free: page 0 is taken first."""
        free = torch.arange(n_pages - 1, -1, -1, dtype=_INT, device=device)
        zero = torch.zeros(n_rows, max_pages + 1, dtype=_INT, device=device)
        return cls(zero[:, 1:].contiguous(), zero[:, 0].contiguous(), free, torch.full((1,), n_pages, dtype=_INT, device=device),
                   page_size)

    def step(self, new, at, seq=None, done=None, start=None, last=None, length_out=None, n_free_out=None):
        """Plan a step of new[b] tokens (int32 [n_rows], negative: none) for each row.

        Rows with done[b] != 0 (int32 [n_rows]) first give their pages back and hold nothing; with
        new[b] > 0 they begin again.  Then rows are served in order while free pages and the step's
        T token rows last; a row that is not served gets no token in this step, and neither does
        one that the whole of them could not serve (which holds up no other).

        With `seq` the tokens of all rows lie one behind the other: at, seq int32 [T] are the
        position and the row of each, -1 behind the last one, and start, int32 [n_rows + 1], the
        first flat row of each row (start[b + 1] - start[b] tokens were served).  Without it, at is
        int32 [n_rows] with the position of the one token of each row, -1 where it has none
        (any new[b] > 0 counts as one).  last: int32 [n_rows], the newest position of each row, -1
        where it holds nothing.

        `pages`, `free`, `length` and `n_free` are brought up to date in place; with length_out and
        n_free_out, int32 of the same sizes, those two go there instead."""
        length_out = self.length if length_out is None else length_out
        n_free_out = self.n_free if n_free_out is None else n_free_out
        rc = _with_device(self.dev, self._step, self._entry, self.dev, self.pages, self.page_size, self.length, new, done,
                          self.free, self.n_free, length_out, n_free_out, at, seq, start, last, _raw_stream(self.dev))
        if rc is None:
            self._refuse(new, at, seq, done, start, last, length_out, n_free_out)
        if rc != 0:
            abi.check(rc, "page_tables_step")

    def _refuse(self, new, at, seq, done, start, last, length_out, n_free_out):
        """Raise for the first argument of `step` that it does not take."""
        dev, n = self.dev, self.n_rows
        _need(new, "new", _INT, (n,), dev)
        _need(at, "at", _INT, (None if seq is not None else n,), dev)
        if seq is not None:
            _need(seq, "seq", _INT, (len(at),), dev)
            if start is None:
                raise ValueError("seq: needs start")
        elif start is not None:
            raise ValueError("start: there is no seq")
        for t, name, size in ((start, "start", n + 1), (done, "done", n), (last, "last", n), (length_out, "length_out", n),
                              (n_free_out, "n_free_out", 1)):
            if t is not None:
                _need(t, name, _INT, (size,), dev)
        raise ValueError("step: arguments that do not fit together")
