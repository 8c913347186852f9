"""A batch of requests served step by step, all of it on the device and captured in one HIP graph: page tables,
a shared projection with each request's adapter, the paged cache, its attention, the head, a token for each row.
Requests come, wait for pages, finish and make room; every token's logits are checked against the request's whole
history in 64 bits, and every token against its logits."""
import math
import random

import pytest
import torch

import _sample_ref as ref
from oracle import qwen35_oracle as orc
from qwen35_amd import abi, adapters, ops, paged, sampling, tables

from _util import bf, gen, quant, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
INT, F32 = torch.int32, torch.float32
ROWS, K, H, KV, D, VOCAB, PAGE, MAX_PAGES, POOL = 6, 256, 2, 1, 128, 1003, 8, 4, 13
N, RANK, ADAPTERS = (H + 2 * KV) * D, 16, 3


class Model:
    """One attention layer of random weights: CPU tensors, and 64-bit logits of a history."""

    def __init__(self, seed):
        g = gen(seed)
        self.embed, self.head = bf(randn(g, VOCAB, K)), bf(randn(g, VOCAB, K, std=0.2))
        self.qkv, self.o = quant(g, N, K, std=1 / math.sqrt(K)), quant(g, K, H * D, std=1 / math.sqrt(H * D))
        low = lambda n, k: (bf(randn(g, ADAPTERS, RANK, k, std=1 / math.sqrt(k))), bf(randn(g, ADAPTERS, n, RANK, std=0.2)))  # noqa: E731
        self.low_qkv, self.low_o, self.scale = low(N, K), low(K, H * D), torch.tensor([0.5, 1.0, 2.0])
        self.norm = randn(g, K, std=0.1)
        self.cos, self.sin = orc.rope_tables(PAGE * MAX_PAGES, 32, 1e4)

    def project(self, x, w, low, a):
        y = x @ orc.dequant(*w).double().t()
        return y if a < 0 else y + float(self.scale[a]) * (x @ low[0][a].double().t()) @ low[1][a].double().t()

    def rotate(self, x):
        """x [tokens, heads, D] at positions 0, 1, ..."""
        c, s = (t[:len(x), None, :16].double() for t in (self.cos, self.sin))
        a, b = x[..., :16], x[..., 16:32]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 32:]], -1)

    def logits(self, history, a):
        x = self.embed[history].double()
        y = self.project(x, self.qkv, self.low_qkv, a).view(len(history), H + 2 * KV, D)
        q, k, v = self.rotate(y[:, :H])[-1], self.rotate(y[:, H:H + KV]), y[:, H + KV:]
        out = [torch.softmax(k[:, h * KV // H] @ q[h] / math.sqrt(D), 0) @ v[:, h * KV // H] for h in range(H)]
        z = x[-1] + self.project(torch.cat(out), self.o, self.low_o, a)
        z = z * torch.rsqrt(z.square().mean() + 1e-6) * (1 + self.norm.double())
        return self.head.double() @ z


def test_requests_come_and_go():
    m, rng = Model(3), random.Random(4)
    lib = abi.load()
    dev = lambda t: t.to(DEV)   # noqa: E731
    t = tables.PageTables.alloc(ROWS, MAX_PAGES, POOL, PAGE, device=DEV)       # 24 pages would serve all
    cache = paged.PagedKVCache.alloc(POOL, PAGE, KV, D, device=DEV)
    rope = paged.RopeAxes(dev(m.cos), dev(m.sin))
    low = [adapters.Adapters(dev(a), dev(b), dev(m.scale)) for a, b in (m.low_qkv, m.low_o)]
    ws = dict(attn=paged.attn_workspace(H, KV, D, device=DEV), low=adapters.adapters_workspace(ROWS, RANK, device=DEV),
              draw=sampling.sample_workspace(ROWS, VOCAB, device=DEV))
    w_qkv, s_qkv, w_o, s_o = (dev(x) for x in (*m.qkv, *m.o))
    embed, head, norm = dev(m.embed), dev(m.head), dev(m.norm)
    new, done, ids = (torch.zeros(ROWS, dtype=INT, device=DEV) for _ in range(3))
    at, last = (torch.zeros(ROWS, dtype=INT, device=DEV) for _ in range(2))
    token = torch.zeros(ROWS, dtype=torch.int64, device=DEV)      # the next token of each row
    u, logprob, drawn = torch.zeros(ROWS, device=DEV), torch.zeros(ROWS, device=DEV), torch.zeros(ROWS, dtype=torch.int64, device=DEV)
    heat, top_p = torch.full((ROWS,), 0.8, device=DEV), torch.full((ROWS,), 0.95, device=DEV)
    top_k, min_p = torch.full((ROWS,), 40, dtype=INT, device=DEV), torch.full((ROWS,), 0.01, device=DEV)
    xn, logits = torch.empty(ROWS, K, dtype=torch.bfloat16, device=DEV), torch.empty(ROWS, VOCAB, dtype=torch.bfloat16, device=DEV)

    def step():
        t.step(new, at, done=done, last=last)
        x = embed.index_select(0, token)
        y = ops.fp8_linear(x, w_qkv, s_qkv)
        low[0].add(x, ids, y, ws["low"], out=y)
        y3 = y.view(ROWS, H + 2 * KV, D)
        q = cache.prep(y3[:, H:H + KV], y3[:, H + KV:], t.pages, at, q=y3[:, :H], rope=rope, pos=at)
        o = cache.attend(q, t.pages, at, ws["attn"]).view(ROWS, H * D)
        z = ops.fp8_linear(o, w_o, s_o)
        z = x + low[1].add(o, ids, z, ws["low"], out=z)
        abi.check(lib.qh_lm_head_rows(abi.ptr(z), abi.ptr(norm), 1e-6, ROWS, K, abi.ptr(head), VOCAB, abi.ptr(xn),
                                      abi.ptr(logits), abi.stream_handle()), "head")
        sampling.sample(logits, u, ws["draw"], temperature=heat, top_k=top_k, top_p=top_p, min_p=min_p, out=drawn, logprob=logprob)
        token.copy_(torch.where(at >= 0, drawn, token))           # a row that waits keeps its token

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                                    # (new = 0: nobody is served)
    torch.cuda.current_stream().wait_stream(side)
    assert at.tolist() == [-1] * ROWS and t.n_free.tolist() == [POOL]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    history, adapter, until, waited, served = [[] for _ in range(ROWS)], [-1] * ROWS, [0] * ROWS, 0, 0
    for i in range(70):
        begin = [b for b in range(ROWS) if len(history[b]) >= until[b]]
        for b in begin:
            until[b] = rng.choice([9, 20, 31])
            history[b], adapter[b] = [rng.randrange(VOCAB)], rng.randrange(-1, ADAPTERS)
            token[b] = history[b][0]
        done.copy_(torch.tensor([int(b in begin) for b in range(ROWS)], dtype=INT))
        ids.copy_(torch.tensor(adapter, dtype=INT))
        new.copy_(torch.tensor([int(rng.random() < 0.95) for _ in range(ROWS)], dtype=INT))
        v = [float(torch.tensor(rng.random(), dtype=F32)) for _ in range(ROWS)]
        u.copy_(torch.tensor(v))
        if i % 5 == 4:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        x, where, got, lp = logits.float().cpu(), at.tolist(), drawn.tolist(), logprob.tolist()
        for b in range(ROWS):
            if where[b] < 0:
                waited += int(new[b])
                continue
            served += 1
            assert where[b] == len(history[b]) - 1, (i, b)
            want = m.logits(history[b], adapter[b])
            # nine roundings to bf16 on the way, each 2^-8 of its tensor's norm at most, through maps that
            # keep norms within about two: 9 / 128
            off = float((x[b].double() - want).norm() / want.norm())
            assert off < 9 / 128, (i, b, off)
            tok, logp, margin = ref.row(x[b], v[b], heat=0.8, k=40, p=0.95, m=0.01)
            assert margin > 2.0 ** -33 and got[b] == tok and abs(lp[b] - logp) < 1e-5, (i, b)
            history[b].append(tok)
        held = [p for row, n in zip(t.pages.tolist(), t.length.tolist()) for p in row[:-(-n // PAGE)]]
        assert sorted(held + t.free.tolist()[:int(t.n_free)]) == list(range(POOL)), i
    assert waited > 5 and served > 150
