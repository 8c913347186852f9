"""The operators of a serving step around the paged key-value cache, as calls that can be timed and
compared.  Each case is a dict of plain values; `kind` names the operator:

  step    the batch's next step planned on the GPU: pages of finished rows given back, pages taken for the
          new tokens, sequence and position of every token of the ragged batch
  adapt   low-rank adapters of many requests added to what a shared projection gave
  sample  a token for each row of logits: temperature, top-k, top-p and min-p, drawn with a given random number

What follows from the case alone (lengths, requests, parameters of the rows) comes from `random.Random` of
its sizes; page numbers, weights, logits and random numbers from the seed.

With `own` false a pass is the operator written out in elementary torch operations, in 32 bits (the
sampler, whose borders between tokens 32 would move, in 64) and rounded once at the end; with `own`
true it is the framework's call.
"""
import math
import random

import torch

own = False

DEV = "cuda"
BF, F32, INT = torch.bfloat16, torch.float32, torch.int32


def listed():
    return [
        # the next token of 64 conversations, three of them over: one row of the batch a sequence
        {"name": "step_decode", "kind": "step", "rows": 64, "prompts": 0, "most": 1, "done": 3, "T": 64, "page": 16,
         "past": 3000, "spare": 64, "flat": False},
        # prompts of new users beside running conversations, more tokens than the step has room for
        {"name": "step_mixed", "kind": "step", "rows": 500, "prompts": 40, "most": 700, "done": 30, "T": 12000, "page": 24,
         "past": 4000, "spare": 300, "flat": True},
        # one user's token through an adapted query projection
        {"name": "adapt_token", "kind": "adapt", "T": 1, "runs": 1, "none": 0, "n": 8, "R": 16, "K": 2560, "N": 8192},
        # a decode batch of 48 users with adapters of their own, some without, gate or up projection
        {"name": "adapt_decode", "kind": "adapt", "T": 48, "runs": 48, "none": 5, "n": 32, "R": 16, "K": 2560, "N": 9216},
        # decode tokens and short prompts together, down projection, larger rank
        {"name": "adapt_ragged", "kind": "adapt", "T": 701, "runs": 23, "none": 3, "n": 16, "R": 64, "K": 9216, "N": 2560},
        # long prompts of four users
        {"name": "adapt_prompt", "kind": "adapt", "T": 3700, "runs": 4, "none": 0, "n": 16, "R": 32, "K": 2560, "N": 9216},
        # one conversation's next token
        {"name": "sample_one", "kind": "sample", "B": 1, "V": 248320, "f32": False, "mix": "chat"},
        # a batch without filters, logits that were worked on in 32 bits
        {"name": "sample_plain", "kind": "sample", "B": 16, "V": 248320, "f32": True, "mix": "plain"},
        # a batch of users with settings of their own; a vocabulary of odd size
        {"name": "sample_batch", "kind": "sample", "B": 48, "V": 50257, "f32": False, "mix": "mixed"},
        # a large serving batch
        {"name": "sample_serve", "kind": "sample", "B": 256, "V": 248320, "f32": False, "mix": "mixed"},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["step", "adapt", "adapt", "adapt", "sample", "sample", "sample"])
    if kind == "step":
        rows, page = _log_int(rng, 8, 2000), rng.choice([8, 16, 24, 32, 40, 64, 128])
        flat = rng.random() < 0.6
        prompts = rng.randint(0, max(1, rows // 10)) if flat else 0
        most = _log_int(rng, 2, 4000) if flat else 1
        want = rows + prompts * most // 2
        return {"kind": kind, "rows": rows, "prompts": prompts, "most": most, "done": rng.randint(0, rows // 4),
                "T": max(1, min(16384, int(want * rng.choice([0.7, 1.1, 1.1])))) if flat else rows, "page": page,
                "past": _log_int(rng, 1, 4000), "spare": 8 + int((rows // page + want // page) * rng.choice([0.5, 1, 2])),
                "flat": flat}
    if kind == "adapt":
        K, N = rng.choice([(2560, 8192), (2560, 9216), (9216, 2560), (4096, 2560), (2560, 1024), (512, 1536), (2560, 12352),
                           (200, 1000), (1000, 264)])
        T, R = _log_int(rng, 1, 3700), rng.choice([8, 16, 16, 32, 32, 64, 24, 128])
        step = rng.random() < 0.5       # a decode step: one token a request
        T = min(T, 256) if step else T
        runs = T if step else min(T, rng.randint(1, 40))
        while 2 * T * R * (K + N) > 2 * 3700 * 32 * 11776:
            R //= 2
        return {"kind": kind, "T": T, "runs": runs, "none": rng.choice([0, 0, runs // 5]), "n": _log_int(rng, 1, 64),
                "R": max(8, R - R % 8), "K": K, "N": N}
    V = rng.choice([248320, 248320, 50257, 32000, _log_int(rng, 2, 300_000)])
    B = _log_int(rng, 1, 256)
    f32 = rng.random() < 0.3
    while B * V * (2 if f32 else 1) > 256 * 248320:
        B = max(1, B // 2)
    return {"kind": kind, "B": B, "V": V, "f32": f32, "mix": rng.choice(["chat", "plain", "mixed", "mixed"])}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _lengths(case):
    """(positions held, new tokens, whether it is over) of each row: `done` rows are over, `prompts` of the others
    begin, the rest run on by one token each, a few of them paused."""
    S = case["rows"]
    rng = random.Random(7 * S + case["past"] + case["T"])
    order = rng.sample(range(S), S)
    over, begin = set(order[:case["done"]]), set(order[case["done"]:case["done"] + case["prompts"]])
    out = []
    for b in range(S):
        if b in begin:
            out.append((0, rng.randint(1, case["most"]), 0))
        else:
            out.append((rng.randint(1, case["past"]), 0 if b in over or rng.random() < 0.03 else 1, int(b in over)))
    return out


def _ids(case):
    """The adapter of each token: runs of tokens of one request, `none` of them without one (-1)."""
    T, runs = case["T"], case["runs"]
    rng = random.Random(11 * T + runs + case["n"])
    cuts = [0] + sorted(rng.sample(range(1, T), runs - 1)) + [T]
    without = set(rng.sample(range(runs), case["none"]))
    ids = []
    for i in range(runs):
        a = -1 if i in without else rng.randrange(case["n"])
        ids += [a] * (cuts[i + 1] - cuts[i])
    return ids


def _settings(case):
    """(temperature, top-k, top-p, min-p) of each row; 0, 0, 1, 0 where a setting is off."""
    rng = random.Random(13 * case["B"] + case["V"])
    plain, chat = (1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0)
    if case["mix"] != "mixed":
        return [plain if case["mix"] == "plain" else chat] * case["B"]
    kinds = [plain, chat, (0.0, 0, 1.0, 0.0), (0.6, 0, 0.95, 0.0), (1.0, 50, 1.0, 0.0), (1.3, 0, 1.0, 0.05),
             (0.9, 400, 0.97, 0.02), (1.0, 1, 1.0, 0.0), (2.0, 0, 0.9, 0.0)]
    return [rng.choice(kinds) for _ in range(case["B"])]


def _logits(g, case):
    """What a head gives: a broad middle, a few tokens far above it; every fourth row with most tokens masked
    (-infinity, or the type's lowest value), one row of a larger batch with nothing left."""
    B, V = case["B"], case["V"]
    dtype = F32 if case["f32"] else BF
    x = _randn(g, B, V) * (1.5 + 1.5 * torch.rand(B, 1, generator=g, device=DEV))
    at = torch.randint(0, V, (B, 24), generator=g, device=DEV)
    x.scatter_(1, at, 4.0 + 10.0 * torch.rand(B, 24, generator=g, device=DEV))
    x = x.to(dtype)
    row = torch.arange(B, device=DEV)
    left = torch.rand(B, V, generator=g, device=DEV) < max(200.0 / V, 0.001)
    low = torch.where(row % 8 == 3, -math.inf, torch.finfo(dtype).min).to(dtype)[:, None]
    x = torch.where((row % 4 != 3)[:, None] | left, x, low)
    if B >= 8:
        x[5] = -math.inf
    return x.contiguous()


def prepare(case, seed):
    g, k = _gen(seed), case["kind"]
    s = {"case": case}
    if k == "step":
        rows, P = _lengths(case), case["page"]
        S = case["rows"]
        held = [-(-n // P) for n, _, _ in rows]
        s["n_pages"] = n_pages = sum(held) + case["spare"]
        s["max_pages"] = max_pages = -(-(case["past"] + case["most"]) // P)
        ids = torch.randperm(n_pages, generator=g, device=DEV).to(INT)
        s["pages"] = torch.zeros(S, max_pages, dtype=INT, device=DEV)
        n = torch.tensor(held, device=DEV)
        j = torch.arange(max_pages, device=DEV)[None]
        mine = (n.cumsum(0) - n)[:, None] + j
        s["pages"] = torch.where(j < n[:, None], ids[mine.clamp(max=n_pages - 1)], s["pages"])
        s["free"] = torch.zeros(n_pages, dtype=INT, device=DEV)
        s["free"][:case["spare"]] = ids[sum(held):]
        s["n_free"] = torch.tensor([case["spare"]], dtype=INT, device=DEV)
        s["length"], s["new"], s["done"] = (torch.tensor(c, dtype=INT, device=DEV) for c in zip(*rows))
        for name, size in (("at", case["T"]), ("seq", case["T"]), ("start", S + 1), ("last", S), ("length_out", S),
                           ("n_free_out", 1)):
            s[name] = torch.empty(size, dtype=INT, device=DEV)
        if own:
            s["tables"] = _pkg("tables").PageTables(s["pages"], s["length"], s["free"], s["n_free"], P)
    elif k == "adapt":
        T, R, K, N, n = (case[c] for c in ("T", "R", "K", "N", "n"))
        s["ids"] = torch.tensor(_ids(case), dtype=INT, device=DEV)
        s["x"], s["y"] = _randn(g, T, K).to(BF), _randn(g, T, N).to(BF)
        s["a"] = (_randn(g, n, R, K) / math.sqrt(K)).to(BF)
        s["b"] = (_randn(g, n, N, R) * (0.3 / math.sqrt(R))).to(BF)
        s["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device=DEV)
        s["out"] = torch.empty(T, N, dtype=BF, device=DEV)
        if own:
            adapters = _pkg("adapters")
            s["pool"] = adapters.Adapters(s["a"], s["b"], s["scale"])
            s["ws"] = adapters.adapters_workspace(T, R, device=DEV)
    else:
        B, V = case["B"], case["V"]
        s["logits"] = _logits(g, case)
        s["u"] = torch.rand(B, generator=g, device=DEV)
        heat, top_k, top_p, min_p = zip(*_settings(case))
        s["temperature"], s["top_p"], s["min_p"] = (torch.tensor(c, device=DEV) for c in (heat, top_p, min_p))
        s["top_k"] = torch.tensor(top_k, dtype=INT, device=DEV)
        s["token"], s["logprob"] = torch.empty(B, dtype=torch.int64, device=DEV), torch.empty(B, device=DEV)
        if own:
            sampling = _pkg("sampling")
            s["draw"], s["ws"] = sampling.sample, sampling.sample_workspace(B, V, device=DEV)
    return s


def _pkg(name):
    import importlib

    import __graft_entry__

    __graft_entry__.load_package()
    return importlib.import_module("qwen35_amd." + name)


# ---------------------------------------------------------------- one pass

def run(s):
    k = s["case"]["kind"]
    if k == "step":
        flat = s["case"]["flat"]
        if own:
            s["tables"].step(s["new"], s["at"], seq=s["seq"] if flat else None, done=s["done"],
                             start=s["start"] if flat else None, last=s["last"], length_out=s["length_out"],
                             n_free_out=s["n_free_out"])
        else:
            _step(s)
        out = {n: s[n] for n in ("pages", "free", "at", "last", "length_out", "n_free_out")}
        return dict(out, seq=s["seq"], start=s["start"]) if flat else out
    if k == "adapt":
        if own:
            return s["pool"].add(s["x"], s["ids"], s["y"], s["ws"], out=s["out"])
        return _adapt(s)
    if own:
        s["draw"](s["logits"], s["u"], s["ws"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                  min_p=s["min_p"], out=s["token"], logprob=s["logprob"])
    else:
        _sample(s)
    return {"token": s["token"], "logprob": s["logprob"]}


def _step(s):
    case = s["case"]
    P, S, T, flat, n_pages, max_pages = case["page"], case["rows"], case["T"], case["flat"], s["n_pages"], s["max_pages"]
    over, length = s["done"] != 0, s["length"].long()
    new = s["new"].long().clamp(min=0)
    j = torch.arange(max_pages, device=DEV)[None]
    # pages of rows that are over go on top of the free ones, row after row
    back = torch.where(over, (length + P - 1) // P, 0)
    n_free = s["n_free"].long()
    to = torch.where(j < back[:, None], n_free + (back.cumsum(0) - back)[:, None] + j, n_pages)
    free = torch.cat([s["free"], s["free"].new_zeros(1)])
    free[to.flatten()] = s["pages"].flatten()
    n_free = n_free + back.sum()
    length = torch.where(over, 0, length)
    # who is served, in order: a row that could not be served on its own holds up nobody
    held = (length + P - 1) // P
    tokens = new if flat else new.clamp(max=1)
    need = (length + tokens + P - 1) // P - held
    fits = (length + tokens <= max_pages * P) & (need <= n_free) & (tokens <= T)
    tokens, need = torch.where(fits, tokens, 0), torch.where(fits, need, 0)
    served = (need == 0) | (need.cumsum(0) <= n_free)
    tokens = torch.where(served, tokens, 0)
    if flat:
        served = served & (tokens.cumsum(0) <= T)
        tokens = torch.where(served, tokens, 0)
    need = torch.where(served & (tokens > 0), need, 0)
    # the pages they take, from the top
    first = (need.cumsum(0) - need)[:, None]
    i = j - held[:, None]
    taken = free[(n_free - 1 - first - i).clamp(0, n_pages)]
    s["pages"].copy_(torch.where((i >= 0) & (i < need[:, None]), taken, s["pages"]))
    s["free"].copy_(free[:n_pages])
    s["n_free_out"].copy_(n_free - need.sum())
    s["length_out"].copy_(length + tokens)
    s["last"].copy_(length + tokens - 1)
    if not flat:
        s["at"].copy_(torch.where(tokens > 0, length, -1))
        return
    end = tokens.cumsum(0)
    s["start"].copy_(torch.cat([end.new_zeros(1), end]))
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(end, t, right=True)
    there, b = b < S, b.clamp(max=S - 1)
    s["seq"].copy_(torch.where(there, b, -1))
    s["at"].copy_(torch.where(there, length[b] + t - (end - tokens)[b], -1))


def _adapt(s):
    n, R, K = s["a"].shape
    h = torch.matmul(s["x"].float(), s["a"].float().view(n * R, K).t()).view(-1, n, R)
    mine = s["ids"][:, None] == torch.arange(n, device=DEV)[None]
    h = torch.where(mine[..., None], h * s["scale"][None, :, None], torch.zeros_like(h)).view(-1, n * R)
    b = s["b"].float().transpose(1, 2).reshape(n * R, -1)
    return (s["y"].float() + torch.matmul(h, b)).to(BF)


def _sample(s):
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x + 0.0)     # -0 is 0
    B, V = x.shape
    top = x.amax(-1, keepdim=True)
    heat = s["temperature"].double()[:, None]
    greedy = ~(heat > 0)
    d = (x - top) / torch.where(greedy, 1.0, heat)
    d = torch.where(x == top, 0.0, d)
    w = torch.where(torch.isinf(x) & (x < 0), 0.0, torch.exp(d))
    # sorted: the largest first, equal ones by their index
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    place = torch.arange(V, device=DEV)[None]
    k, p = s["top_k"].long()[:, None], s["top_p"].double()[:, None]
    ws = torch.where((k <= 0) | (place < k), ws, 0.0)
    upto = ws.cumsum(-1)
    before = torch.cat([torch.zeros_like(top), upto[:, :-1]], 1)
    keep = (p >= 1) | (before < p * upto[:, -1:])
    keep = keep & (ws >= s["min_p"].double()[:, None]) | (place == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    upto = kept.cumsum(-1)
    token = (upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(-1, keepdim=True)
    token = torch.where(greedy, order[:, :1], token.clamp(max=V - 1))
    logprob = d.gather(1, token) - torch.log(w.sum(-1, keepdim=True))
    dead = torch.isinf(top) & (top < 0)
    s["token"].copy_(torch.where(dead, -1, token)[:, 0])
    s["logprob"].copy_(torch.where(dead, -math.inf, logprob)[:, 0])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "step":
        P = case["page"]
        rows = _lengths(case)
        moved = sum(-(-n // P) for n, _, over in rows if over) + sum(-(-(n + new) // P) - -(-n // P) for n, new, _ in rows)
        return {"bytes": 4 * (case["rows"] * 6 + case["T"] * (2 if case["flat"] else 1) + 2 * moved),
                "flops": 10 * case["rows"] + case["T"]}
    if case["kind"] == "adapt":
        T, R, K, N = (case[c] for c in ("T", "R", "K", "N"))
        ids = _ids(case)
        n = sum(a >= 0 for a in ids)
        return {"bytes": 2 * n * K + 4 * T * N + 2 * R * (K + N) * len(set(ids) - {-1}) + 4 * T, "flops": 2 * n * R * (K + N)}
    return {"bytes": case["B"] * (case["V"] * (4 if case["f32"] else 2) + 32), "flops": 4 * case["B"] * case["V"]}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_adapt(case, s):
    out = s["y"].double()
    ids = _ids(case)
    for a in sorted(set(ids) - {-1}):
        mine = torch.tensor([t for t, i in enumerate(ids) if i == a], device=DEV)
        h = torch.mm(s["x"][mine].double(), s["a"][a].double().t().contiguous())
        out[mine] += float(s["scale"][a]) * torch.mm(h, s["b"][a].double().t().contiguous())
    return out


def _exact_row(x, u, heat, k, p, least):
    """(token, logarithm of its probability before the filters) of one row of logits."""
    if not bool((x > -math.inf).any()):
        return -1, -math.inf
    if heat <= 0:
        token = int((x == x.max()).nonzero()[0])
        return token, float(x[token] - torch.logsumexp(x, 0))
    x = x / heat
    q = torch.exp(x - torch.logsumexp(x, 0))
    order = torch.argsort(-x, stable=True)
    if k > 0:
        order = order[:k]
    if p < 1:
        c = torch.cumsum(q[order], 0)
        order = order[:1 + int((c[:-1] < p * c[-1]).sum())]
    order = order[(q[order] >= least * q.max()) | (order == order[0])]
    index = torch.sort(order)[0]
    c = torch.cumsum(q[index], 0)
    token = int(index[min(len(index) - 1, int(torch.searchsorted(c, u * c[-1], right=True)))])
    return token, float(x[token] - torch.logsumexp(x, 0))


def exact(case, seed):
    if case["kind"] == "step":
        return None     # whole numbers alone
    s = prepare(case, seed)
    if case["kind"] == "adapt":
        return _exact_adapt(case, s)
    settings = zip(*(s[n].tolist() for n in ("u", "temperature", "top_k", "top_p", "min_p")))
    token, logprob = zip(*(_exact_row(x.double(), *row) for x, row in zip(s["logits"], settings)))
    return {"token": torch.tensor(token, device=DEV), "logprob": torch.tensor(logprob, dtype=torch.float64, device=DEV)}
