"""Sampling by row in 64 bits: the definition, and how near the draw came to another token."""
import math

import torch


def row(x, u, heat=1.0, k=0, p=1.0, m=0.0):
    """(token, log-probability before the filters, margin) of one row of logits (a CPU tensor).

    margin: the least distance of a decision to its border, as a share of the weight that it is taken in (of the
    kept weight for the draw, of what top-k leaves for top-p, of the largest weight for min-p); 0 on it."""
    x = x.double()
    x = torch.where(x.isnan(), -math.inf, x) + 0.0
    heat, p, m, u = (float(torch.tensor(v, dtype=torch.float32)) for v in (heat, p, m, u))
    top = float(x.max()) if len(x) else -math.inf
    if top == -math.inf:
        return -1, -math.inf, 1.0
    greedy = not heat > 0
    t = 1.0 if greedy else heat
    d = torch.where(x == top, 0.0, (x - top) / t)
    w = torch.where(x == -math.inf, 0.0, d.exp())
    logw = lambda i: float(d[i] - w.sum().log())   # noqa: E731
    if greedy:
        i = int((x == top).nonzero()[0])
        return i, logw(i), 1.0
    order = torch.sort(x, descending=True, stable=True)[1]
    margin = 1.0
    if k > 0:
        order = order[:k]
    if not p >= 1:
        ws = w[order]
        upto = ws.cumsum(0)
        before = torch.cat([upto.new_zeros(1), upto[:-1]])
        inside = before < p * upto[-1]
        inside[0] = True
        live = (ws > 0) & (torch.arange(len(ws)) > 0)       # a border counts where a weight lies behind it
        if bool(live.any()):
            margin = min(margin, float((before - p * upto[-1]).abs()[live].min() / upto[-1]))
        order = order[inside]
    if not m <= 0:
        inside = w[order] >= m
        inside[0] = True
        below = order[x[order] < top]                       # the largest's weight is 1, not near it
        if len(below):
            margin = min(margin, float((w[below] - m).abs().min()))
        order = order[inside]
    index = order.sort()[0]
    c = w[index].cumsum(0)
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    at = int((c <= u * c[-1]).sum())
    live = w[index] > 0
    if at >= len(index):
        at = int(live.nonzero()[-1])
    if 0 < u < 1:
        margin = min(margin, float((c - u * c[-1]).abs()[live].min() / c[-1]))
    return int(index[at]), logw(index[at]), margin
