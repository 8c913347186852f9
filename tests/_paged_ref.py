"""The paged cache's operators written out in 64 bits on the CPU, token by token."""
import math

import torch

MIN_SCALE = 2.0 ** -100


def axes_of(half, sections, interleaved):
    """The axis of each of the `half` rotary pairs."""
    n = len(sections)
    if not interleaved:
        return [a for a in range(n) for _ in range(sections[a])]
    return [i % n if i < n * sections[i % n] else 0 for i in range(half)]


def head_norm(x, w, eps=1e-6):
    x = x.double()
    if w is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1.0 + w.double())


def rotate(x, cos, sin, pos, axes):
    """x [T, H, D] (64 bits), pos [n_axes, T], axes: the axis of each pair."""
    half = len(axes)
    if half == 0:
        return x
    y = x.clone()
    for i, a in enumerate(axes):
        c, s = cos[pos[a].long(), i].double()[:, None], sin[pos[a].long(), i].double()[:, None]
        y[..., i] = x[..., i] * c - x[..., i + half] * s
        y[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return y


def pair_size(x, half):
    """|x_c| + |its partner| for rotated dimensions, |x_c| elsewhere: what an fp32
    rotation's error is relative to."""
    a = x.abs()
    y = a.clone()
    y[..., :half] = a[..., :half] + a[..., half:2 * half]
    y[..., half:2 * half] = y[..., :half]
    return y


def gather(x, scale, table, b, n, page):
    """Rows 0 .. n-1 of sequence b [n_kv, n, D] in 64 bits and which of them lie on a
    page that exists [n]."""
    j = torch.arange(n)
    ids = table[b].long()[j // page]
    ok = (ids >= 0) & (ids < x.shape[0])
    ids = ids.clamp(0, x.shape[0] - 1)
    y = x[ids, :, j % page].double()                       # [n, n_kv, D]
    if scale is not None:
        y = y * scale[ids, :, j % page].double()[..., None]
    return y.transpose(0, 1), ok


def attend(q, k, v, ks, vs, table, last, gate=None):
    """(out [B, H, D], bound [B, H, 1]): the attention in 64 bits, and how far fp32
    arithmetic may move an output before it is rounded.  A score is a sum of D fp32
    products, scaled twice: off by at most e = (D + 4) 2^-24 sum|q_i k_i| / sqrt(D);
    a weight e^(s - m) is then off by the factor 1 + 2 e + 2^-20 (the exponential and the
    weight's own split into two bf16 parts, 2^-17 of it, once more), in the numerator and
    in the sum, and no value is above max|v|."""
    B, H, D = q.shape
    page, n_kv = k.shape[2], k.shape[1]
    out = torch.zeros(B, H, D, dtype=torch.float64)
    tol = torch.zeros(B, H, 1, dtype=torch.float64)
    for b in range(B):
        n = min(int(last[b]) + 1, table.shape[1] * page)
        if n <= 0:
            continue
        kk, ok = gather(k, ks, table, b, n, page)
        vv, _ = gather(v, vs, table, b, n, page)
        kk, vv = kk[:, ok], vv[:, ok]
        if not kk.shape[1]:
            continue
        for h in range(H):
            g = h // (H // n_kv)
            prod = kk[g] * q[b, h].double()
            p = torch.softmax(prod.sum(-1) / math.sqrt(D), -1)
            out[b, h] = p @ vv[g]
            e = (D + 4) * 2.0 ** -24 * float(prod.abs().sum(-1).max()) / math.sqrt(D)
            tol[b, h] = 2 * (2 * e + 2.0 ** -20 + 2.0 ** -17) * float(vv[g].abs().max())
    if gate is not None:
        sg = torch.sigmoid(gate.double())
        out = out * sg
        tol = tol * sg + 2.0 ** -20 * out.abs()
    return out, tol
