"""A token for each row of a batch's logits.

The reference draws for one sequence (main.py:49-87); ``Qwen35FP8Engine.set_sampling`` does the same on the
GPU (qh_sample_top_p).  Here every row of a batch has settings and a random number of its own:

  sample    temperature, top-k, top-p and min-p, drawn with given random numbers (qh_sample_rows)

The call goes on the current torch stream of the logits' device and allocates nothing but an output that was
not given, so it can be captured in a HIP graph; settings and random numbers are device tensors that may
change between replays.
"""
import torch

from . import abi
from .paged import _BF, _F32, _INT, _U8, _need, _raw_stream, _serve_host, _with_device

_entry = _sample = None


def sample(logits, u, ws, temperature=None, top_k=None, top_p=None, min_p=None, out=None, logprob=None):
    """The tokens int64 [B] of logits [B, V] (bf16 or fp32, a dense last axis, any row stride),
    for instance what qh_lm_head_rows gives, drawn with the random numbers u (fp32 [B], of [0, 1)).

    Per row, over weights exp((x - max x) / temperature) in falling order of the logits (equal ones by
    index): the first `top_k` (int32; 0 or below: all), of those the ones before which less than
    `top_p` (fp32; 1 or above: all) of their weight lies, of those the ones of at least `min_p` (fp32; 0 or
    below: all) of the largest weight; the first always.  The token is the first kept index whose running
    sum in index order is above u times the whole.  temperature (fp32; 0 or below: the largest logit,
    the first of equal ones) and the others are [B], None: 1, all, all, all.  NaN counts as -infinity; a row
    with nothing else has token -1.  logprob: fp32 [B], where the logarithm of the token's weight over
    those of all logits, before any filter, goes (at temperature 1 for the largest logit).

    ws: ``sample_workspace`` for B rows and V logits or more (calls that share one must not overlap).
    Without top_k, top_p and min_p (None, not tensors of what switches them off) two launches of four do."""
    global _entry, _sample
    if _entry is None:
        _entry, _sample = abi.address("qh_sample_rows"), _serve_host().sample
    dev = logits.get_device()
    if dev < 0:
        raise ValueError("sample: tensors must be on the GPU (there is no CPU fallback)")
    if out is None:
        out = torch.empty(logits.shape[:1], dtype=torch.int64, device=logits.device)
    rc = _with_device(dev, _sample, _entry, dev, logits, u, ws, temperature, top_k, top_p, min_p, out, logprob,
                      _raw_stream(dev))
    if rc is None:
        if logits.dtype not in (_BF, _F32):
            raise TypeError(f"logits: bf16 or fp32, got {logits.dtype}")
        _need(logits, "logits", logits.dtype, (None, None), dev, contiguous=False)
        if logits.stride(1) != 1:
            raise ValueError("logits: the last axis must be contiguous")
        B = len(logits)
        for t, name, dtype in ((u, "u", _F32), (temperature, "temperature", _F32), (top_k, "top_k", _INT), (top_p, "top_p", _F32),
                               (min_p, "min_p", _F32), (out, "out", torch.int64), (logprob, "logprob", _F32)):
            if t is not None or name == "u":
                _need(t, name, dtype, (B,), dev)
        _need(ws, "ws", _U8, (None,), dev)
        raise ValueError("sample: arguments that do not fit together")
    if rc != 0:
        abi.check(rc, "sample_rows")
    return out


def sample_workspace(rows, vocab, device="cuda"):
    """A workspace for `sample` of up to so many rows and logits a row."""
    n = abi.size("qh_sample_rows_workspace_size", rows, vocab)
    if n == 0:
        raise ValueError(f"sample_workspace: rows={rows} vocab={vocab} unsupported")
    return torch.empty(n, dtype=torch.uint8, device=device)
