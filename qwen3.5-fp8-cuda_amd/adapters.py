"""Low-rank adapters of many requests at once, beside a projection that they share.

The reference runs one request with the checkpoint's weights (main.py:242-279); here each token of a
batch may name an adapter of its own, whose product is added to what ``ops.fp8_linear`` gave for the
whole batch:

  Adapters.add    out[t] = y[t] + scale[i] * b[i] (a[i] x[t]), i = ids[t] (qh_adapters_add)

The call goes on the current torch stream of the adapters' device and allocates nothing but an output
that was not given, so it can be captured in a HIP graph; ids are a device tensor that may change
between replays, and so may the adapters' own values.
"""
import torch

from . import abi
from .paged import _BF, _F32, _INT, _U8, _need, _raw_stream, _serve_host, _with_device


class Adapters:
    """The adapters of one projection.  a: bf16 [n, R, K], b: bf16 [n, N, R], scale: fp32 [n] (for instance
    alpha / rank).  R (at most 128), K and N are multiples of 8; an adapter of a smaller rank has zeros in
    the rows of a (and the columns of b) that it does not use."""

    def __init__(self, a, b, scale):
        dev = a.get_device()
        if dev < 0:
            raise ValueError("Adapters: tensors must be on the GPU (there is no CPU fallback)")
        _need(a, "a", _BF, (None, None, None), dev)
        n, R, K = a.shape
        _need(b, "b", _BF, (n, None, R), dev)
        _need(scale, "scale", _F32, (n,), dev)
        self.a, self.b, self.scale = a, b, scale
        self.n, self.rank, self.K, self.N, self.dev, self.device = n, R, K, b.shape[1], dev, a.device
        self._entry, self._add = abi.address("qh_adapters_add"), _serve_host().add

    def add(self, x, ids, y, ws, out=None):
        """out[t] = y[t] + scale[i] * b[i] (a[i] x[t]) with i = ids[t] (int32 [T]), y[t] where i is outside
        [0, n) (-1: no adapter).  x: bf16 [T, K], y, out: bf16 [T, N], each with a dense last axis and any
        token stride of 8 n (a slice of a fused projection's columns, for instance); out=y adds in place,
        rows without an adapter untouched.  ws: ``adapters_workspace`` for T tokens or more (calls that
        share one must not overlap).  Returns out."""
        if out is None:
            out = torch.empty(y.shape, dtype=_BF, device=self.device)
        rc = _with_device(self.dev, self._add, self._entry, self.dev, self.a, self.b, self.scale, x, ids, y, ws, out,
                          _raw_stream(self.dev))
        if rc is None:
            dev, T = self.dev, x.shape[0] if x.dim() else 0
            for t, name, n, width in ((x, "x", None, self.K), (y, "y", T, self.N), (out, "out", T, self.N)):
                _need(t, name, _BF, (n, width), dev, contiguous=False)
                if t.stride(1) != 1:
                    raise ValueError(f"{name}: the last axis must be contiguous")
            _need(ids, "ids", _INT, (T,), dev)
            _need(ws, "ws", _U8, (None,), dev)
            raise ValueError("add: arguments that do not fit together")
        if rc != 0:
            abi.check(rc, "adapters_add")
        return out


def adapters_workspace(max_tokens, rank, device="cuda"):
    """A workspace for `Adapters.add` of up to max_tokens tokens, whatever the projection's sizes."""
    n = abi.size("qh_adapters_workspace_size", max_tokens, rank)
    if n == 0:
        raise ValueError(f"adapters_workspace: max_tokens={max_tokens} rank={rank} unsupported")
    return torch.empty(n, dtype=torch.uint8, device=device)
