"""Paged KV cache of the full-attention layers, for several sequences at once.

The reference serves one sequence from a dense bf16 cache (main.py:1034-1059), as
``Qwen35FP8Engine`` does; here a layer's cache is a pool of pages that page tables
share out among sequences, in bf16 or in E4M3 with an fp32 scale per token and head:

  PagedKVCache.prep    tokens written: head norm, rotary positions on one or several
                       axes (RopeAxes), quantisation, q handed on (qh_attn_prep_paged)
  PagedKVCache.read    a sequence's rows as a dense bf16 cache (qh_kv_read_paged)
  PagedKVCache.attend  attention of one new token a sequence (qh_attn_decode_paged)

A decode step of a layer is ``prep`` and ``attend``; a prompt is ``prep`` with an fp32
``q_out``, ``read`` and the prompt attention ``qh_attn_prefill`` over what it wrote.
Every call goes on the current torch stream of the cache's device and allocates
nothing but an output that was not given, so it can be captured in a HIP graph; page
tables, positions and lengths are device tensors that may change between replays.
"""
import ctypes

import torch

from . import abi

FP8 = torch.float8_e4m3fn
_INT, _BF, _F32, _U8 = torch.int32, torch.bfloat16, torch.float32, torch.uint8
# torch.cuda.current_device() and torch.cuda.current_stream(dev).cuda_stream without the Python
# around them, which a decode step's host would spend a microsecond on (a torch without a GPU
# build has neither, and no cache to call them for)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _host():
    """The extension module that checks and launches the calls (csrc/paged_host.cpp)."""
    try:
        from . import _paged_host
    except ImportError as e:
        raise ImportError("_paged_host.so does not load: build it with `python qwen3.5-fp8-cuda_amd/build.py`") from e
    return _paged_host


def _serve_host():
    """The extension module that checks and launches a serving step's calls (csrc/serve_host.cpp)."""
    try:
        from . import _serve_host
    except ImportError as e:
        raise ImportError("_serve_host.so does not load: build it with `python qwen3.5-fp8-cuda_amd/build.py`") from e
    return _serve_host


def _with_device(dev, fn, *args):
    """Launch with `dev` as the current device."""
    if _current_device() == dev:
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _need(t, name, dtype, shape, dev, contiguous=True):
    """Raise unless t is a `dtype` tensor of `shape` (None: any size) on GPU `dev`."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: expects {dtype}, got {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name}: must be on cuda:{dev}")
    if len(t.shape) != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape} (None: any size)")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")


class RopeAxes:
    """Rotary positions on `len(sections)` axes.  cos, sin: fp32 [max_pos, rot] as
    ``engine.rope_tables`` gives them; sections: how many of the rot/2 pairs each axis
    turns, one after the other, or with `interleaved` in turn (pair i on axis
    i % axes while that axis has pairs left, otherwise on the first)."""

    def __init__(self, cos, sin, sections=None, interleaved=False):
        dev = cos.get_device()
        if dev < 0:
            raise ValueError("RopeAxes: tables must be on the GPU")
        _need(cos, "cos", torch.float32, (None, None), dev)
        _need(sin, "sin", torch.float32, tuple(cos.shape), dev)
        sections = [cos.shape[1] // 2] if sections is None else [int(s) for s in sections]
        if not 1 <= len(sections) <= 4:
            raise ValueError("RopeAxes: 1 to 4 sections")
        self.cos, self.sin, self.sections, self.interleaved = cos, sin, sections, bool(interleaved)
        self.n_axes, self.dev = len(sections), dev
        self._desc = abi.RopeAxesDesc(cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.shape[1],
                                      len(sections), int(self.interleaved),
                                      (ctypes.c_int * 4)(*sections, *([0] * (4 - len(sections)))))
        self._ref = ctypes.addressof(self._desc)


class PagedKVCache:
    """One layer's pages.  k, v: [n_pages, n_kv, page_size, head_dim], bf16, or
    float8_e4m3fn with k_scale, v_scale: fp32 [n_pages, n_kv, page_size]."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        dev = k.get_device()
        if dev < 0:
            raise ValueError("PagedKVCache: tensors must be on the GPU (there is no CPU fallback)")
        if k.dtype not in (_BF, FP8):
            raise TypeError(f"PagedKVCache: bf16 or float8_e4m3fn pages, got {k.dtype}")
        _need(k, "k", k.dtype, (None,) * 4, dev)
        _need(v, "v", k.dtype, tuple(k.shape), dev)
        self.fp8 = k.dtype == FP8
        if self.fp8 != (k_scale is not None) or self.fp8 != (v_scale is not None):
            raise ValueError("PagedKVCache: scales belong to an E4M3 cache, and to every one")
        if self.fp8:
            _need(k_scale, "k_scale", torch.float32, tuple(k.shape[:3]), dev)
            _need(v_scale, "v_scale", torch.float32, tuple(k.shape[:3]), dev)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv, self.page_size, self.head_dim = k.shape
        self.dev, self.device = dev, k.device
        self._desc = abi.PagedCacheDesc(k.data_ptr(), v.data_ptr(),
                                        k_scale.data_ptr() if self.fp8 else None,
                                        v_scale.data_ptr() if self.fp8 else None,
                                        self.n_pages, self.page_size, self.n_kv, self.head_dim, int(self.fp8))
        self._ref = ctypes.addressof(self._desc)
        lib, host = abi.load(), _host()
        entries = (lib.qh_attn_prep_paged, lib.qh_kv_read_paged, lib.qh_attn_decode_paged)
        self._prep_at, self._read_at, self._attend_at = (ctypes.cast(f, ctypes.c_void_p).value for f in entries)
        self._prep, self._read, self._attend = host.prep, host.read, host.attend

    @classmethod
    def alloc(cls, n_pages, page_size, n_kv, head_dim, dtype=_BF, device="cuda"):
        """A zeroed pool."""
        shape = (n_pages, n_kv, page_size, head_dim)
        kv = [torch.zeros(shape, dtype=torch.uint8 if dtype == FP8 else dtype, device=device) for _ in range(2)]
        if dtype != FP8:
            return cls(*kv)
        return cls(*(t.view(FP8) for t in kv), *(torch.zeros(shape[:3], device=device) for _ in range(2)))

    # The native module checks a call's tensors and launches it; it hands back None where one
    # does not fit, and only then are they gone through one by one, for the message.

    def _call(self, fn, *args):
        """Launch with the cache's device as the current one (`_with_device` without a second frame, whose packing of
        the arguments is a twentieth of a single token's call)."""
        if _current_device() == self.dev:
            return fn(*args)
        with torch.cuda.device(self.dev):
            return fn(*args)

    def prep(self, k, v, pages, at, seq=None, q=None, q_out=None, rope=None, pos=None, q_norm=None, k_norm=None,
             eps=1e-6):
        """Write T tokens: k, v bf16 [T, n_kv, D] (heads dense, any token stride of 8 n) to
        position at[t] (int32 [T]) of sequence seq[t] (int32 [T]; None: token t is
        sequence t's), pages int32 [n_seqs, max_pages].  q bf16 [T, n_heads, D] (any
        strides of 8 n, for instance the q half of interleaved q | gate rows) goes through the
        same norm and rotation to q_out [T, n_heads, D], bf16 (what `attend` takes; the
        default) or fp32 (what qh_attn_prefill takes: not rounded behind the norm, so it multiplies
        the low halves of all dimensions, 13 % longer at 3700 tokens than for the dense path's q, which is
        bf16 in the dimensions that are not turned).  rope: RopeAxes with pos int32
        [axes, T] (or [T] for one axis).  A token with an index out of range (padding:
        -1) is left out altogether.  Returns q_out."""
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=_BF, device=self.device)
        if rope is not None and rope.dev != self.dev:
            raise ValueError(f"rope: must be on cuda:{self.dev}")
        rc = self._call(self._prep, self._prep_at, self._ref, self.dev, 0 if rope is None else rope._ref, k, v, pages, at,
                        seq, q, q_out, pos, q_norm, k_norm, eps, _raw_stream(self.dev))
        if rc is None:
            self._refuse_prep(k, v, pages, at, seq, q, q_out, rope, pos, q_norm, k_norm)
        if rc != 0:
            abi.check(rc, "attn_prep_paged")
        return q_out

    def _refuse_prep(self, k, v, pages, at, seq, q, q_out, rope, pos, q_norm, k_norm):
        """Raise for the first argument of `prep` that it does not take."""
        D, dev, T = self.head_dim, self.dev, k.shape[0] if k.dim() else 0
        for t, name in ((k, "k"), (v, "v")):
            self._need_heads(t, name, T, self.n_kv)
            if self.n_kv > 1 and t.stride(1) != D:
                raise ValueError(f"{name}: a token's heads must be contiguous")
        _need(pages, "pages", _INT, (None, None), dev)
        _need(at, "at", _INT, (T,), dev)
        if seq is not None:
            _need(seq, "seq", _INT, (T,), dev)
        if rope is not None:
            if pos is None:
                raise ValueError("rope: needs pos")
            _need(pos, "pos", _INT, (T,) if pos.dim() == 1 and rope.n_axes == 1 else (rope.n_axes, T), dev)
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None:
                _need(w, name, _F32, (D,), dev)
        if q is None:
            raise ValueError("q_out: there is no q")
        self._need_heads(q, "q", T, None)
        if q_out.dtype not in (_BF, _F32):
            raise TypeError("q_out: bf16 or fp32")
        _need(q_out, "q_out", q_out.dtype, tuple(q.shape), dev)
        raise ValueError("prep: arguments that do not fit together")

    def _need_heads(self, t, name, n, heads):
        """Raise unless t is a bf16 [n, heads, head_dim] view whose last axis is dense."""
        _need(t, name, _BF, (n, heads, self.head_dim), self.dev, contiguous=False)
        if t.stride(2) != 1:
            raise ValueError(f"{name}: the last axis must be contiguous")

    def read(self, pages, last, k_out, v_out):
        """Positions 0 .. last[b] (int32 [B]) of each sequence to k_out, v_out bf16
        [B, n_kv, max_seq, D]; rows behind them keep what they hold."""
        rc = self._call(self._read, self._read_at, self._ref, self.dev, pages, last, k_out, v_out, _raw_stream(self.dev))
        if rc is None:
            dev = self.dev
            _need(pages, "pages", _INT, (None, None), dev)
            B = len(pages)
            _need(last, "last", _INT, (B,), dev)
            _need(k_out, "k_out", _BF, (B, self.n_kv, None, self.head_dim), dev)
            _need(v_out, "v_out", _BF, tuple(k_out.shape), dev)
            raise ValueError("read: arguments that do not fit together")
        if rc != 0:
            abi.check(rc, "kv_read_paged")

    def attend(self, q, pages, last, ws, gate=None, out=None):
        """out[b, h] = softmax(q[b, h] . K^T / sqrt(D)) V over positions 0 .. last[b]
        (int32 [B]) of sequence b, times sigmoid(gate[b, h]) with a gate; zeros for an
        empty sequence (last[b] < 0).  q, gate: bf16 [B, n_heads, D], any strides of 8 n, q as
        `prep` wrote it; ws: ``attn_workspace`` (calls that share one must not overlap).
        Returns out, bf16 [B, n_heads, D]."""
        if out is None:
            out = torch.empty(q.shape, dtype=_BF, device=self.device)
        rc = self._call(self._attend, self._attend_at, self._ref, self.dev, q, pages, last, ws, gate, out,
                        _raw_stream(self.dev))
        if rc is None:
            dev = self.dev
            self._need_heads(q, "q", None, None)
            B, H = q.shape[:2]
            if gate is not None:
                self._need_heads(gate, "gate", B, H)
            _need(pages, "pages", _INT, (B, None), dev)
            _need(last, "last", _INT, (B,), dev)
            _need(ws, "ws", _U8, (None,), dev)
            _need(out, "out", _BF, tuple(q.shape), dev)
            raise ValueError("attend: arguments that do not fit together")
        if rc != 0:
            abi.check(rc, "attn_decode_paged")
        return out


def attn_workspace(n_heads, n_kv, head_dim, device="cuda"):
    """A zeroed workspace for `PagedKVCache.attend`, any number of sequences and any length."""
    n = int(abi.load().qh_attn_decode_paged_workspace_size(n_heads, n_kv, head_dim))
    if n == 0:
        raise ValueError(f"attn_workspace: n_heads={n_heads} n_kv={n_kv} head_dim={head_dim} unsupported")
    return torch.zeros(n, dtype=torch.uint8, device=device)
