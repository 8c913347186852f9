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
_INT = torch.int32
_BF = torch.bfloat16


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
        self.lib = abi.load()
        self._desc = abi.PagedCacheDesc(k.data_ptr(), v.data_ptr(),
                                        k_scale.data_ptr() if self.fp8 else None,
                                        v_scale.data_ptr() if self.fp8 else None,
                                        self.n_pages, self.page_size, self.n_kv, self.head_dim, int(self.fp8))
        self._ref = ctypes.addressof(self._desc)

    @classmethod
    def alloc(cls, n_pages, page_size, n_kv, head_dim, dtype=_BF, device="cuda"):
        """A zeroed pool."""
        shape = (n_pages, n_kv, page_size, head_dim)
        kv = [torch.zeros(shape, dtype=torch.uint8 if dtype == FP8 else dtype, device=device) for _ in range(2)]
        if dtype != FP8:
            return cls(*kv)
        return cls(*(t.view(FP8) for t in kv), *(torch.zeros(shape[:3], device=device) for _ in range(2)))

    def _call(self, what, fn, *args):
        """Launch on the current stream of the cache's device."""
        if torch.cuda.current_device() == self.dev:
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        else:
            with torch.cuda.device(self.dev):
                rc = fn(*args, torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            abi.check(rc, what)

    def _heads(self, t, name, n, heads):
        """Strides (first, second) of a bf16 [n, heads, head_dim] view whose last axis is dense."""
        _need(t, name, _BF, (n, heads, self.head_dim), self.dev, contiguous=False)
        a, b, c = t.stride()
        if c != 1:
            raise ValueError(f"{name}: the last axis must be contiguous")
        return a, b

    def prep(self, k, v, pages, at, seq=None, q=None, q_out=None, rope=None, pos=None, q_norm=None, k_norm=None,
             eps=1e-6):
        """Write T tokens: k, v bf16 [T, n_kv, D] (heads dense, any token stride) to
        position at[t] (int32 [T]) of sequence seq[t] (int32 [T]; None: token t is
        sequence t's), pages int32 [n_seqs, max_pages].  q bf16 [T, n_heads, D] (any
        strides, for instance the q half of interleaved q | gate rows) goes through the
        same norm and rotation to q_out [T, n_heads, D], bf16 (what `attend` takes; the
        default) or fp32 (what qh_attn_prefill takes).  rope: RopeAxes with pos int32
        [axes, T] (or [T] for one axis).  A token with an index out of range (padding:
        -1) is left out altogether.  Returns q_out."""
        D, dev = self.head_dim, self.dev
        T = k.shape[0]
        ks, kh = self._heads(k, "k", T, self.n_kv)
        vs, vh = self._heads(v, "v", T, self.n_kv)
        if T > 0 and self.n_kv > 1 and (kh != D or vh != D):
            raise ValueError("k, v: a token's heads must be contiguous")
        _need(pages, "pages", _INT, (None, None), dev)
        _need(at, "at", _INT, (T,), dev)
        if seq is not None:
            _need(seq, "seq", _INT, (T,), dev)
        if rope is not None:
            if rope.dev != dev:
                raise ValueError(f"rope: must be on cuda:{dev}")
            if pos is None:
                raise ValueError("rope: needs pos")
            _need(pos, "pos", _INT, (T,) if pos.dim() == 1 and rope.n_axes == 1 else (rope.n_axes, T), dev)
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None:
                _need(w, name, torch.float32, (D,), dev)
        H = qs = qh = 0
        if q is not None:
            H = q.shape[1]
            qs, qh = self._heads(q, "q", T, H)
            if q_out is None:
                q_out = torch.empty(T, H, D, dtype=_BF, device=self.device)
            elif q_out.dtype not in (_BF, torch.float32):
                raise TypeError("q_out: bf16 or fp32")
            _need(q_out, "q_out", q_out.dtype, (T, H, D), dev)
        elif q_out is not None:
            raise ValueError("q_out: there is no q")
        self._call("attn_prep_paged", self.lib.qh_attn_prep_paged, self._ref, None if rope is None else rope._ref,
                   None if q is None else q.data_ptr(), qs, qh, k.data_ptr(), ks, v.data_ptr(), vs,
                   None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps,
                   None if pos is None else pos.data_ptr(), None if seq is None else seq.data_ptr(), at.data_ptr(), T,
                   pages.data_ptr(), pages.shape[0], pages.shape[1], None if q is None else q_out.data_ptr(),
                   int(q is not None and q_out.dtype == torch.float32), H)
        return q_out

    def read(self, pages, last, k_out, v_out):
        """Positions 0 .. last[b] (int32 [B]) of each sequence to k_out, v_out bf16
        [B, n_kv, max_seq, D]; rows behind them keep what they hold."""
        _need(pages, "pages", _INT, (None, None), self.dev)
        B = pages.shape[0]
        _need(last, "last", _INT, (B,), self.dev)
        _need(k_out, "k_out", _BF, (B, self.n_kv, None, self.head_dim), self.dev)
        _need(v_out, "v_out", _BF, tuple(k_out.shape), self.dev)
        self._call("kv_read_paged", self.lib.qh_kv_read_paged, self._ref, pages.data_ptr(), B, pages.shape[1],
                   last.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), k_out.shape[2])

    def attend(self, q, pages, last, ws, gate=None, out=None):
        """out[b, h] = softmax(q[b, h] . K^T / sqrt(D)) V over positions 0 .. last[b]
        (int32 [B]) of sequence b, times sigmoid(gate[b, h]) with a gate; zeros for an
        empty sequence (last[b] < 0).  q, gate: bf16 [B, n_heads, D], any strides, q as
        `prep` wrote it; ws: ``attn_workspace`` (calls that share one must not overlap).
        Returns out, bf16 [B, n_heads, D]."""
        B, H = q.shape[0], q.shape[1]
        qs, qh = self._heads(q, "q", B, H)
        gs = gh = 0
        if gate is not None:
            gs, gh = self._heads(gate, "gate", B, H)
        _need(pages, "pages", _INT, (B, None), self.dev)
        _need(last, "last", _INT, (B,), self.dev)
        _need(ws, "ws", torch.uint8, (None,), self.dev)
        if out is None:
            out = torch.empty(B, H, self.head_dim, dtype=_BF, device=self.device)
        else:
            _need(out, "out", _BF, (B, H, self.head_dim), self.dev)
        self._call("attn_decode_paged", self.lib.qh_attn_decode_paged, self._ref, q.data_ptr(), qs, qh,
                   None if gate is None else gate.data_ptr(), gs, gh, pages.data_ptr(), B, pages.shape[1],
                   last.data_ptr(), H, out.data_ptr(), ws.data_ptr(), ws.numel())
        return out


def attn_workspace(n_heads, n_kv, head_dim, device="cuda"):
    """A zeroed workspace for `PagedKVCache.attend`, any number of sequences and any length."""
    n = int(abi.load().qh_attn_decode_paged_workspace_size(n_heads, n_kv, head_dim))
    if n == 0:
        raise ValueError(f"attn_workspace: n_heads={n_heads} n_kv={n_kv} head_dim={head_dim} unsupported")
    return torch.zeros(n, dtype=torch.uint8, device=device)
