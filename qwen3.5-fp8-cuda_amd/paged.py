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
_NO_STRIDE = (0, 0, 1)
# torch.cuda.current_device() and torch.cuda.current_stream(dev).cuda_stream without the Python
# around them, which a decode step's host would spend a microsecond on (a torch without a GPU
# build has neither, and no cache to call them for)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


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
        lib = abi.load()
        self._prep, self._read, self._attend = lib.qh_attn_prep_paged, lib.qh_kv_read_paged, lib.qh_attn_decode_paged

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
        if _current_device() == self.dev:
            rc = fn(*args, _raw_stream(self.dev))
        else:
            with torch.cuda.device(self.dev):
                rc = fn(*args, _raw_stream(self.dev))
        if rc != 0:
            abi.check(rc, what)

    # Each call checks its tensors in one expression, which costs a decode step's host a
    # few microseconds; only where it fails are they gone through one by one, for the message.

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
        dev, D, n_kv = self.dev, self.head_dim, self.n_kv
        kn = k.shape
        T = kn[0] if kn else 0
        H, shape, row = 0, (T, n_kv, D), (T,)
        ks, vs, pn = k.stride(), v.stride(), pages.shape
        good = (k.dtype is _BF and v.dtype is _BF and pages.dtype is _INT and at.dtype is _INT
                and k.get_device() == dev and v.get_device() == dev and pages.get_device() == dev
                and at.get_device() == dev and kn == shape and v.shape == shape and at.shape == row
                and len(pn) == 2 and pages.is_contiguous() and at.is_contiguous()
                and ks[2] == 1 and vs[2] == 1 and (n_kv == 1 or ks[1] == D and vs[1] == D))
        p_seq = p_q = p_out = p_rope = p_pos = p_qn = p_kn = None
        f32 = qs = qh = 0
        if good and seq is not None:
            good = seq.dtype is _INT and seq.get_device() == dev and seq.shape == row and seq.is_contiguous()
            p_seq = seq.data_ptr()
        if good and rope is not None:
            good = (pos is not None and pos.dtype is _INT and pos.get_device() == dev and rope.dev == dev
                    and (pos.shape == (rope.n_axes, T) or rope.n_axes == 1 and pos.shape == row)
                    and pos.is_contiguous())
            p_rope, p_pos = rope._ref, pos.data_ptr() if good else None
        if good and q_norm is not None:
            good = (q_norm.dtype is _F32 and q_norm.get_device() == dev and q_norm.shape == (D,)
                    and q_norm.is_contiguous())
            p_qn = q_norm.data_ptr()
        if good and k_norm is not None:
            good = (k_norm.dtype is _F32 and k_norm.get_device() == dev and k_norm.shape == (D,)
                    and k_norm.is_contiguous())
            p_kn = k_norm.data_ptr()
        if good and q is not None:
            n = q.shape
            good = q.dtype is _BF and q.get_device() == dev and len(n) == 3 and n[0] == T and n[2] == D
            if good:
                H = n[1]
                qs, qh, last = q.stride()
                if q_out is None:
                    q_out = torch.empty(T, H, D, dtype=_BF, device=self.device)
                f32 = q_out.dtype is _F32
                good = (last == 1 and (f32 or q_out.dtype is _BF) and q_out.get_device() == dev and q_out.shape == n
                        and q_out.is_contiguous())
                p_q, p_out = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            good = False
        if not good:
            self._refuse_prep(k, v, pages, at, seq, q, q_out, rope, pos, q_norm, k_norm)
        args = (self._ref, p_rope, p_q, qs, qh, k.data_ptr(), ks[0], v.data_ptr(), vs[0], p_qn, p_kn, eps, p_pos, p_seq,
                at.data_ptr(), T, pages.data_ptr(), pn[0], pn[1], p_out, f32, H, _raw_stream(dev))
        if _current_device() == dev:
            rc = self._prep(*args)
        else:
            with torch.cuda.device(dev):
                rc = self._prep(*args)
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
            if rope.dev != dev:
                raise ValueError(f"rope: must be on cuda:{dev}")
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
        dev, pn, n = self.dev, pages.shape, k_out.shape
        if not (pages.dtype is _INT and last.dtype is _INT and k_out.dtype is _BF and v_out.dtype is _BF
                and pages.get_device() == dev and last.get_device() == dev and k_out.get_device() == dev
                and v_out.get_device() == dev and len(pn) == 2 and last.shape == pn[:1] and len(n) == 4
                and n[0] == pn[0] and n[1] == self.n_kv and n[3] == self.head_dim and v_out.shape == n
                and pages.is_contiguous() and last.is_contiguous() and k_out.is_contiguous()
                and v_out.is_contiguous()):
            B = pn[0]
            _need(pages, "pages", _INT, (None, None), dev)
            _need(last, "last", _INT, (B,), dev)
            _need(k_out, "k_out", _BF, (B, self.n_kv, None, self.head_dim), dev)
            _need(v_out, "v_out", _BF, tuple(n), dev)
            raise ValueError("read: arguments that do not fit together")
        self._call("kv_read_paged", self._read, self._ref, pages.data_ptr(), pn[0], pn[1], last.data_ptr(),
                   k_out.data_ptr(), v_out.data_ptr(), n[2])

    def attend(self, q, pages, last, ws, gate=None, out=None):
        """out[b, h] = softmax(q[b, h] . K^T / sqrt(D)) V over positions 0 .. last[b]
        (int32 [B]) of sequence b, times sigmoid(gate[b, h]) with a gate; zeros for an
        empty sequence (last[b] < 0).  q, gate: bf16 [B, n_heads, D], any strides, q as
        `prep` wrote it; ws: ``attn_workspace`` (calls that share one must not overlap).
        Returns out, bf16 [B, n_heads, D]."""
        dev, n, pn = self.dev, q.shape, pages.shape
        qs = q.stride()
        good = (q.dtype is _BF and pages.dtype is _INT and last.dtype is _INT and ws.dtype is _U8
                and q.get_device() == dev and pages.get_device() == dev and last.get_device() == dev
                and ws.get_device() == dev and len(n) == 3 and n[2] == self.head_dim and len(pn) == 2
                and pn[0] == n[0] and last.shape == n[:1] and qs[2] == 1
                and pages.is_contiguous() and last.is_contiguous() and ws.is_contiguous())
        p_gate, gs = None, _NO_STRIDE
        if good and gate is not None:
            gs = gate.stride()
            good = gate.dtype is _BF and gate.get_device() == dev and gate.shape == n and gs[2] == 1
            p_gate = gate.data_ptr()
        if good and out is not None:
            good = out.dtype is _BF and out.get_device() == dev and out.shape == n and out.is_contiguous()
        if not good:
            B, H = (n[0], n[1]) if len(n) == 3 else (None, None)
            self._need_heads(q, "q", B, None)
            if gate is not None:
                self._need_heads(gate, "gate", B, H)
            _need(pages, "pages", _INT, (B, None), dev)
            _need(last, "last", _INT, (B,), dev)
            _need(ws, "ws", _U8, (None,), dev)
            if out is not None:
                _need(out, "out", _BF, tuple(n), dev)
            raise ValueError("attend: arguments that do not fit together")
        if out is None:
            out = torch.empty(n, dtype=_BF, device=self.device)
        self._call("attn_decode_paged", self._attend, self._ref, q.data_ptr(), qs[0], qs[1], p_gate, gs[0], gs[1],
                   pages.data_ptr(), n[0], pn[1], last.data_ptr(), n[1], out.data_ptr(), ws.data_ptr(), ws.numel())
        return out


def attn_workspace(n_heads, n_kv, head_dim, device="cuda"):
    """A zeroed workspace for `PagedKVCache.attend`, any number of sequences and any length."""
    n = int(abi.load().qh_attn_decode_paged_workspace_size(n_heads, n_kv, head_dim))
    if n == 0:
        raise ValueError(f"attn_workspace: n_heads={n_heads} n_kv={n_kv} head_dim={head_dim} unsupported")
    return torch.zeros(n, dtype=torch.uint8, device=device)
