"""Sampling by row: what the entry point refuses before anything touches a GPU, what the host module hands on,
and the definition itself in closed form."""
import ctypes
import math

import pytest
import torch

import _sample_ref as ref
from qwen35_amd import _serve_host, abi, sampling

P = [ctypes.c_void_p(1 << 20 | 4096 * k) for k in range(12)]
BF, INT = torch.bfloat16, torch.int32


def call(**kw):
    a = dict(x=P[0], stride=100, f32=0, B=3, V=100, u=P[1], heat=P[2], k=P[3], p=P[4], m=P[5], token=P[6], lp=P[7], ws=P[8],
             ws_bytes=1 << 40)
    a.update(kw)
    return abi.load().qh_sample_rows(*a.values(), None)


@pytest.mark.parametrize("bad,said", [
    (dict(B=-1), "rows=-1"), (dict(B=65536), "65535"), (dict(V=0), "vocab=0"), (dict(V=2**20 + 1), "1048576"),
    (dict(x=None), "null"), (dict(u=None), "null"), (dict(token=None), "null"), (dict(ws=None), "null"),
    (dict(x=ctypes.c_void_p(4097)), "aligned"), (dict(x=ctypes.c_void_p(4098), f32=1), "aligned"),
    (dict(ws=ctypes.c_void_p(4096 + 64)), "256-byte"), (dict(ws_bytes=1000), "workspace")])
def test_refusals(bad, said):
    assert call(**bad) == -1
    assert "sample_rows" in abi.last_error() and said in abi.last_error()


def test_nothing_to_do_launches_nothing():
    assert call(B=0) == 0


def test_workspace_size():
    size = abi.load().qh_sample_rows_workspace_size
    for bad in [(-1, 5), (65536, 5), (3, 0), (3, 2**20 + 1)]:
        assert size(*bad) == 0
        with pytest.raises(ValueError):
            sampling.sample_workspace(*bad)
    for V in (1, 8192, 8193, 248320):
        assert size(1, V) <= size(2, V) <= size(100, V)
    for B in (1, 64):
        assert size(B, 1) <= size(B, 8192) <= size(B, 8193) <= size(B, 50257) <= size(B, 2**20)
    assert size(0, 5) > 0


def host(args, status=0):
    seen = []
    rest, types = abi.NATIVE_SIGNATURES["qh_sample_rows"]

    def record(*a):
        seen.append(a)
        return status
    f = ctypes.CFUNCTYPE(rest, *types)(record)
    got = _serve_host.sample(ctypes.cast(f, ctypes.c_void_p).value, -1, *args)
    return got, (seen[0] if seen else None)


def args(**kw):
    a = dict(logits=torch.zeros(3, 110, dtype=BF)[:, 3:103], u=torch.zeros(3), ws=torch.zeros(99, dtype=torch.uint8),
             temperature=torch.zeros(3), top_k=torch.zeros(3, dtype=INT), top_p=torch.zeros(3), min_p=torch.zeros(3),
             out=torch.zeros(3, dtype=torch.int64), logprob=torch.zeros(3), stream=77)
    a.update(kw)
    return a


def test_host_hands_on_pointers_strides_and_sizes():
    a = args()
    p = {k: t.data_ptr() for k, t in a.items() if isinstance(t, torch.Tensor)}
    got, s = host(a.values(), status=-1)
    assert got == -1
    assert s == (p["logits"], 110, 0, 3, 100, p["u"], p["temperature"], p["top_k"], p["top_p"], p["min_p"], p["out"],
                 p["logprob"], p["ws"], 99, 77)
    got, s = host(args(logits=torch.zeros(1, 100).expand(3, 100), temperature=None, top_k=None, top_p=None, min_p=None,
                       logprob=None).values())
    assert got == 0 and s[1:3] == (0, 1) and s[6:10] == (None,) * 4 and s[11] is None


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(logits=torch.zeros(3, 100, dtype=torch.float16)), dict(logits=torch.zeros(100, dtype=BF)),
    dict(logits=torch.zeros(100, 3, dtype=BF).t()), dict(logits=torch.zeros(4, 100, dtype=BF)), dict(u=None),
    dict(u=torch.zeros(3, dtype=torch.float64)), dict(u=torch.zeros(4)), dict(ws=torch.zeros(99)), dict(temperature=torch.zeros(2)),
    dict(top_k=torch.zeros(3)), dict(top_k=torch.zeros(3, dtype=torch.int64)), dict(top_p=torch.zeros(3, 1)),
    dict(min_p=torch.zeros(6)[::2]), dict(out=torch.zeros(3, dtype=INT)), dict(out=None), dict(logprob=torch.zeros(3, dtype=BF)),
    dict(temperature=0.7), dict(logits=torch.zeros(3, 100, dtype=BF, device="meta"))], ids=lambda b: next(iter(b)))
def test_host_leaves_a_misfit_to_the_caller(bad):
    assert host(args(**bad).values()) == (None, None)


def test_wrapper_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="GPU"):
        sampling.sample(torch.zeros(3, 100, dtype=BF), torch.zeros(3), torch.zeros(99, dtype=torch.uint8))


def test_definition():
    """Weights 4, 2, 1, 1 of 8 in an order of their own: what each filter leaves, drawn at every eighth."""
    x = torch.tensor([1.0, 4.0, 1.0, 2.0]).log()

    def tokens(**kw):
        return [ref.row(x, (i + 0.5) / 8, **kw)[0] for i in range(8)]
    assert tokens() == [0, 1, 1, 1, 1, 2, 3, 3]
    assert tokens(k=2) == [1] * 5 + [3] * 3
    assert tokens(k=3) == [0] + [1] * 5 + [3] * 2          # of the equal ones the first
    assert tokens(p=0.4) == [1] * 8
    assert tokens(p=0.7) == tokens(k=2)
    assert tokens(p=0.8) == tokens(k=3)
    assert tokens(m=0.4) == tokens(k=2)
    assert tokens(k=2, p=0.6) == [1] * 8                   # 4 of the 6 that top-k leaves, not of 8
    assert tokens(heat=0) == [1] * 8
    assert ref.row(x, 0.3)[1] == pytest.approx(math.log(0.5))
    assert ref.row(x, 0.3, heat=0)[1] == pytest.approx(math.log(0.5))
    assert ref.row(x * 2, 0.0, heat=2.0)[1] == pytest.approx(math.log(0.125))
    assert ref.row(torch.full((4,), -math.inf), 0.5)[0] == -1
