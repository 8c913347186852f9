"""Adapters of many requests: what the entry point refuses before anything touches a GPU, and what the host
module hands on."""
import ctypes

import pytest
import torch

from qwen35_amd import _serve_host, abi, adapters

P = [ctypes.c_void_p(1 << 20 | 4096 * k) for k in range(12)]
BF, INT = torch.bfloat16, torch.int32
T, K, N, R, A = 5, 64, 48, 16, 3


def call(**kw):
    a = dict(a=P[0], b=P[1], scale=P[2], n=A, R=R, K=K, N=N, x=P[3], x_ts=K, ids=P[4], T=T, y=P[5], y_ts=N, out=P[6], o_ts=N,
             ws=P[7], ws_bytes=1 << 30)
    a.update(kw)
    return abi.load().qh_adapters_add(*a.values(), None)


@pytest.mark.parametrize("bad,said", [
    (dict(n=0), "n_adapters=0"), (dict(R=0), "rank=0"), (dict(R=12), "rank=12"), (dict(R=136), "rank at most 128"),
    (dict(K=0), "K=0"), (dict(K=60), "K=60"), (dict(N=0), "N=0"), (dict(N=44), "N=44"), (dict(N=-8), "N=-8"),
    (dict(T=-1), "T=-1"), (dict(T=2**20 - 63), "at most 1048512"), (dict(a=None), "null"), (dict(b=None), "null"),
    (dict(scale=None), "null"), (dict(x=None), "null"), (dict(ids=None), "null"), (dict(y=None), "null"), (dict(out=None), "null"),
    (dict(ws=None), "null"), (dict(a=ctypes.c_void_p(4104)), "aligned"), (dict(x=ctypes.c_void_p(4098)), "aligned"),
    (dict(y=ctypes.c_void_p(4104)), "aligned"), (dict(x_ts=K + 4), "multiples of 8"), (dict(o_ts=N + 1), "multiples of 8"),
    (dict(out=P[3]), "alias"), (dict(out=P[5], o_ts=N + 8), "alias"), (dict(o_ts=0), "overlap"), (dict(o_ts=N - 8), "overlap"),
    (dict(ws=ctypes.c_void_p(4096 + 64)), "256-byte"), (dict(ws_bytes=100), "workspace")])
def test_refusals(bad, said):
    assert call(**bad) == -1
    assert "adapters_add" in abi.last_error() and said in abi.last_error()


@pytest.mark.parametrize("bad", [dict(K=2**30 + 8), dict(K=2**31 - 8), dict(N=2**30 + 8, y_ts=2**30 + 8, o_ts=2**30 + 8),
                                 dict(N=2**31 - 8, y_ts=2**31 - 8, o_ts=2**31 - 8)])
def test_projections_whose_columns_32_bits_do_not_count(bad):
    assert call(T=1, **bad) == -1
    assert "at most 2^30" in abi.last_error()


def test_nothing_to_do_launches_nothing():
    assert call(T=0) == 0


def test_workspace_size():
    size = abi.load().qh_adapters_workspace_size
    for bad in [(-1, 16), (2**20 - 63, 16), (5, 0), (5, 12), (5, 136)]:
        assert size(*bad) == 0
        with pytest.raises(ValueError):
            adapters.adapters_workspace(*bad)
    last = 0
    for n in [0, 1, 2, 100, 1023, 1024, 1025, 5000, 8191, 8192, 8193, 20000, 2**20 - 64]:
        assert size(n, 24) >= last            # a workspace for more tokens serves fewer
        assert size(n, 24) == size(n, 32)     # ranks go sixteen at a time
        last = size(n, 24)
    assert call(ws_bytes=size(T, R)) != -1 or "workspace" not in abi.last_error()


def host(args, status=0):
    seen = []
    rest, types = abi.NATIVE_SIGNATURES["qh_adapters_add"]

    def record(*a):
        seen.append(a)
        return status
    f = ctypes.CFUNCTYPE(rest, *types)(record)
    got = _serve_host.add(ctypes.cast(f, ctypes.c_void_p).value, -1, *args)
    return got, (seen[0] if seen else None)


def args(**kw):
    wide = torch.zeros(T, 2 * N + 16, dtype=BF)
    a = dict(a=torch.zeros(A, R, K, dtype=BF), b=torch.zeros(A, N, R, dtype=BF), scale=torch.zeros(A),
             x=torch.zeros(T, K + 8, dtype=BF)[:, :K], ids=torch.zeros(T, dtype=INT), y=wide[:, 8:N + 8],
             ws=torch.zeros(99, dtype=torch.uint8), out=torch.zeros(T, N, dtype=BF), stream=77)
    a.update(kw)
    return a


def test_host_hands_on_pointers_strides_and_sizes():
    a = args()
    p = {k: t.data_ptr() for k, t in a.items() if isinstance(t, torch.Tensor)}
    got, s = host(a.values(), status=-1)
    assert got == -1
    assert s == (p["a"], p["b"], p["scale"], A, R, K, N, p["x"], K + 8, p["ids"], T, p["y"], 2 * N + 16, p["out"], N, p["ws"],
                 99, 77)
    one = torch.zeros(1, N, dtype=BF).as_strided((1, N), (3, 1))      # one token: its stride is not read
    got, s = host(args(x=torch.zeros(1, K, dtype=BF), ids=torch.zeros(1, dtype=INT), y=one, out=one).values())
    assert got == 0 and s[8] == s[12] == s[14] == 0


@pytest.mark.parametrize("bad", [
    dict(a=torch.zeros(A, R, K)), dict(a=torch.zeros(A, K, R, dtype=BF).transpose(1, 2)), dict(a=torch.zeros(R, K, dtype=BF)),
    dict(b=torch.zeros(A, N, R + 8, dtype=BF)), dict(b=torch.zeros(A + 1, N, R, dtype=BF)), dict(b=None),
    dict(scale=torch.zeros(A, dtype=BF)), dict(scale=torch.zeros(A + 1)), dict(x=torch.zeros(T, K)), dict(x=None),
    dict(x=torch.zeros(T, K + 8, dtype=BF)), dict(x=torch.zeros(K, T, dtype=BF).t()), dict(x=torch.zeros(1, T, K, dtype=BF)),
    dict(ids=torch.zeros(T, dtype=torch.int64)), dict(ids=torch.zeros(T + 1, dtype=INT)), dict(ids=[0] * T),
    dict(y=torch.zeros(T, N + 8, dtype=BF)), dict(y=torch.zeros(T, 2 * N, dtype=BF)[:, ::2]), dict(y=torch.zeros(T + 1, N, dtype=BF)),
    dict(out=torch.zeros(T, N)), dict(out=None), dict(out=torch.zeros(N, T, dtype=BF).t()), dict(ws=torch.zeros(99)),
    dict(ws=None), dict(y=torch.zeros(T, N, dtype=BF, device="meta"))], ids=lambda b: next(iter(b)))
def test_host_leaves_a_misfit_to_the_caller(bad):
    assert host(args(**bad).values()) == (None, None)


def test_wrapper_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="GPU"):
        adapters.Adapters(torch.zeros(A, R, K, dtype=BF), torch.zeros(A, N, R, dtype=BF), torch.zeros(A))
