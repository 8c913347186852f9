"""What lies between a paged cache's methods and the native module, which single tokens' calls wait for."""
import sys

import torch

from qwen35_amd import paged


def frames(dev, current, monkeypatch):
    """The Python frames between the caller and the function that launches, outermost first."""
    cache = object.__new__(paged.PagedKVCache)
    cache.dev = dev
    monkeypatch.setattr(paged, "_current_device", lambda: current)
    seen = []

    def launch(*args):
        f = sys._getframe(1)
        while f.f_code is not frames.__code__:
            seen.insert(0, f.f_code.co_name)
            f = f.f_back
        return args
    assert cache._call(launch, 1, "two", 3.0) == (1, "two", 3.0)
    return seen


def test_a_call_is_one_frame(monkeypatch):
    assert frames(3, 3, monkeypatch) == ["_call"]


def test_a_call_on_another_device_makes_it_the_current_one(monkeypatch):
    made = []

    class Device:
        def __init__(self, dev):
            made.append(dev)

        def __enter__(self):
            made.append("in")

        def __exit__(self, *e):
            made.append("out")
    monkeypatch.setattr(torch.cuda, "device", Device)
    assert frames(3, 0, monkeypatch) == ["_call"] and made == [3, "in", "out"]
