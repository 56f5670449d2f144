"""Outputs that a call makes for itself are allocated on the stream that writes them (CPU: torch's streams, the library and
the tensors are stand-ins)."""
import contextlib
import ctypes

import pytest
import torch

import nllb_attn as na


class Stand:
    """What the binding asks of a CUDA tensor."""
    device, is_cuda = torch.device("cuda:0"), True

    def __init__(self, shape, dtype, seen):
        self.shape = (shape,) if isinstance(shape, int) else tuple(shape)
        self.dtype, self.seen = dtype, seen

    def get_device(self):
        return 0

    def data_ptr(self):
        return 1 << 20

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return torch.Size(self.shape).numel()

    def stride(self, i=None):
        s = tuple(torch.Size(self.shape[j + 1:]).numel() for j in range(len(self.shape)))
        return s if i is None else s[i]

    def new_empty(self, shape, dtype):
        self.seen["made"].append(self.seen["current"])
        return Stand(shape, dtype, self.seen)


@pytest.fixture
def seen(monkeypatch):
    seen = {"current": "current", "made": [], "ran": []}

    class Lib:
        def __getattr__(self, name):
            def call(*a):
                if name.endswith("_bytes"):
                    return 100
                if name != "nllb_linear_free":
                    seen["ran"].append(a[-1])
                return na.OK
            return call

    @contextlib.contextmanager
    def stream(s):
        before, seen["current"] = seen["current"], s
        yield
        seen["current"] = before

    monkeypatch.setattr(na, "load", lambda *a: Lib())
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: handle)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(na, "current_stream", lambda device=0: 77)
    monkeypatch.setitem(na._types(), "stream", lambda device: 77)
    monkeypatch.setitem(na._types(), "current", lambda: 0)
    # (new_empty is the only way by which the binding may make a tensor here)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (seen["made"].append(seen["current"]), Stand(a[0], kw["dtype"], seen))[1])
    return seen


def calls(seen):
    x, w = Stand((3, 64), torch.float16, seen), Stand((5, 64), torch.float16, seen)
    logits, u = Stand((3, 100), torch.float32, seen), Stand((3,), torch.float32, seen)
    target = Stand((3,), torch.int32, seen)
    prepared = na.PreparedLinear(w, u)
    seen["ran"].clear()
    return {"linear16": (1, lambda **kw: na.linear16(x, w, **kw)),
            "logprobs": (4, lambda **kw: na.logprobs(logits, target, top_n=2, **kw)),
            "sample": (2, lambda **kw: na.sample(logits, u, **kw)),
            "logsoftmax_topk": (3, lambda **kw: na.logsoftmax_topk(logits, 8, **kw)),
            "linear_int8": (1, lambda **kw: na.linear_int8(x, w, u, **kw)),
            "prepared": (1, lambda **kw: prepared(x, **kw))}


NAMES = ["linear16", "logprobs", "sample", "logsoftmax_topk", "linear_int8", "prepared"]
DEFAULT = NAMES[3:]  # without a stream on the legacy default one


@pytest.mark.parametrize("name", NAMES)
def test_made_on_the_named_stream(seen, name):
    n, call = calls(seen)[name]
    for stream in (4096, ctypes.c_void_p(4096)):
        seen["made"].clear()
        call(stream=stream)
        assert seen["made"] == [4096] * n and seen["current"] == "current"
        assert seen["ran"].pop() is stream


@pytest.mark.parametrize("name", NAMES)
def test_the_current_stream_named(seen, name):
    n, call = calls(seen)[name]
    call(stream=77)
    assert seen["made"] == ["current"] * n and seen["ran"] == [77]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("stream", [0, 1])
def test_the_legacy_default_stream(seen, name, stream):
    n, call = calls(seen)[name]
    call(stream=stream)
    assert seen["made"] == ["default"] * n and seen["ran"] == [stream]


@pytest.mark.parametrize("name", NAMES)
def test_no_stream(seen, name):
    """Made and run on torch's current one, or both on the legacy default one."""
    n, call = calls(seen)[name]
    call()
    assert seen["made"] == ["default" if name in DEFAULT else "current"] * n
    assert seen["ran"] == [None if name in DEFAULT else 77]


@pytest.mark.parametrize("name", DEFAULT)
def test_the_default_stream_is_the_current_one(seen, name, monkeypatch):
    monkeypatch.setitem(na._types(), "stream", lambda device: 0)
    n, call = calls(seen)[name]
    call()
    assert seen["made"] == ["current"] * n and seen["ran"] == [None]
