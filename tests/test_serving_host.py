"""Host-side rules of the serving entry points that need no GPU."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from dslcompiler_b200 import serving  # noqa: E402


class _Stream:
    cuda_stream = 7


def test_what_a_call_makes_is_made_on_its_stream(monkeypatch):
    current = ["torch's"]

    @contextlib.contextmanager
    def stream(s):
        current.append(s)
        yield
        current.pop()

    recorded = []
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: current[-1])
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda raw, device=None: ("raw", raw))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append(s))
    at = []
    for name in ("empty_like", "zeros_like"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda t, real=real, name=name: at.append((name, current[-1])) or real(t))
    q, s = torch.ones(2, 3, 4, 8), _Stream()
    assert (serving._out_like(q, torch.ones(2), s) == 0).all()
    serving._out_like(q, None, 9)
    serving._out_like(q, torch.ones(2), None)
    assert at == [("zeros_like", s), ("empty_like", ("raw", 9)), ("zeros_like", "torch's")]
    assert recorded == ["torch's", "torch's"]
    seen = []
    serving._made_on(s, q.device, lambda: seen.append(current[-1]))
    assert seen == [s] and current == ["torch's"]


def test_window_and_sinks_are_whole_numbers():
    assert serving._ranges(None, 0) == (0, 0)
    assert serving._ranges(7, 3) == (7, 3)
    assert serving._ranges(torch.tensor(7), True) == (7, 1)
    assert serving._ranges(2**70, 2**70) == (2**62, 2**62)
    assert serving._ranges(100.0, 2.0) == (100, 2)
    for window, sinks in ((-1, 0), (0, -1), (0.5, 0), (99.9, 0), (4, 1.5), ("4", 0)):
        with pytest.raises(ValueError):
            serving._ranges(window, sinks)
