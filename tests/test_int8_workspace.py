"""Whose memory the Python binding's workspace of int8_linear is: of the pool of the stream that the call runs on, given back
after the call's launches whatever becomes of them."""
import contextlib

import pytest
import torch

import gonngpu as G

DEFAULT, LIBRARY, MINE, OTHER = 0, 4096, 8192, 12288  # handles; the binding does not look behind them


def _linear(stream_ptr=None, rows=40):
    w = G.int8_empty(5, 100, device="cpu")
    G.int8_linear(torch.zeros((rows, 100)), w, torch.zeros((rows, 5)), stream_ptr=stream_ptr)


@pytest.fixture
def allocator(monkeypatch):
    """Stands in for torch's allocator, the streams and the library's calls; keeps what happened."""
    seen = []
    monkeypatch.setattr(G, "_device_of", lambda *t: 0)
    monkeypatch.setattr(G, "stream", lambda: LIBRARY)
    monkeypatch.setattr(G, "library_device", lambda: 0)
    G._types()
    monkeypatch.setattr(G, "_alloc", lambda n, s: seen.append(("alloc", n, s)) or 1 << 20)
    monkeypatch.setattr(G, "_free", lambda p: seen.append(("free", p)))
    monkeypatch.setattr(G, "call", lambda name, *a: seen.append((name, a[-3], a[-2], a[-1])))
    monkeypatch.setattr(G, "_run_ordered", lambda name, *a: seen.append((name, a[-2], a[-1], "ordered")))
    return seen


@pytest.mark.parametrize("current,asked,pool,runs", [
    (DEFAULT, None, DEFAULT, "ordered"), (DEFAULT, 0, LIBRARY, 0), (DEFAULT, OTHER, OTHER, OTHER), (MINE, None, MINE, MINE),
    (MINE, 0, LIBRARY, 0), (MINE, MINE, MINE, MINE), (MINE, OTHER, OTHER, OTHER), (LIBRARY, 0, LIBRARY, 0)])
def test_pool_of_the_workspace(allocator, monkeypatch, current, asked, pool, runs):
    """Handle 0 asked for is the library's own stream, never torch's default one, whose handle is 0 as well."""
    monkeypatch.setattr(G, "_current_stream", lambda device=None: current)
    _linear(asked)
    n = G.load().gn_int8_linear_workspace(40, 5, 100)
    assert n > 0 and allocator == [("alloc", n, pool), ("gn_int8_linear", 1 << 20, n, runs), ("free", 1 << 20)]


def test_a_call_that_needs_none_has_none(allocator, monkeypatch):
    monkeypatch.setattr(G, "_current_stream", lambda device=None: MINE)
    _linear(rows=1)
    assert G.load().gn_int8_linear_workspace(1, 5, 100) == 0 and allocator == [("gn_int8_linear", None, 0, MINE)]


def test_given_back_after_a_refusal(allocator, monkeypatch):
    monkeypatch.setattr(G, "_current_stream", lambda device=None: MINE)

    def refused(*_):
        raise G.GonngpuError(-1, "refused")

    monkeypatch.setattr(G, "call", refused)
    with pytest.raises(G.GonngpuError):
        _linear()
    assert [e[0] for e in allocator] == ["alloc", "free"]


@pytest.mark.parametrize("current,asked,pool", [(DEFAULT, None, "current"), (DEFAULT, 0, LIBRARY), (MINE, OTHER, OTHER), (MINE, MINE, "current")])
def test_without_the_allocators_functions_a_tensor(allocator, monkeypatch, current, asked, pool):
    used = []

    @contextlib.contextmanager
    def on(stream):
        used.append(stream)
        yield

    monkeypatch.setattr(G, "_alloc", None)
    monkeypatch.setattr(G, "_current_stream", lambda device=None: current)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: handle)
    monkeypatch.setattr(torch.cuda, "stream", on)
    _linear(asked)
    (name, ws, n, _), = allocator
    assert name == "gn_int8_linear" and ws and n == G.load().gn_int8_linear_workspace(40, 5, 100)
    assert used == ([] if pool == "current" else [pool])


@pytest.mark.gpu
def test_blocks_on_the_gpu(dev):
    """Calls on two streams at once, again and again, and the memory is all given back."""
    x, w = torch.randn((300, 700), device=dev), G.int8_empty(200, 700, device=dev)
    G.int8_quantize(torch.randn((200, 700), device=dev), *w)
    want, ys = torch.empty((300, 200), device=dev), [torch.empty((300, 200), device=dev) for _ in range(2)]
    G.int8_linear(x, w, want)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            G.int8_linear(x, w, ys[i % 2])
    G.int8_linear(x, w, want, stream_ptr=streams[0].cuda_stream)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    assert torch.equal(ys[0], want) and torch.equal(ys[1], want)
