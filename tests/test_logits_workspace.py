"""Whose memory the Python binding's workspaces of logits are: of the pool of the stream that the call runs on, where a
block given back on return cannot be handed to work that is not ordered with the call's kernels."""
import contextlib

import pytest
import torch

import gonngpu as G

DEFAULT, LIBRARY, MINE, OTHER = 0, 4096, 8192, 12288  # handles; the binding does not look behind them


@pytest.mark.parametrize("current,asked,pool", [
    (DEFAULT, None, "current"), (DEFAULT, 0, LIBRARY), (DEFAULT, OTHER, OTHER), (DEFAULT, LIBRARY, LIBRARY),
    (MINE, None, "current"), (MINE, 0, LIBRARY), (MINE, MINE, "current"), (MINE, OTHER, OTHER),
    (LIBRARY, 0, "current"), (LIBRARY, LIBRARY, "current"), (LIBRARY, None, "current")])
def test_pool_of_the_workspace(monkeypatch, current, asked, pool):
    """Handle 0 asked for is the library's own stream, never torch's default one, whose handle is 0 as well."""
    used = []

    @contextlib.contextmanager
    def on(stream):
        used.append(stream)
        yield

    monkeypatch.setattr(G, "_current_stream", lambda device=None: current)
    monkeypatch.setattr(G, "stream", lambda: LIBRARY)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: handle)
    monkeypatch.setattr(torch.cuda, "stream", on)
    for dtype in (torch.float32, torch.float16):
        for k in (0, 20):
            used.clear()
            ws, n = G._logits_workspace(torch.zeros((1, 8), dtype=dtype), 1, 1 << 20, k, 0, asked)
            assert used == ([] if pool == "current" else [pool])
            assert ws.numel() * ws.element_size() == n == G.load().gn_logits_workspace(1, 1 << 20, k)


@pytest.mark.gpu
@pytest.mark.parametrize("distill", [False, True])
def test_library_stream_with_the_default_stream_current(dev, monkeypatch, distill):
    """The workspace is none of the default stream's blocks: allocations there, overwritten at once, do not meet it, and the
    results are right."""
    rows, cols, k = 3, 300000, 20
    g = torch.Generator().manual_seed(1)
    x = torch.randn((rows, cols), generator=g).to(dev)
    t = torch.tensor([1, 2, 3], device=dev)
    ids0, teacher = torch.randint(0, cols, (rows, 6), generator=g).to(dev), torch.randn((rows, 6), generator=g).to(dev)
    new = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=dev)  # noqa: E731
    lp, lse, ids, tops = new(rows), new(rows), new(rows, k, dtype=torch.int64), new(rows, k)

    def call(stream_ptr):
        if distill:
            G.distill(x, ids0, teacher, lp, lse=lse, stream_ptr=stream_ptr)
        else:
            G.token_logprobs(x, t, lp, lse=lse, top_ids=ids, top_logprobs=tops, stream_ptr=stream_ptr)

    call(None)
    torch.cuda.synchronize()
    want = [v.clone() for v in (lp, lse, ids, tops)]
    at = []
    real = G.call

    def spy(name, *args):
        if name in ("gn_token_logprobs", "gn_distill_forward"):
            at.append((args[-3], args[-2]))  # workspace, bytes
        return real(name, *args)

    monkeypatch.setattr(G, "call", spy)
    for v in (lp, lse, ids, tops):
        v.zero_()
    with torch.cuda.stream(torch.cuda.default_stream()):
        torch.empty((64 << 20,), dtype=torch.uint8, device=dev)  # the default stream's pool has something to give
        torch.cuda.synchronize()
        call(0)
        ws, n = at[0]
        blocks = [torch.full((n // 4,), float("nan"), device=dev) for _ in range(8)]
        assert n > 0 and all(b.data_ptr() + n <= ws or ws + n <= b.data_ptr() for b in blocks)
        G.synchronize()
    torch.cuda.synchronize()
    for a, b in zip((lp, lse, ids, tops), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("current,asked,where", [
    (DEFAULT, None, 0), (DEFAULT, 0, 0), (MINE, 0, 0), (MINE, None, 1), (DEFAULT, MINE, 1)])
def test_library_stream_on_another_gpu(monkeypatch, current, asked, where):
    """A call that would run on the library's stream is refused for tensors of another GPU than that stream's; a stream of theirs is
    used as it is."""
    ran = []
    monkeypatch.setattr(G, "_current_stream", lambda device=None: current)
    monkeypatch.setattr(G, "library_device", lambda: 0, raising=False)
    monkeypatch.setattr(G, "call", lambda name, *args: ran.append(args[-1]))
    monkeypatch.setattr(G, "_run_ordered", lambda name, *args: ran.append("ordered"))
    G._dispatch_on(0, asked, "gn_mxfp4_quantize", 5)
    assert ran == ["ordered" if current == DEFAULT and asked is None else asked if asked is not None else current]
    ran.clear()
    if where == 1:
        G._dispatch_on(1, asked, "gn_mxfp4_quantize", 5)
        assert ran == [asked or current]
    else:
        with pytest.raises(G.GonngpuError, match="library's stream is on GPU 0"):
            G._dispatch_on(1, asked, "gn_mxfp4_quantize", 5)
        assert ran == []
