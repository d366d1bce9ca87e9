"""Logits adjusted in their own place, and gradients in theirs, without a mask: only the tokens' columns are read and written.
Against int8_ref.py, bit for bit; everything else has to stay as it was."""
import pytest
import torch

import gonngpu as G
from tests import int8_ref as R
from tests.test_adjust_gpu import _case, _on, _same, _say

pytestmark = pytest.mark.gpu

# Histories of a few tokens, of more than a thread's first four (1024 and 4096 to a workgroup), around the border of 1024.
SIZES = [(1, 1, 1, 1), (2, 40, 3, 0), (3, 33, 600, 5), (2, 2049, 300, 64), (3, 5000, 1023, 0), (3, 5000, 1024, 30), (2, 8193, 1025, 1024), (4, 20011, 4097, 9),
         (1, 20011, 9000, 300), (1, 40000, 70000, 7), (300, 130, 60, 3), (70, 9000, 50, 2)]


def _gradient(x, seed=9):
    return torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).to(x.dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,h,nb", SIZES)
def test_forward(dev, rows, cols, h, nb, dtype):
    _say("in place", rows, cols, h, nb, dtype)
    c = _case(rows, cols, h, nb, dtype, 2, share=None)
    want = R.adjust(**c)
    d = _on(dev, c)
    x = d.pop("x")
    G.adjust_logits(x, x, **d)
    assert _same(x, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,h,nb", SIZES)
def test_backward(dev, rows, cols, h, nb, dtype):
    _say("in place, gradient", rows, cols, h, dtype)
    c = _case(rows, cols, h, 0, dtype, 3, share=None)
    g, back = _gradient(c["x"]), {k: c[k] for k in ("history", "repetition")}
    d = _on(dev, back)
    x = c["x"].to(dev)
    for keys in (("history", "repetition"), ("history",), ()):
        dx = g.to(dev)
        G.adjust_logits_backward(x, dx, dx, **{k: d[k] for k in keys})
        assert _same(dx, R.adjust_grad(c["x"], g, **{k: back[k] for k in keys}))
        assert torch.equal(x.cpu(), c["x"])
    G.adjust_logits_backward(x, x, x, **d)  # the logits as their own gradient
    assert _same(x, R.adjust_grad(c["x"], c["x"], **back))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("h", [1, 2000, 9000])
def test_one_token_over_and_over(dev, dtype, h):
    """Put right once."""
    x = torch.linspace(-2, 2, 300).repeat(3, 1).to(dtype)
    history = torch.full((3, h), 299)
    history[1], history[2] = 0, -1
    g, back = _gradient(x), dict(history=history, repetition=torch.tensor([1.7, 0.6, 3.0]))
    dx = g.to(dev)
    G.adjust_logits_backward(x.to(dev), dx, dx, **_on(dev, back))
    assert _same(dx, R.adjust_grad(x, g, **back))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("cols,h", [(2501, 70), (9001, 1500)])
def test_strided_rows_at_odd_addresses(dev, cols, h, dtype):
    rows = 6
    c = _case(rows, cols, h, 11, dtype, 4, share=None)
    g, back = _gradient(c["x"]), {k: c[k] for k in ("history", "repetition")}
    d = _on(dev, c)
    d.pop("x")

    def put(t):
        base = torch.full((2 * rows + 1, cols + 6), 3.0, dtype=dtype, device=dev)
        view = base[1:2 * rows:2, 5:5 + cols]
        view.copy_(t)
        return base, view

    (xb, x), (gb, dx) = put(c["x"]), put(g)
    G.adjust_logits_backward(x, dx, dx, **{k: d[k] for k in back})
    G.adjust_logits(x, x, **d)
    for got, base, ref in ((x, xb, R.adjust(**c)), (dx, gb, R.adjust_grad(c["x"], g, **back))):
        assert _same(got, ref)
        got.fill_(3.0)
        assert bool((base == 3.0).all()), "a value outside the rows was written"


@pytest.mark.parametrize("h", [50, 1500])
def test_captured_and_replayed(dev, h):
    rows, cols = 5, 9000
    c = _case(rows, cols, h, 10, torch.float16, 5, share=None)
    d = _on(dev, c)
    x = d.pop("x")
    back = {k: d[k] for k in ("history", "repetition")}
    g, y, dx = _gradient(c["x"]).to(dev), torch.empty_like(x), torch.empty_like(x)

    def step():
        y.copy_(x)
        dx.copy_(g)
        G.adjust_logits_backward(x, dx, dx, **back)
        G.adjust_logits(y, y, **d)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        new = _case(rows, cols, h, 10, torch.float16, 6 + i, share=None)
        x.copy_(new["x"])
        for k in d:
            d[k].copy_(new[k])
        y.zero_()
        dx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert _same(y, R.adjust(**new))
        assert _same(dx, R.adjust_grad(new["x"], g.cpu(), **{k: new[k] for k in back}))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_most_rows(dev, dtype, in_place):
    """As many rows as one call takes: every one of them, by its own tokens and penalty."""
    rows = 2**24 - 1
    x = (torch.arange(rows, device=dev) % 17 - 8.0)[:, None].to(dtype)
    history = (torch.arange(rows, device=dev) % 3 - 1)[:, None].contiguous()  # none, the column, one past the last
    rho = torch.full((rows,), 2.0, device=dev)
    want = torch.where(history == 0, torch.where(x > 0, x / 2, x * 2), x)
    g = (torch.arange(rows, device=dev) % 5 - 2.0)[:, None].to(dtype)
    want_g = torch.where(history == 0, torch.where(x > 0, g / 2, g * 2), g)
    dx = g.clone() if in_place else torch.full_like(g, 7.0)
    G.adjust_logits_backward(x, dx if in_place else g, dx, history=history, repetition=rho)
    assert torch.equal(dx, want_g)
    out = x if in_place else torch.full_like(x, 7.0)
    G.adjust_logits(x, out, history=history, repetition=rho)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_penalty_is_rounded_before_the_next_is_taken_off(dev, dtype, in_place):
    """x rho needs more than 24 bits and nearly equals the frequency's n: what is left shows whether it was rounded."""
    cols, e = 64, 2.0**-11
    x = torch.full((1, cols), -(1 + e)).to(dtype)
    rho = torch.tensor([1 + 2.0**-23])
    history = torch.arange(cols)[None]
    c = dict(history=history, repetition=rho, frequency=torch.tensor([-(1 + e)]))
    if dtype == torch.float16:
        x = torch.full((1, cols), -(1 + 2.0**-10), dtype=dtype)
        c["frequency"] = torch.tensor([-(1 + 2.0**-10)])
    want = R.adjust(x, **c)
    d = x.to(dev)
    out = d if in_place else torch.empty_like(d)
    G.adjust_logits(d, out, **_on(dev, c))
    assert _same(out, want)
