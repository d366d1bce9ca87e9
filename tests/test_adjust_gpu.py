"""Logits adjusted before sampling, and their gradient, against int8_ref.py, whose steps round in fp32 as the definition's do:
all values have to be equal bit for bit."""
import math

import pytest
import torch

import gonngpu as G
from tests import int8_ref as R

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


def _words(rows, cols, share, seed):
    g = torch.Generator().manual_seed(seed)
    words = -(-cols // 32)
    bits = torch.rand((rows, words, 32), generator=g) < share
    w = (bits.long() << torch.arange(32)).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def _case(rows, cols, h, nb, dtype, seed=0, share=0.5):
    g = torch.Generator().manual_seed(rows * cols + h + seed)
    c = {"x": (3 * torch.randn((rows, cols), generator=g)).to(dtype)}
    ids = torch.randint(-2, cols + 2, (rows, h), generator=g)  # some stand for no token
    ids = torch.where(torch.rand((rows, h), generator=g) < 0.4, ids % max(1, cols // 20), ids)  # some occur often
    c["history"] = ids
    c["prompt"] = torch.randint(-1, h + 2, (rows,), generator=g)
    c["repetition"] = 0.7 + torch.rand(rows, generator=g)
    c["frequency"], c["presence"] = torch.rand(rows, generator=g) - 0.3, torch.rand(rows, generator=g) - 0.3
    if nb:
        c["bias_ids"] = torch.randint(-1, cols + 1, (rows, nb), generator=g)
        c["bias"] = 5 * torch.randn((rows, nb), generator=g)
    if share is not None:
        c["mask"] = _words(rows, cols, share, seed)
        c["mask"][rows // 2] = 0  # nothing is left of this row
        c["x"][rows // 2, 0] = math.nan
    return c


def _on(dev, c):
    return {k: v.to(dev) for k, v in c.items()}


def _same(a, b):
    a, b = a.cpu().float(), b.cpu().float()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=9e9), torch.nan_to_num(b, nan=9e9))


SIZES = [(1, 1, 1, 1), (1, 7, 3, 0), (3, 31, 40, 2), (2, 32, 1, 5), (4, 33, 600, 0), (2, 2047, 100, 9), (3, 2048, 257, 0), (2, 2049, 300, 64),
         (1, 5000, 2000, 300), (5, 8191, 30, 0), (1, 20011, 5000, 1024), (70, 130, 60, 3), (600, 100, 40, 2), (520, 8300, 20, 1), (1, 40000, 70000, 7)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,h,nb", SIZES)
def test_adjust(dev, rows, cols, h, nb, dtype):
    _say("adjust", rows, cols, h, nb, dtype)
    if rows * cols > 1000000 and dtype == torch.float32:
        rows = 515
    c = _case(rows, cols, h, nb, dtype)
    want = R.adjust(**c)
    d = _on(dev, c)
    out = torch.full((rows, cols), 7.0, dtype=dtype, device=dev)
    G.adjust_logits(d.pop("x"), out, **d)
    assert _same(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("keys", [(), ("mask",), ("history", "repetition"), ("history", "frequency"), ("history", "prompt", "presence"),
                                  ("history", "prompt"), ("bias",), ("bias", "mask"), ("history", "repetition", "mask")])
@pytest.mark.parametrize("in_place", [False, True])
def test_parts_of_it(dev, keys, dtype, in_place):
    rows, cols = 3, 4100
    c = _case(rows, cols, 90, 20, dtype, 1)
    if "bias" in keys:
        keys = keys + ("bias_ids",)
    c = {k: v for k, v in c.items() if k == "x" or k in keys}
    want = R.adjust(**c)
    d = _on(dev, c)
    x = d.pop("x")
    out = x if in_place else torch.full((rows, cols), 7.0, dtype=dtype, device=dev)
    G.adjust_logits(x, out, **d)
    assert _same(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_one_token_over_and_over(dev, dtype, in_place):
    """A history of one token, biases of one token in an order that shows, and no token at all."""
    rows, cols, h = 3, 300, 5000
    x = torch.linspace(-2, 2, cols).repeat(rows, 1).to(dtype)
    history = torch.full((rows, h), 299)
    history[1], history[2] = 0, -1
    bias_ids = torch.full((rows, 6), 17)
    bias = torch.tensor([1e8, 1.0, -1e8, 3.0, 0.5, 1e-3]).repeat(rows, 1) * (1 if dtype == torch.float32 else 1e-4)
    kw = dict(history=history, prompt=torch.tensor([10, 5000, 0]), repetition=torch.full((rows,), 1.3), frequency=torch.full((rows,), 0.01),
              presence=torch.full((rows,), 0.4), bias_ids=bias_ids, bias=bias)
    want = R.adjust(x, **kw)
    xd = x.to(dev)
    out = xd if in_place else torch.empty_like(xd)
    G.adjust_logits(xd, out, **_on(dev, kw))
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cols,h,nb", [(40, 0, 64), (40, 300, 65), (300, 1023, 700), (300, 1024, 700), (2500, 100, 1024), (9000, 1100, 1024), (9000, 5000, 257)])
def test_many_biases_of_few_tokens(dev, cols, h, nb, dtype, in_place):
    """Tokens with many biases each beside tokens with one, in all of a workgroup's rounds; the sums in their order."""
    _say("biases", cols, h, nb, dtype, in_place)
    c = _case(3, cols, h, nb, dtype, 5, share=None)
    g = torch.Generator().manual_seed(nb)
    c["bias_ids"][:, ::3] = torch.randint(0, min(cols, 9), c["bias_ids"][:, ::3].shape, generator=g) * (cols // 9)
    c["bias"] = c["bias"] * 10.0 ** torch.randint(-3, 3, c["bias"].shape, generator=g)
    want = R.adjust(**c)
    d = _on(dev, c)
    x = d.pop("x")
    out = x if in_place else torch.empty_like(x)
    G.adjust_logits(x, out, **d)
    assert _same(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_infinities_and_nan(dev, dtype):
    """Where they are masked -inf, else what the arithmetic gives; the type's lowest value is a number as others."""
    low = torch.finfo(dtype).min
    x = torch.tensor([[math.inf, -math.inf, math.nan, low, 0.0, -0.0, 1.0, low] * 5] * 2).to(dtype)
    history = torch.tensor([[0, 1, 2, 3, 4, 5, 8, 9, 10, 11]] * 2)
    mask = torch.tensor([[0x00FF00FF, 0x0F], [0, 0]], dtype=torch.int32)
    kw = dict(history=history, repetition=torch.tensor([0.5, 1.5]), presence=torch.tensor([1.0, 1.0]), mask=mask)
    out = torch.zeros_like(x, device=dev)
    G.adjust_logits(x.to(dev), out, **_on(dev, kw))
    assert _same(out, R.adjust(x, **kw)) and bool(torch.isneginf(out[1]).all())
    g = x.flip(1)
    dx = torch.zeros_like(x, device=dev)
    back = {k: kw[k] for k in ("history", "repetition", "mask")}
    G.adjust_logits_backward(x.to(dev), g.to(dev), dx, **_on(dev, back))
    assert _same(dx, R.adjust_grad(x, g, **back)) and bool((dx[1] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,h,nb", [s for s in SIZES if s[0] * s[1] < 1000000])
def test_backward(dev, rows, cols, h, nb, dtype):
    _say("adjust backward", rows, cols, h, dtype)
    c = _case(rows, cols, h, 0, dtype)
    g = torch.randn((rows, cols), generator=torch.Generator().manual_seed(9)).to(dtype)
    back = {k: c[k] for k in ("history", "repetition", "mask")}
    want = R.adjust_grad(c["x"], g, **back)
    d = _on(dev, back)
    x, gd = c["x"].to(dev), g.to(dev)
    dx = torch.full((rows, cols), 7.0, dtype=dtype, device=dev)
    G.adjust_logits_backward(x, gd, dx, **d)
    assert _same(dx, want)
    for keys in ((), ("mask",), ("history", "repetition")):
        some = {k: back[k] for k in keys}
        G.adjust_logits_backward(x, gd, dx, **{k: d[k] for k in keys})
        assert _same(dx, R.adjust_grad(c["x"], g, **some))
    at = x.clone()
    G.adjust_logits_backward(at, gd, at, **d)  # in the logits' place
    assert _same(at, want)
    G.adjust_logits_backward(x, gd, gd, **d)  # in the gradient's
    assert _same(gd, want)


def test_gradient_against_differences(dev):
    """In fp32 on powers of two, where the differences of the adjusted logits are exact."""
    rows, cols = 2, 500
    g = torch.Generator().manual_seed(2)
    x = torch.sign(torch.randn((rows, cols), generator=g)) * torch.exp2(torch.randint(-2, 3, (rows, cols), generator=g).float())
    c = _case(rows, cols, 80, 0, torch.float32, share=0.8)
    kw = dict(history=c["history"], repetition=torch.tensor([2.0, 0.5]), mask=c["mask"])
    d, ys = _on(dev, kw), []
    for step in (0.125, -0.125):
        y = torch.empty((rows, cols), device=dev)
        G.adjust_logits((x + step * x.abs()).to(dev), y, **d)
        ys.append(y.cpu())
    slope = torch.where(torch.isinf(ys[0]), 0.0, (ys[0] - ys[1]) / (0.25 * x.abs()))
    dy = torch.randn((rows, cols), generator=g)
    dx = torch.empty((rows, cols), device=dev)
    G.adjust_logits_backward(x.to(dev), dy.to(dev), dx, **d)
    assert torch.equal(dx.cpu(), dy * slope)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_strided_rows_at_odd_addresses(dev, dtype, in_place):
    rows, cols = 6, 2501
    c = _case(rows, cols, 70, 11, dtype, 4)
    want = R.adjust(**c)
    g = torch.randn((rows, cols), generator=torch.Generator().manual_seed(9)).to(dtype)
    back = {k: c[k] for k in ("history", "repetition", "mask")}
    want_g = R.adjust_grad(c["x"], g, **back)
    words = c["mask"].shape[1]
    wide_mask = torch.full((rows, words + 3), -1, dtype=torch.int32)
    wide_mask[:, 1:1 + words] = c["mask"]
    d = _on(dev, c)
    d["mask"] = wide_mask.to(dev)[:, 1:1 + words]
    d.pop("x")

    def put(t):
        base = torch.full((2 * rows + 1, cols + 6), 3.0, dtype=dtype, device=dev)
        view = base[1:2 * rows:2, 5:5 + cols]
        view.copy_(t)
        return base, view

    (xb, x), (gb, gd) = put(c["x"]), put(g)
    ob, out = (xb, x) if in_place else put(torch.zeros((rows, cols)))
    db, dx = (gb, gd) if in_place else put(torch.zeros((rows, cols)))
    G.adjust_logits_backward(x, gd, dx, **{k: d[k] for k in back})
    G.adjust_logits(x, out, **d)
    for got, base, ref in ((out, ob, want), (dx, db, want_g)):
        assert _same(got, ref)
        got.fill_(3.0)
        assert bool((base == 3.0).all()), "a value outside the rows was written"


def test_captured_and_replayed(dev):
    rows, cols = 5, 9000
    c = _case(rows, cols, 50, 10, torch.float16, 5)
    d = _on(dev, c)
    x = d.pop("x")
    g = torch.randn((rows, cols), device=dev).half()
    y, dx, want, want_dx = (torch.empty((rows, cols), dtype=torch.float16, device=dev) for _ in range(4))
    back = {k: d[k] for k in ("history", "repetition", "mask")}

    def step(y, dx):
        G.adjust_logits(x, y, **d)
        G.adjust_logits_backward(x, g, dx, **back)

    step(y, dx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(y, dx)
    for i in range(4):
        new = _case(rows, cols, 50, 10, torch.float16, 6 + i)
        x.copy_(new["x"])
        for k in d:
            d[k].copy_(new[k])
        step(want, want_dx)
        y.zero_()
        dx.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert _same(y, want) and _same(dx, want_dx)


def test_empty_and_streams(dev):
    G.adjust_logits(torch.empty((0, 9), device=dev), torch.empty((0, 9), device=dev))
    c = _case(2, 700, 0, 0, torch.float32)  # a history without tokens
    d = _on(dev, c)
    x, out = d.pop("x"), torch.empty((2, 700), device=dev)
    want = R.adjust(c["x"], mask=c["mask"])
    G.adjust_logits(x, out, **d)
    assert _same(out, want)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (other.cuda_stream, 0):
        out.zero_()
        torch.cuda.synchronize()
        G.adjust_logits(x, out, stream_ptr=s, **d)
        torch.cuda.synchronize()
        assert _same(out, want)
    with torch.cuda.stream(torch.cuda.default_stream()):
        out.zero_()
        G.adjust_logits(x, out, **d)
        assert _same(out, want)


def test_offsets_past_32_bits(dev):
    """More than 2^31 logits."""
    rows, cols = 70000, 32776
    x = torch.zeros((rows, cols), dtype=torch.float16, device=dev)
    x += 1.0
    history = torch.arange(rows, device=dev)[:, None] % cols
    rho = torch.full((rows,), 2.0, device=dev)
    G.adjust_logits(x, x, history=history, repetition=rho)
    for r in (0, 1, 32775, 32776, 65535, 65536, rows - 1):
        want = torch.ones(cols, dtype=torch.float16)
        want[r % cols] = 0.5
        assert torch.equal(x[r].cpu(), want)
    assert int((x == 0.5).sum(dtype=torch.int64)) == rows
