"""Int8 products by every kind of kernel that the library chooses from. The sizes are picked for that: a test on the CPU applies the
rule and the table of launch_product, as they stand in the source, and says which kind a size takes. K has more pieces than a kernel has
slots for them, so that each slot is filled anew, and is no multiple of 16; the last rows and columns end inside a tile."""
import math
import os
import re

import pytest
import torch

import gonngpu as G
from tests import int8_ref as R
from tests.lowbit_ref import act as act64
from tests.test_int8_gpu import E, _ints, _same, _say, _scales, _stored, _x

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-nngpu_amd", "csrc", "int8_gemm.hip")

# Each kind's size, and how many bytes of K its slots hold.
LONG = "16 x 32, a long stream"
SIZES = [((3, 150, 2203), 0, 4 * 4 * 128), ((5, 8221, 2235), 1, 8 * 2 * 128), ((9, 4215, 2297), 2, 8 * 2 * 128), ((18, 8345, 1059), 3, 8 * 2 * 64),
         ((70, 6001, 1035), 4, 6 * 128), ((70, 6001, 651), 5, 4 * 128), ((70, 8262, 909), 6, 6 * 128), ((654, 11263, 523), 7, 3 * 128),
         ((201, 9001, 651), 8, 3 * 128), ((261, 11319, 651), 9, 3 * 128), ((521, 11001, 651), 10, 3 * 128), ((1001, 9001, 395), 11, 2 * 128),
         ((13, 16411, 3605), LONG, 4 * 2 * 128)]
TILES = [s for s, kind, _ in SIZES if kind != LONG and kind >= 4]


def _table():
    with open(SOURCE) as f:
        text = re.search(r"TileCost kTiles\[\] = \{(.*?)\};", f.read(), re.S).group(1)
    return [tuple(int(n) for n in row.split(",")) for row in re.findall(r"\{([\d, ]+)\}", text)]


def _kind(M, N, K):
    if M <= 16 and N > 64 * 256 and K > 3584:
        return LONG
    stages, costs = -(-K // 128), []
    for bm, bn, fixed, stage, further, more in _table():
        others = (-(-M // bm) * -(-N // bn) - 1) // 256
        costs.append(fixed + stages * stage + others * (further + stages * more))
    return costs.index(min(costs))


def test_the_sizes_take_every_kind():
    assert len(_table()) == 12
    for size, kind, slots in SIZES:
        assert _kind(*size) == kind, size
        M, N, K = size
        assert K > slots and K % 16 and N % 4
    assert {kind for _, kind, _ in SIZES} == {LONG, *range(12)}


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [s for s, _, _ in SIZES])
def test_product_and_linear(dev, M, N, K):
    """Bit for bit; and the same for K a multiple of 16."""
    _say("kinds", M, N, K)
    a, b, sa, sb = _ints(M, K, M), _ints(N, K, N + 1), _scales(M, 5), _scales(N, 6)
    x = _x(M, K, torch.float16, K)
    bd, sbd = _stored(dev, b, -99), sb.to(dev)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_gemm((_stored(dev, a), sa.to(dev)), (bd, sbd), y)
    assert torch.equal(y.cpu(), R.product(a, sa, b, sb))
    y.fill_(math.nan)
    G.int8_linear(x.to(dev), (bd, sbd), y)
    assert torch.equal(y.cpu(), R.product(*R.quantize(x), b, sb))
    K = K // 16 * 16
    y.fill_(math.nan)
    G.int8_gemm((_stored(dev, a)[:, :K], sa.to(dev)), (bd[:, :K], sbd), y)
    assert torch.equal(y.cpu(), R.product(a[:, :K], sa, b[:, :K], sb))


@pytest.mark.gpu
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("M,N,K", [s for s, _, _ in SIZES])
def test_epilogue(dev, M, N, K, linear):
    """alpha, beta, bias and activations on a C of wider rows. With S the sum: fl(S) and its product with the column's scale, alpha
    times the row's, beta C + bias (two at most) and the last sum are rounded, each by at most E = 2^-24 of something no larger than the sum of
    magnitudes: below 6 E of it with the terms of second order."""
    _say("epilogue", M, N, K, linear)
    b, sb = _ints(N, K, 10), _scales(N, 13)
    bd, sbd = _stored(dev, b, 88), sb.to(dev)
    if linear:
        x = _x(M, K, torch.float16, 14)
        a, sa = R.quantize(x)
        wide = torch.full((M, K + 9), math.nan, dtype=torch.float16, device=dev)
        wide[:, 3:3 + K] = x.to(dev)
    else:
        a, sa = _ints(M, K, 11), _scales(M, 12)
        ad = (_stored(dev, a), sa.to(dev))
    g = torch.Generator().manual_seed(12)
    bias, c0 = torch.randn(N, generator=g), torch.randn((M, N), generator=g)
    alpha, beta, slope = (float(torch.tensor(v)) for v in (0.3, -0.7, 0.1))
    product = R.sums(a, b) * sb.double() * sa.double()[:, None]
    pre = alpha * product + beta * c0.double() + bias.double()
    size = alpha * product.abs() + abs(beta) * c0.double().abs() + bias.double().abs()
    for act in (G.ACT_NONE, G.ACT_RELU, G.ACT_GELU, G.ACT_LEAKY_RELU):
        y = torch.full((M + 2, N + 3), 5.0, device=dev)
        y[1:-1, 1:-2] = c0.to(dev)
        kw = dict(alpha=alpha, beta=beta, bias=bias.to(dev), act=act, act_alpha=slope if act == G.ACT_LEAKY_RELU else 0.0)
        if linear:
            G.int8_linear(wide[:, 3:3 + K], (bd, sbd), y[1:-1, 1:-2], **kw)
        else:
            G.int8_gemm(ad, (bd, sbd), y[1:-1, 1:-2], **kw)
        got = y.cpu()
        inner = got[1:-1, 1:-2].double()
        got[1:-1, 1:-2] = 5.0
        assert bool((got == 5.0).all()), "a value outside the matrix was written"
        ref, bound = act64(pre, act, slope), 6 * E * size
        if act == G.ACT_GELU:
            # its slope is at most 1.13; its own error: the exponent 2u (|u| <= 0.8 (|y| + 0.045 |y|^3)) in 4 roundings, times
            # y sigmoid(2u) <= |y|, and as much again for the exponential and the reciprocal
            u = 2.0 * 0.8 * (pre.abs() + 0.045 * pre.abs() ** 3)
            bound = 1.13 * bound + 2 * E * ref.abs() * (8 + 4 * u) + 1e-30
        elif act == G.ACT_LEAKY_RELU:
            bound = bound + E * ref.abs()
        assert bool(((inner - ref).abs() <= bound).all()), act
    # One of them at a time: each on exact numbers, so bit for bit.
    y = torch.full((M, N), math.nan, device=dev)
    plain = R.product(a, sa, b, sb)
    call = (lambda **kw: G.int8_linear(wide[:, 3:3 + K], (bd, sbd), y, **kw)) if linear else (lambda **kw: G.int8_gemm(ad, (bd, sbd), y, **kw))
    call(alpha=-0.25, act=G.ACT_RELU)  # beta 0 does not read C
    assert torch.equal(y.cpu(), (-0.25 * plain).clamp_min(0.0))
    y.copy_(c0)
    call(alpha=0.0, beta=-0.5)
    assert torch.equal(y.cpu(), -0.5 * c0)
    call(alpha=0.0, bias=bias.to(dev))
    assert torch.equal(y.cpu(), bias.repeat(M, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", TILES)
def test_rows_with_nan_and_inf(dev, M, N, K):
    """Their rows are NaN and no others."""
    x, b = _x(M, K, torch.float32, 8), _ints(N, K, 9)
    x[M - 1, 77], x[1, K - 1], x[33 % M, 0] = math.inf, math.nan, -math.inf
    y = torch.empty((M, N), device=dev)
    G.int8_linear(x.to(dev), (_stored(dev, b), None), y)
    want = R.product(*R.quantize(x), b, None)
    assert bool(torch.isnan(want[[1, 33 % M, M - 1]]).all()) and _same(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", TILES)
def test_captured_and_replayed(dev, M, N, K):
    """Two graphs of the same calls, with eager calls between their replays."""
    x, w = _x(M, K, torch.float16, 13).to(dev), _x(N, K, torch.float32, 14).to(dev)
    wq, xq = G.int8_empty(N, K, device=dev), G.int8_empty(M, K, device=dev)
    ys = [torch.empty((M, N), device=dev) for _ in range(3)]

    def step(y):
        G.int8_quantize(w, *wq)
        G.int8_linear(x, wq, y)
        G.int8_quantize(x, *xq)
        G.int8_gemm(xq, wq, y, beta=1.0)

    step(ys[2])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, y in zip(graphs, ys):
        with torch.cuda.graph(graph):
            step(y)
    for i in range(3):
        x.copy_(_x(M, K, torch.float16, 20 + i))
        w.copy_(_x(N, K, torch.float32, 30 + i))
        step(ys[2])
        for y in ys[:2]:
            y.fill_(math.nan)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[2]) and torch.equal(ys[1], ys[2])
