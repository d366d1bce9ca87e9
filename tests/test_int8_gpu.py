"""Int8 rows and their products on the GPU against int8_ref.py. Integers, scales and sums are exact, and the definition rounds
at named places: without an activation and with alpha 1 everything has to be equal bit for bit. With alpha, beta and a bias each
step is off by at most half a unit (2^-24) of the sum of magnitudes; an activation's own errors are beside it."""
import math

import pytest
import torch

import gonngpu as G
from tests import int8_ref as R
from tests.lowbit_ref import act as act64

pytestmark = pytest.mark.gpu

E = 2.0**-24


def _say(*a):
    print(*a, flush=True)


def _x(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-9, 6, (rows, 1), generator=g).float())
    return x.to(dtype)


def _ints(rows, cols, seed, lo=-127):
    return torch.randint(lo, 128, (rows, cols), generator=torch.Generator().manual_seed(seed)).to(torch.int8)


def _scales(rows, seed):
    return torch.exp2(6 * torch.rand(rows, generator=torch.Generator().manual_seed(seed)) - 12)


def _stored(dev, q, fill=77):
    """q in the layout of int8_empty; the bytes past its rows' ends are not zero."""
    full = torch.full((q.shape[0], -(-q.shape[1] // 16) * 16), fill, dtype=torch.int8)
    full[:, :q.shape[1]] = q
    return full.to(dev)[:, :q.shape[1]]


def _quantized(dev, x, col_scale=None):
    q, s = G.int8_empty(*x.shape, device=dev)
    q.fill_(55)
    s.fill_(-1.0)
    G.int8_quantize(x, q, s, col_scale=col_scale)
    return q, s


def _same(a, b):
    """Equal, NaN to NaN."""
    a, b = a.cpu(), b.cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=9e9), torch.nan_to_num(b, nan=9e9))


QSIZES = [(1, 1), (3, 7), (2, 8), (5, 9), (70, 100), (7, 511), (9, 512), (4, 513), (16, 1000), (3, 1024), (3, 1025), (2, 2048), (33, 2049),
          (3, 4096), (5, 4100), (2, 8192), (3, 8200), (2, 32768), (2, 32776), (1, 70001), (2, 131072)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("rows,cols", QSIZES)
def test_quantize_and_back(dev, rows, cols, dtype, scaled):
    _say("quantize", rows, cols, dtype, scaled)
    x = _x(rows, cols, dtype, rows * cols)
    c = torch.exp(torch.randn(cols, generator=torch.Generator().manual_seed(3))) if scaled else None
    q, s = _quantized(dev, x.to(dev), c.to(dev) if scaled else None)
    want = R.quantize(x, c)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
    y = torch.full((rows, cols), 7.0, dtype=dtype, device=dev)
    G.int8_dequantize(q, s, y)
    assert torch.equal(y.cpu(), R.values(*want).to(dtype))


@pytest.mark.parametrize("top", [127.0, 126.99999, 1.0, 3.3, 2.0**-130, 3e38, 2.0**-149, 255 * 2.0**-140])
def test_quantize_next_to_the_middles(dev, top):
    """Values that are a middle of two integers, and the fp32 numbers beside it, for every integer: of scales that are exact,
    rounded, subnormal and the largest."""
    s = torch.clamp_min(torch.tensor(top).double() / 127, 2.0**-126).float()
    mid = ((torch.arange(-127, 127).double() + 0.5) * s.double()).float()
    up, down = torch.nextafter(mid, torch.tensor(math.inf)), torch.nextafter(mid, torch.tensor(-math.inf))
    row = torch.cat((mid, up, down, torch.tensor([top, -top, 0.0, -0.0])))
    row = torch.where(row.abs() <= top, row, 0.0).to(torch.float32)
    assert float(row.abs().max()) == float(torch.tensor(top))
    x = torch.stack((row, -row, row.flip(0)))
    q, sc = _quantized(dev, x.to(dev))
    want = R.quantize(x)
    assert torch.equal(sc.cpu(), want[1]) and torch.equal(q.cpu(), want[0])


@pytest.mark.parametrize("cols", [5, 600, 3000, 40000])
def test_quantize_extremes(dev, cols):
    """Zeros, infinities, NaN, and products with a column's factor that overflow: their rows and no others."""
    x = torch.ones((9, cols))
    x[0], x[1, cols - 1], x[2, 3], x[3, cols // 2] = 0.0, math.inf, -math.inf, math.nan
    x[4] = -0.0
    x[5, 0], x[6, 1], x[7] = 3.4e38, 1e-45, 1e-42
    q, s = _quantized(dev, x.to(dev))
    want = R.quantize(x)
    assert torch.equal(q.cpu(), want[0]) and _same(s, want[1])
    y = torch.empty((9, cols), device=dev)
    G.int8_dequantize(q, s, y)
    assert _same(y, R.values(*want))
    c = torch.ones(cols)
    c[0], c[1] = 2.0, 0.0
    q, s = _quantized(dev, x.to(dev), c.to(dev))
    want = R.quantize(x, c)
    assert math.isnan(float(want[1][5])) and torch.equal(q.cpu(), want[0]) and _same(s, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("cols", [37, 297, 1500, 5001])
def test_strided_rows_at_odd_addresses(dev, dtype, cols):
    base = _x(40, cols + 4, dtype, 3).to(dev)
    x = base[1:38:2, 3:3 + cols]
    q = torch.full((40, cols + 6), 99, dtype=torch.int8, device=dev)
    at = q[2:21, 5:5 + cols]
    s = torch.empty(19, device=dev)
    G.int8_quantize(x, at, s)
    want = R.quantize(x.cpu())
    assert torch.equal(at.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
    at.fill_(99)
    assert bool((q == 99).all()), "a byte outside the rows was written"
    G.int8_quantize(x, at, s)
    out = torch.full((40, cols + 4), 5.0, dtype=dtype, device=dev)
    G.int8_dequantize(at, s, out[1:38:2, 3:3 + cols])
    full = torch.full((40, cols + 4), 5.0, dtype=dtype)
    full[1:38:2, 3:3 + cols] = R.values(*want).to(dtype)
    assert torch.equal(out.cpu(), full)


SIZES = [(1, 1, 1), (2, 3, 9), (70, 90, 1), (80, 100, 8), (100, 70, 33), (65, 1, 128), (300, 1, 264), (1, 16, 64), (1, 300, 4096), (2, 33, 100),
         (3, 128, 129), (4, 40, 2000), (5, 77, 1000), (8, 60, 1030), (9, 333, 512), (16, 1000, 512), (17, 64, 640), (27, 500, 2027), (31, 70, 127),
         (32, 200, 1152), (33, 257, 384), (48, 130, 2050), (64, 130, 96), (65, 129, 257), (100, 260, 1024), (128, 128, 128), (129, 256, 256),
         (200, 300, 515), (256, 512, 768), (300, 700, 1300), (513, 300, 260), (520, 1030, 4096), (1, 8200, 300), (7, 9000, 777), (20, 9100, 200),
         (60, 8300, 330), (100, 9000, 200), (200, 9000, 130), (300, 11000, 260), (1000, 11000, 140), (400, 11000, 328), (3900, 4000, 200),
         (2, 20, 40000), (40, 20, 131071), (70, 40, 20001), (1, 50, 20000), (3, 33, 7000), (4, 5000, 100), (4, 17, 6000), (4, 17, 6200)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(dev, M, N, K):
    _say("int8 product", M, N, K)
    a, b, sa, sb = _ints(M, K, M), _ints(N, K, N + 1), _scales(M, 5), _scales(N, 6)
    ad, bd, sad, sbd = _stored(dev, a), _stored(dev, b, -99), sa.to(dev), sb.to(dev)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_gemm((ad, sad), (bd, sbd), y)
    assert torch.equal(y.cpu(), R.product(a, sa, b, sb))
    for ps, qs in ((None, None), (None, sb), (sa, None)):
        y.fill_(math.nan)
        G.int8_gemm((ad, None if ps is None else sad), (bd, None if qs is None else sbd), y)
        assert torch.equal(y.cpu(), R.product(a, ps, b, qs))


@pytest.mark.parametrize("M,N,K", [(190, 9000, K) for K in (1, 16, 100, 128, 129, 140, 255, 256, 257, 300, 384, 400, 512, 515, 640, 700, 777)] +
                         [(200, 3000, K) for K in (1025, 1040, 1152, 1153, 1279, 1280, 1285, 1408, 1500)])
def test_ends_of_k(dev, M, N, K):
    """K that ends at, inside and next to each piece of a stage; A's bytes past it are not zeros."""
    _say("ends of K", M, N, K)
    a, b = _ints(M, K, K), _ints(N, K, K + 1)
    ad, bd = _stored(dev, a, 77), _stored(dev, b, -99)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_gemm((ad, None), (bd, None), y)
    assert torch.equal(y.cpu(), R.product(a, None, b, None))


@pytest.mark.parametrize("M,N,K", [(1, 16385, 3585), (16, 16400, 3600), (5, 16390, 4097), (16, 16416, 5003), (17, 16400, 3600), (16, 16384, 3600), (16, 16400, 3584)])
def test_few_rows_of_a_long_stream(dev, M, N, K):
    _say("long stream", M, N, K)
    a, b, sa, sb = _ints(M, K, M), _ints(N, K, N), _scales(M, 5), _scales(N, 6)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_gemm((_stored(dev, a), sa.to(dev)), (_stored(dev, b, -99), sb.to(dev)), y)
    assert torch.equal(y.cpu(), R.product(a, sa, b, sb))


@pytest.mark.parametrize("M,N", [(1, 20), (10, 20), (40, 20), (70, 20)])
def test_largest_sums(dev, M, N):
    """Every product 128 x 128 over the largest K, and the same with the other sign."""
    K = 131071
    a, b = torch.full((M, K), -128, dtype=torch.int8), torch.full((N, K), -128, dtype=torch.int8)
    b[1::2] = 127
    y = torch.empty((M, N), device=dev)
    G.int8_gemm((_stored(dev, a), None), (_stored(dev, b), None), y)
    assert torch.equal(y.cpu(), torch.tensor([16384.0 * K, -128 * 127.0 * K]).repeat(N // 2).repeat(M, 1).float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(dev, M, N, K, dtype, scaled):
    """The same, bit for bit, as quantised first and multiplied then."""
    _say("int8 linear", M, N, K, dtype, scaled)
    x, b, sb = _x(M, K, dtype, K), _ints(N, K, N + 2), _scales(N, 7)
    c = torch.exp(torch.randn(K, generator=torch.Generator().manual_seed(4))) if scaled else None
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_linear(x.to(dev), (_stored(dev, b), sb.to(dev)), y, col_scale=c.to(dev) if scaled else None)
    q, s = R.quantize(x, c)
    assert torch.equal(y.cpu(), R.product(q, s, b, sb))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("N,K", [(16384, 100), (16385, 100), (16400, 515), (40003, 1), (20000, 4100)])
def test_few_rows_of_many_columns(dev, M, N, K, dtype):
    _say("few rows", M, N, K, dtype)
    x = (torch.randn((M, K), generator=torch.Generator().manual_seed(M + N))).to(dtype)
    b, sb = _ints(N, K, N), _scales(N, 6)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_linear(x.to(dev), (_stored(dev, b, -99), sb.to(dev)), y)
    q, s = R.quantize(x)
    assert torch.equal(y.cpu(), R.product(q, s, b, sb))


@pytest.mark.parametrize("M", [1, 3, 9, 20, 50, 90, 300])
def test_linear_rows_with_nan_and_inf(dev, M):
    """Their rows are NaN and no others."""
    N, K = 150, 300
    x, b = _x(M, K, torch.float32, 8), _ints(N, K, 9)
    x[M - 1, 77] = math.inf
    if M > 2:
        x[1, K - 1] = math.nan
    y = torch.empty((M, N), device=dev)
    G.int8_linear(x.to(dev), (_stored(dev, b), None), y)
    q, s = R.quantize(x)
    want = R.product(q, s, b, None)
    assert bool(torch.isnan(want[M - 1]).all()) and _same(y, want)


@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("M,N", [(1, 40), (4, 75), (14, 75), (40, 75), (90, 140), (300, 260)])
def test_epilogue_strides_and_edges(dev, M, N, linear):
    K = 170
    a, b, sa, sb = _ints(M, K, 11), _ints(N, K, 10), _scales(M, 12), _scales(N, 13)
    x = _x(M, K, torch.float16, 14)
    if linear:
        a, sa = R.quantize(x)
        wide = torch.full((M, K + 9), math.nan, dtype=torch.float16, device=dev)
        wide[:, 3:3 + K] = x.to(dev)  # rows at odd addresses
        xd = wide[:, 3:3 + K]
    else:
        wide = torch.full((M, K + 6 + 48), 88, dtype=torch.int8, device=dev)  # views of wider matrices, whose other bytes count for nothing
        wide[:, 16:16 + K] = a.to(dev)
        ad, sad = wide[:, 16:16 + K], sa.to(dev)
    wideb = torch.full((N, K + 6 + 16), 88, dtype=torch.int8, device=dev)
    wideb[:, :K] = b.to(dev)
    bd, sbd = wideb[:, :K], sb.to(dev)
    g = torch.Generator().manual_seed(12)
    bias, c0 = torch.randn(N, generator=g), torch.randn((M, N), generator=g)
    exact = R.product(a, sa, b, sb).double()
    for act, slope in ((G.ACT_NONE, 0.0), (G.ACT_RELU, 0.0), (G.ACT_GELU, 0.0), (G.ACT_LEAKY_RELU, 0.1)):
        y = torch.full((M + 2, N + 3), 5.0, device=dev)
        y[1:-1, 1:-2] = c0.to(dev)
        kw = dict(alpha=0.25, beta=-0.5, bias=bias.to(dev), act=act, act_alpha=slope)
        if linear:
            G.int8_linear(xd, (bd, sbd), y[1:-1, 1:-2], **kw)
        else:
            G.int8_gemm((ad, sad), (bd, sbd), y[1:-1, 1:-2], **kw)
        got = y.cpu()
        inner = got[1:-1, 1:-2].clone()
        got[1:-1, 1:-2] = 5.0
        assert bool((got == 5.0).all()), "a value outside the matrix was written"
        pre = 0.25 * exact - 0.5 * c0.double() + bias.double()
        size = 0.25 * exact.abs() + 0.5 * c0.double().abs() + bias.double().abs()
        ref = act64(pre, act, slope)
        # at most three roundings of terms and sums, each of half a unit of something no larger than size
        bound = 4 * E * size
        if act == G.ACT_GELU:
            # GELU's slope is at most 1.13; its own error: the exponent 2u (|u| <= |y| + y^2 |y| / 20) in 4 roundings,
            # times x sigmoid(2u) <= |y|, and as much again for the exponential and the reciprocal
            u = 2.0 * 0.8 * (pre.abs() + 0.045 * pre.abs() ** 3)
            bound = 1.13 * bound + 2 * E * ref.abs() * (8 + 4 * u) + 1e-30
        elif act == G.ACT_LEAKY_RELU:
            bound = bound + E * ref.abs()
        assert bool(((inner.double() - ref).abs() <= bound).all()), act
    y = torch.full((M, N), math.nan, device=dev)  # beta 0 does not read C
    G.int8_gemm((_stored(dev, a), sa.to(dev)), (bd, sbd), y)
    assert torch.equal(y.cpu(), exact.float())


@pytest.mark.parametrize("M,N,K", [(1, 100, 640), (12, 300, 256), (50, 200, 130), (150, 200, 700)])
def test_input_gradient(dev, M, N, K):
    """The gradient of a frozen layer's inputs against that of the layer as it is defined, in 64 bits: dX = (dY s_w) W, off by what
    bringing dY s_w to 8 bits loses, half a step of the row's scale in each value. And that the formula is the derivative: the
    layer is linear in the values that its inputs stand for, so differences are exact."""
    g = torch.Generator().manual_seed(M)
    w = torch.randn((N, K), generator=g)
    wq, ws = R.quantize(w)
    dy = torch.randn((M, N), generator=g)
    wt = _stored(dev, wq.t().contiguous())
    dx = torch.full((M, K), math.nan, device=dev)
    G.int8_linear(dy.to(dev), (wt, None), dx, col_scale=ws.to(dev))
    t = dy.double() * ws.double()
    ref = t @ wq.double()
    step = (t.abs().amax(1) / 127)[:, None]
    # half a step in each of N terms, and the roundings of the product dy s_w, the scale and the result
    bound = (0.5 * step + 2 * E * t.abs()) @ wq.double().abs() + 3 * E * (step * 127) @ torch.ones((1, N)).double() @ wq.double().abs()
    assert bool(((dx.cpu().double() - ref).abs() <= bound).all())
    x = torch.randn((M, K), generator=g).double()
    v = torch.randn((M, K), generator=g).double()
    loss = lambda z: ((z @ (wq.double() * ws.double()[:, None]).t()) * dy.double()).sum()  # noqa: E731
    slope = (loss(x + 0.5 * v) - loss(x - 0.5 * v))
    assert abs(float(slope - (ref * v).sum())) <= 1e-10 * float((ref.abs() * v.abs()).sum())


def test_empty_sizes(dev):
    y = torch.full((3, 5), 2.0, device=dev)
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8, device=dev)  # noqa: E731
    G.int8_gemm((i8(3, 0), torch.ones(3, device=dev)), (i8(5, 0), None), y, beta=0.5, bias=torch.ones(5, device=dev))
    assert bool((y == 2.0).all())
    G.int8_linear(torch.empty((3, 0), device=dev), (i8(5, 0), None), y, beta=1.0)
    assert bool((y == 2.0).all())
    G.int8_gemm((i8(3, 0), None), (i8(5, 0), None), y)
    assert bool((y == 0.0).all())
    G.int8_gemm((i8(0, 64), torch.empty(0, device=dev)), (i8(5, 64), None), y[:0])
    G.int8_linear(torch.empty((0, 64), device=dev), (i8(5, 64), None), y[:0])
    G.int8_linear(torch.empty((3, 64), device=dev), (i8(0, 64), None), y[:, :0])
    s = torch.full((4,), 7.0, device=dev)
    G.int8_quantize(torch.empty((0, 64), device=dev), i8(0, 64), s[:0])
    G.int8_quantize(torch.empty((4, 0), device=dev), i8(4, 0), s)
    assert bool((s == 2.0**-126).all())  # a row of nothing has the scale of a row of zeros
    G.int8_dequantize(i8(0, 64), s[:0], torch.empty((0, 64), device=dev))
    G.int8_dequantize(i8(4, 0), s, torch.empty((4, 0), device=dev))


@pytest.mark.parametrize("M", [1, 6, 33, 150])
def test_captured_and_replayed(dev, M):
    """Two graphs of the same calls, captured before either runs, with eager calls between their replays."""
    N, K = 200, 301
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
    for i in range(4):
        x.copy_(_x(M, K, torch.float16, 20 + i))
        w.copy_(_x(N, K, torch.float32, 30 + i))
        step(ys[2])
        for y in ys[:2]:
            y.fill_(math.nan)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[2]) and torch.equal(ys[1], ys[2])


@pytest.mark.parametrize("M", [2, 90])
def test_streams(dev, M):
    """On a stream of its own, on the library's, on the default one, and several at once with workspaces of their own."""
    N, K = 300, 500
    x, b = _x(M, K, torch.float16, 15).to(dev), _stored(dev, _ints(N, K, 16))
    want, y = torch.empty((M, N), device=dev), torch.empty((M, N), device=dev)
    G.int8_linear(x, (b, None), want)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    G.int8_linear(x, (b, None), y, stream_ptr=other.cuda_stream)
    other.synchronize()
    assert torch.equal(y, want)
    y.fill_(0)
    torch.cuda.synchronize()
    G.int8_linear(x, (b, None), y, stream_ptr=0)
    G.synchronize()
    assert torch.equal(y, want)
    y.fill_(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.default_stream()):
        G.int8_linear(x, (b, None), y)
        assert torch.equal(y, want)
    streams, outs = [torch.cuda.Stream() for _ in range(4)], [torch.zeros((M, N), device=dev) for _ in range(4)]
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 4]):
            G.int8_linear(x * (1 + i % 4), (b, None), outs[i % 4])
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        q, s = R.quantize((x * (1 + i)).cpu())
        assert torch.equal(o.cpu(), R.product(q, s, b.cpu(), None))


def test_offsets_past_32_bits(dev):
    """More than 2^32 weights and more than 2^31 outputs."""
    rows, cols = 135000, 32768
    w = torch.empty((rows, cols), dtype=torch.float16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    wq = G.int8_empty(rows, cols, device=dev)
    G.int8_quantize(w, *wq)
    pick = torch.tensor([0, 1, 65535, 65536, 131071, 131072, 134999], device=dev)
    ref = R.quantize(w[pick].cpu())
    assert torch.equal(wq[0][pick].cpu(), ref[0]) and torch.equal(wq[1][pick].cpu(), ref[1])
    G.int8_dequantize(*wq, w)
    assert torch.equal(w[pick].cpu(), R.values(*ref).half())
    del w
    for M in (2, 30, 80):
        x = _x(M, cols, torch.float16, 2)
        y = torch.empty((M, rows), device=dev)
        G.int8_linear(x.to(dev), wq, y)
        assert torch.equal(y[:, pick].cpu(), R.product(*R.quantize(x), *ref))
        del y
    K, N = 64, 16500
    a, b = torch.randint(-127, 128, (rows, K), dtype=torch.int8, device=dev), _ints(N, K, 3)
    y = torch.full((rows, N), math.nan, device=dev)
    cols_at = torch.tensor([0, 15, 16383, 16499], device=dev)
    G.int8_gemm((a, None), (b.to(dev), None), y)
    assert torch.equal(y[pick][:, cols_at].cpu(), R.product(a[pick].cpu(), None, b[cols_at.cpu()], None))
    assert bool(torch.isfinite(y[-1]).all())
