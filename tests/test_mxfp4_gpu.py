"""MXFP4 quantisation, dequantisation and products on the GPU against the 64-bit restatements of
lowbit_ref.py. Codes, scale bytes and fp32 values have to be equal bit for bit. A product's error is bounded by
arithmetic: its K products are exact in fp32 (4-bit values times 11- or 2-bit ones), each of at most K + 8 additions
and scalings of partial sums is off by at most one unit (2^-23) of the sum of magnitudes (matrix
instructions need not round to nearest), and so is each step of the epilogue."""
import math

import numpy as np
import pytest
import torch

import gonngpu as G
from tests import lowbit_ref as R

pytestmark = pytest.mark.gpu

STEP = 2.0**-23


def _say(*a):
    print(*a, flush=True)


def _x(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp2(torch.randint(-9, 10, (rows, 1), generator=g).float())
    return x.to(dtype)


def _quantize(dev, x):
    data, scales = G.mxfp4_empty(*x.shape, device=dev)
    data.fill_(0xEE)
    scales.fill_(0xEE)
    G.mxfp4_quantize(x, data, scales)
    return data, scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 127), (4, 128), (2, 129), (16, 1000), (33, 2027), (70, 4096)])
def test_quantize_and_back(dev, rows, cols, dtype):
    x = _x(rows, cols, dtype, rows * cols)
    data, scales = _quantize(dev, x.to(dev))
    ref = R.quantize(x)
    assert torch.equal(data.cpu(), ref[0]) and torch.equal(scales.cpu(), ref[1])
    y = torch.full((rows, cols), 7.0, dtype=dtype, device=dev)
    G.mxfp4_dequantize(data, scales, y)
    assert torch.equal(y.cpu(), R.values(*ref, cols).to(dtype))


def test_quantize_rounds_ties_to_even_and_saturates(dev):
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    near = [v * f for v in mids for f in (1 - 2**-20, 1.0, 1 + 2**-20)]
    row = [4.0] + near + [6.0, 6.9, 7.0, 7.5, 7.99, 0.0, -0.0, 1e-30, -1e-30]
    row = (row + [0.0] * 32)[:32]
    x = torch.tensor([row, [-v for v in row], [v * 2.0**-100 for v in row], [v * 2.0**100 for v in row]])
    data, scales = _quantize(dev, x.to(dev))
    ref = R.quantize(x)
    assert torch.equal(data.cpu(), ref[0]) and torch.equal(scales.cpu(), ref[1])


def test_quantize_extremes(dev):
    """Subnormals, the largest values, zeros of both signs, infinities and NaN in one block and not in the next."""
    t = 2.0**-149
    rows = [[t, -t, 3 * t, 0.0], [2.0**-126, 2.0**-127, 5 * 2.0**-129, -(2.0**-128)], [2.0**-125, 1.5 * 2.0**-126, 0.0, -0.0],
            [2.0**-124, 7 * 2.0**-127, 2.0**-126, 0.0], [2.0**-123, 2.0**-125, 3 * 2.0**-127, 2.0**-140],
            [3.4e38, -3.4e38, 1e38, 5e37], [0.0, -0.0, 0.0, -0.0], [math.inf, 1.0, 2.0, 3.0], [-math.inf, 1.0, 2.0, 3.0],
            [math.nan, 1.0, 2.0, 3.0], [1.0, math.nan, math.inf, 3.0]]
    x = torch.zeros((len(rows), 70))
    x[:, :4] = torch.tensor(rows, dtype=torch.float64).float()
    x[:, 40] = 1.0  # the next block is an ordinary one
    data, scales = _quantize(dev, x.to(dev))
    ref = R.quantize(x)
    assert torch.equal(scales.cpu(), ref[1])
    assert torch.equal(data.cpu(), ref[0])
    y = torch.empty((len(rows), 70), device=dev)
    G.mxfp4_dequantize(data, scales, y)
    assert torch.equal(torch.nan_to_num(y.cpu(), nan=9e9), torch.nan_to_num(R.values(*ref, 70).float(), nan=9e9))
    xh = x.half()  # infinities from 3.4e38, fp16 subnormals from the small ones are 0
    xh[0, :4] = torch.tensor([2.0**-24, -(2.0**-24), 3 * 2.0**-24, 2.0**-14])
    data, scales = _quantize(dev, xh.to(dev))
    ref = R.quantize(xh)
    assert torch.equal(data.cpu(), ref[0]) and torch.equal(scales.cpu(), ref[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strided_rows_at_odd_addresses(dev, dtype):
    base = _x(40, 301, dtype, 3).to(dev)
    x = base[1:38:2, 3:300]  # rows 602 elements apart, each at an odd element
    data, scales = _quantize(dev, x)
    ref = R.quantize(x.cpu())
    assert torch.equal(data.cpu(), ref[0]) and torch.equal(scales.cpu(), ref[1])
    out = torch.full((40, 301), 5.0, dtype=dtype, device=dev)
    G.mxfp4_dequantize(data, scales, out[1:38:2, 3:300])
    want = torch.full((40, 301), 5.0, dtype=dtype)
    want[1:38:2, 3:300] = R.values(*ref, 297).to(dtype)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_dequantize_every_code_and_scale(dev, dtype):
    data = torch.zeros((256, 64), dtype=torch.uint8)
    data[:, :16] = torch.tensor([(2 * i) % 16 + 16 * ((2 * i + 1) % 16) for i in range(16)], dtype=torch.uint8)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 4)
    y = torch.empty((256, 128), dtype=dtype, device=dev)
    G.mxfp4_dequantize(data.to(dev), scales.to(dev), y)
    want = R.values(data, scales, 128).numpy()
    with np.errstate(over="ignore"):
        want = want.astype(np.float16 if dtype == torch.float16 else np.float32)
    assert np.array_equal(y.cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(np.signbit(y.cpu().numpy())[:255], np.signbit(want)[:255])


def _weights(rows, cols, seed, lo=119, hi=125):
    g = torch.Generator().manual_seed(seed)
    groups = -(-cols // 128)
    code = torch.randint(0, 16, (rows, groups * 128), generator=g)
    code[:, cols:] = 0
    scales = torch.randint(lo, hi, (rows, groups * 4), generator=g).to(torch.uint8)
    scales[:, -(-cols // 32):] = 127
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), scales


def _bounded(y, a, w, K, more=0.0, alpha=1.0, slope=1.0):
    """Checks y against a w^T (+ more) in 64 bits; returns that."""
    ref = alpha * (a @ w.t()) + more
    size = abs(alpha) * (a.abs() @ w.abs().t()) + (more.abs() if torch.is_tensor(more) else abs(more))
    bound = slope * STEP * (K + 8) * size + 1e-37
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float((err / bound).max()))
    return ref


SIZES = [(1, 1, 1), (2, 3, 9), (70, 90, 1), (80, 100, 8), (100, 70, 33), (65, 1, 128), (300, 1, 264),
         (1, 16, 32), (1, 300, 4096), (2, 33, 100), (3, 128, 129), (5, 77, 1000), (16, 1000, 512), (17, 64, 640),
         (27, 500, 2027), (33, 257, 384), (64, 130, 96), (65, 129, 257), (100, 260, 1024), (128, 128, 128), (129, 256, 256),
         (200, 300, 515), (256, 512, 768), (300, 700, 1300), (513, 300, 260), (520, 1030, 4096),
         (100, 9000, 200), (200, 9000, 130), (300, 11000, 260), (1000, 11000, 140),
         (400, 11000, 328), (3900, 4000, 200)]  # these: each tile of both kinds


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_with_fp16_activations(dev, M, N, K):
    _say("fp16 product", M, N, K)
    x, w = _x(M, K, torch.float16, M), _weights(N, K, N)
    y = torch.full((M, N), math.nan, device=dev)
    G.mxfp4_gemm(x.to(dev), tuple(t.to(dev) for t in w), y)
    _bounded(y.cpu(), x.double(), R.values(*w, K), K)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_with_4_bit_activations(dev, M, N, K):
    _say("mxfp4 product", M, N, K)
    x, w = _weights(M, K, M + 1), _weights(N, K, N)
    y = torch.full((M, N), math.nan, device=dev)
    G.mxfp4_gemm(tuple(t.to(dev) for t in x), tuple(t.to(dev) for t in w), y, K=K)
    _bounded(y.cpu(), R.values(*x, K), R.values(*w, K), K)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("M,N,K", [(3, 70, 200), (40, 64, 256), (150, 300, 300), (300, 520, 512)])
def test_product_scales_over_the_whole_range(dev, M, N, K, fp4):
    """Each weight takes part with its exact value whatever its scale: bytes 1 to 230 side by side."""
    w = _weights(N, K, 5, 1, 200 if fp4 else 230)
    x = _weights(M, K, 6, 90, 140) if fp4 else _x(M, K, torch.float16, 6)
    y = torch.empty((M, N), device=dev)
    a = R.values(*x, K) if fp4 else x.double()
    G.mxfp4_gemm(tuple(t.to(dev) for t in x) if fp4 else x.to(dev), tuple(t.to(dev) for t in w), y, K=K)
    _bounded(y.cpu(), a, R.values(*w, K), K)
    w = _weights(N, K, 7, 1, 60)  # all of them small
    G.mxfp4_gemm(tuple(t.to(dev) for t in x) if fp4 else x.to(dev), tuple(t.to(dev) for t in w), y, K=K)
    _bounded(y.cpu(), a, R.values(*w, K), K)


@pytest.mark.parametrize("M,N,K", [(1, 40, 256), (20, 600, 384), (70, 200, 512), (270, 300, 128), (140, 9000, 64), (400, 11000, 64),
                                   (1000, 11000, 64), (3000, 5700, 64), (3900, 4000, 64)])
@pytest.mark.parametrize("lo,hi", [(104, 114), (114, 141), (137, 145), (100, 108)])
def test_product_scales_at_the_ends_of_fp16(dev, M, N, K, lo, hi):
    """Scales whose weights are all fp16 numbers, the subnormal ones included, and scales around both ends of that range."""
    w, x = _weights(N, K, 25, lo, hi), _x(M, K, torch.float16, 26)
    y = torch.empty((M, N), device=dev)
    G.mxfp4_gemm(x.to(dev), tuple(t.to(dev) for t in w), y)
    _bounded(y.cpu(), x.double(), R.values(*w, K), K)
    w[1][N - 1, 1] = 3  # one block elsewhere
    G.mxfp4_gemm(x.to(dev), tuple(t.to(dev) for t in w), y)
    _bounded(y.cpu(), x.double(), R.values(*w, K), K)


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("M", [2, 200])
def test_product_nan_and_inf(dev, M, fp4):
    """A NaN block makes its row's or column's outputs NaN and no others; an infinity among fp16 activations reaches
    its row with the signs of the weights, NaN where the weight is 0."""
    N, K = 150, 256
    w = _weights(N, K, 8)
    w[1][7, 3] = 255
    x = _weights(M, K, 9) if fp4 else _x(M, K, torch.float16, 9)
    if fp4:
        x[1][1, 6] = 255
    else:
        x[1, 77] = math.inf
    y = torch.empty((M, N), device=dev)
    G.mxfp4_gemm(tuple(t.to(dev) for t in x) if fp4 else x.to(dev), tuple(t.to(dev) for t in w), y, K=K)
    y = y.cpu()
    want = torch.zeros((M, N))
    if fp4:
        want[1] = math.nan
    else:
        want[1] = torch.sign(R.values(*w, K)[:, 77]).float() * math.inf
    want[:, 7] = math.nan
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(torch.sign(y[1][torch.isinf(y[1])]), torch.sign(want[1][torch.isinf(want[1])]))


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("M,N", [(4, 75), (90, 140), (300, 260)])
def test_product_epilogue_strides_and_edges(dev, M, N, fp4):
    K = 160
    w = _weights(N, K, 10)
    x = _weights(M, K, 11) if fp4 else _x(M, K, torch.float16, 11)
    a, wv = (R.values(*x, K) if fp4 else x.double()), R.values(*w, K)
    wd = tuple(t.to(dev) for t in w)
    if fp4:
        xd = tuple(t.to(dev) for t in x)
    else:  # rows at odd addresses
        wide = torch.full((M, K + 9), math.nan, dtype=torch.float16, device=dev)
        wide[:, 3:3 + K] = x.to(dev)
        xd = wide[:, 3:3 + K]
    g = torch.Generator().manual_seed(12)
    bias, c0 = torch.randn(N, generator=g), torch.randn((M, N), generator=g)
    for act, alpha in ((G.ACT_NONE, 0.0), (G.ACT_RELU, 0.0), (G.ACT_GELU, 0.0), (G.ACT_LEAKY_RELU, 0.1)):
        y = torch.full((M + 2, N + 3), 5.0, device=dev)
        y[1:-1, 1:-2] = c0.to(dev)
        G.mxfp4_gemm(xd, wd, y[1:-1, 1:-2], K=K, alpha=0.25, beta=-0.5, bias=bias.to(dev), act=act, act_alpha=alpha)
        got = y.cpu()
        inner = got[1:-1, 1:-2].clone()
        got[1:-1, 1:-2] = 5.0
        assert bool((got == 5.0).all()), "a value outside the matrix was written"
        more = -0.5 * c0.double() + bias.double()
        if act == G.ACT_GELU:
            pre = 0.25 * (a @ wv.t()) + more
            size = 0.25 * (a.abs() @ wv.abs().t()) + more.abs()
            # GELU's slope is at most 1.13; its own error: the exponent 2u (|u| <= |y| + y^2 |y| / 20) in 4 roundings,
            # times x sigmoid(2u) <= |y|, and as much again for the exponential and the reciprocal
            ref = R.act(pre, act)
            u = 2.0 * 0.8 * (pre.abs() + 0.045 * pre.abs() ** 3)
            bound = 1.13 * STEP * (K + 8) * size + STEP * ref.abs() * (8 + 4 * u) + 1e-30
            assert bool(((inner.double() - ref).abs() <= bound).all())
        else:
            pre = _bounded(inner, a, wv, K, more, 0.25) if act == G.ACT_NONE else 0.25 * (a @ wv.t()) + more
            size = 0.25 * (a.abs() @ wv.abs().t()) + more.abs()
            assert bool(((inner.double() - R.act(pre, act, alpha)).abs() <= STEP * (K + 10) * size).all())
    y = torch.full((M, N), math.nan, device=dev)  # beta 0 does not read C
    G.mxfp4_gemm(xd, wd, y, K=K)
    assert bool(torch.isfinite(y).all())


def test_empty_sizes(dev):
    w0 = G.mxfp4_empty(5, 0, device=dev)
    y = torch.full((3, 5), 2.0, device=dev)
    G.mxfp4_gemm(torch.empty((3, 0), dtype=torch.float16, device=dev), w0, y, beta=0.5, bias=torch.ones(5, device=dev))
    assert bool((y == 2.0).all())
    G.mxfp4_gemm(G.mxfp4_empty(3, 0, device=dev), w0, y, K=0)
    assert bool((y == 0.0).all())
    G.mxfp4_gemm(torch.empty((0, 64), dtype=torch.float16, device=dev), G.mxfp4_empty(5, 64, device=dev), y[:0])
    G.mxfp4_gemm(torch.empty((3, 64), dtype=torch.float16, device=dev), G.mxfp4_empty(0, 64, device=dev), y[:, :0])
    G.mxfp4_quantize(torch.empty((0, 64), device=dev), *G.mxfp4_empty(0, 64, device=dev))
    G.mxfp4_quantize(torch.empty((4, 0), device=dev), *G.mxfp4_empty(4, 0, device=dev))
    G.mxfp4_dequantize(*G.mxfp4_empty(0, 64, device=dev), torch.empty((0, 64), device=dev))


def test_captured_and_replayed(dev):
    M, N, K = 33, 200, 300
    x, w = _x(M, K, torch.float16, 13).to(dev), _x(N, K, torch.float32, 14).to(dev)
    wq, xq = G.mxfp4_empty(N, K, device=dev), G.mxfp4_empty(M, K, device=dev)
    y16, y4 = torch.empty((M, N), device=dev), torch.empty((M, N), device=dev)

    def step():
        G.mxfp4_quantize(w, *wq)
        G.mxfp4_gemm(x, wq, y16)
        G.mxfp4_quantize(x, *xq)
        G.mxfp4_gemm(xq, wq, y4, K=K)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        x.copy_(_x(M, K, torch.float16, 20 + i))
        w.copy_(_x(N, K, torch.float32, 30 + i))
        step()
        want = y16.clone(), y4.clone()
        y16.fill_(math.nan)
        y4.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y16, want[0]) and torch.equal(y4, want[1])


def test_on_another_stream_and_the_default_one(dev):
    M, N, K = 9, 300, 500
    x, w = _x(M, K, torch.float16, 15).to(dev), tuple(t.to(dev) for t in _weights(N, K, 16))
    want, y = torch.empty((M, N), device=dev), torch.empty((M, N), device=dev)
    G.mxfp4_gemm(x, w, want)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    G.mxfp4_gemm(x, w, y, stream_ptr=other.cuda_stream)
    other.synchronize()
    assert torch.equal(y, want)
    y.fill_(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.default_stream()):
        G.mxfp4_gemm(x, w, y)
        assert torch.equal(y, want)


def test_offsets_past_32_bits(dev):
    """More than 2^32 weights quantised, read back and multiplied, and more than 2^31 outputs."""
    rows, cols = 135000, 32768
    w = torch.empty((rows, cols), dtype=torch.float16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    wq = G.mxfp4_empty(rows, cols, device=dev)
    G.mxfp4_quantize(w, *wq)
    pick = torch.tensor([0, 1, 65535, 65536, 131071, 131072, 134999], device=dev)
    some = w[pick].cpu()
    ref = R.quantize(some)
    assert torch.equal(wq[0][pick].cpu(), ref[0]) and torch.equal(wq[1][pick].cpu(), ref[1])
    G.mxfp4_dequantize(*wq, w)
    wv = R.values(*ref, cols)
    assert torch.equal(w[pick].cpu(), wv.half())
    for M in (2, 80):
        x = _x(M, cols, torch.float16, 2)
        y = torch.empty((M, rows), device=dev)
        G.mxfp4_gemm(x.to(dev), wq, y)
        _bounded(y[:, pick].cpu(), x.double(), wv, cols)
    del w
    K, N = 64, 16500
    a = torch.empty((rows, K), dtype=torch.float16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(2))
    aq = G.mxfp4_empty(rows, K, device=dev)
    G.mxfp4_quantize(a, *aq)
    b = _weights(N, K, 3)
    y = torch.empty((rows, N), device=dev)
    cols_at = torch.tensor([0, 15, 16383, 16499], device=dev)
    bv = R.values(*b, K)[cols_at.cpu()]
    bd = tuple(t.to(dev) for t in b)
    G.mxfp4_gemm(a, bd, y)
    _bounded(y[pick][:, cols_at].cpu(), a[pick].cpu().double(), bv, K)
    y.fill_(math.nan)
    G.mxfp4_gemm(aq, bd, y, K=K)
    _bounded(y[pick][:, cols_at].cpu(), R.values(aq[0][pick].cpu(), aq[1][pick].cpu(), K), bv, K)
    assert bool(torch.isfinite(y[-1]).all())


@pytest.mark.parametrize("M,N,K", [(1, 40, 32), (3, 40, 20), (12, 40, 32), (27, 60, 32), (50, 64, 31), (70, 200, 32), (90, 140, 29),
                                   (140, 9000, 32), (400, 11000, 32), (1000, 11000, 32), (3900, 4000, 32)])
@pytest.mark.parametrize("codes", [(0, 1, 2, 3, 5, 20), (104, 103, 140, 141), (254, 253, 252, 251, 250, 230)])
@pytest.mark.parametrize("fp4", [False, True])
def test_product_of_single_scale_rows_at_both_ends(dev, M, N, K, codes, fp4):
    """Every row of the weights has one scale, among them the smallest and the largest that a stored matrix may have. All values
    are of one sign in a row, and the activations such that every product is a normal fp32 number: the bound is
    relative throughout, and weights flushed to 0 or to infinity do not pass it."""
    g = torch.Generator().manual_seed(M + codes[0])
    code = torch.randint(0, 8, (N, 128), generator=g) + 8 * (torch.arange(N) % 3 == 0)[:, None]
    code[:, K:] = 0
    w = ((code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8),
         torch.tensor(codes, dtype=torch.uint8)[torch.arange(N) % len(codes)][:, None].repeat(1, 4))
    wv = R.values(*w, K)
    low, high = codes[0] == 0, codes[0] == 254
    # the largest outputs are below 32 * 6 * 2^127 * 2^-9, the smallest products above 2^-128 * 2^10
    span = (2.0**10, 2.0**15) if low else (2.0**-13, 2.0**-9) if high else (2.0**-3, 2.0**3)
    if fp4:
        x = _weights(M, K, M + 1)
        x[0].bitwise_and_(0x77)
        x[1].fill_(127 + (11 if low else -14 if high else 0))
        a = R.values(*x, K)
        xd = tuple(t.to(dev) for t in x)
    else:
        x = (span[0] * torch.exp2(torch.rand((M, K), generator=g) * math.log2(span[1] / span[0]))).half()
        x[:, ::2] = torch.exp2(torch.floor(torch.log2(x[:, ::2].float()))).half()  # every other one a power of two
        a, xd = x.double(), x.to(dev)
    y = torch.full((M, N), math.nan, device=dev)
    G.mxfp4_gemm(xd, tuple(t.to(dev) for t in w), y, K=K)
    ref = a @ wv.t()
    bound = STEP * (K + 8) * (a.abs() @ wv.abs().t())
    assert bool(((y.cpu().double() - ref).abs() <= bound).all()), [
        (c, bool(((y.cpu().double() - ref).abs() <= bound)[:, i::len(codes)].all())) for i, c in enumerate(codes)]
