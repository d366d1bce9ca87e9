"""Int8 matrices without padding behind their last row: what lies between a row's end and the next multiple of 16 bytes belongs to
others, or to nobody, and counts for nothing in the products."""
import math

import pytest
import torch

import gonngpu as G
from tests import int8_ref as R
from tests.test_int8_gpu import _ints, _scales, _x

pytestmark = pytest.mark.gpu

# A row by itself, a few, and sizes of the kernels with small and with large tiles.
SIZES = [(1, 1, 1), (1, 1, 1000), (1, 50, 129), (3, 1, 1003), (4, 70, 515), (30, 90, 1001), (70, 6001, 651), (201, 9001, 651)]


def _ends(dev, q, behind):
    """q in rows that begin at multiples of 16 bytes, -128 in all bytes between them; `behind` more of these at the end."""
    rows, cols = q.shape
    ld = -(-cols // 16) * 16 + 32
    flat = torch.full(((rows - 1) * ld + cols + behind,), -128, dtype=torch.int8, device=dev)
    view = flat.as_strided((rows, cols), (ld, 1))
    view.copy_(q)
    return view


@pytest.mark.parametrize("behind", [0, 5, 4096])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products(dev, M, N, K, behind):
    a, b, sa, sb, x = _ints(M, K, 1), _ints(N, K, 2), _scales(M, 3), _scales(N, 4), _x(M, K, torch.float16, 5)
    ad, bd, sbd = _ends(dev, a, behind), _ends(dev, b, behind), sb.to(dev)
    y = torch.full((M, N), math.nan, device=dev)
    G.int8_gemm((ad, sa.to(dev)), (bd, sbd), y)
    assert torch.equal(y.cpu(), R.product(a, sa, b, sb))
    G.int8_linear(x.to(dev), (bd, sbd), y)
    assert torch.equal(y.cpu(), R.product(*R.quantize(x), b, sb))


@pytest.mark.parametrize("M,N,K", SIZES)
def test_quantised_into_them(dev, M, N, K):
    """The quantiser writes none of these bytes."""
    x = _x(M, K, torch.float32, 6)
    q, s = _ends(dev, torch.zeros((M, K), dtype=torch.int8), 3), torch.empty(M, device=dev)
    G.int8_quantize(x.to(dev), q, s)
    want = R.quantize(x)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
    q.fill_(-128)
    ld = -(-K // 16) * 16 + 32
    assert bool((q.as_strided(((M - 1) * ld + K + 3,), (1,)) == -128).all())
