"""Int8 values are the integers nearest to the exact quotients also where half of a row's scale is no fp32 number: scales
between 2^-126 and 2^-125 whose last place is odd."""
import math

import pytest
import torch

import gonngpu as G
from tests import int8_ref as R

pytestmark = pytest.mark.gpu

TOPS = [n * 2.0**-149 for n in (1065353344, 1065353216 + 127, 1300000001, 1500000127, 1700000511, 2000000001, 2130706304)]


def _row(top):
    """The middles of all integers times the row's scale, the fp32 numbers beside them, and the largest magnitude."""
    top = torch.tensor(top)
    s = torch.clamp_min(top.double() / 127, 2.0**-126).float()
    assert 2.0**-126 <= float(s) < 2.0**-125
    mid = ((torch.arange(-127, 127).double() + 0.5) * s.double()).float()
    up, down = torch.nextafter(mid, torch.tensor(math.inf)), torch.nextafter(mid, torch.tensor(-math.inf))
    row = torch.cat((mid, up, down, torch.stack((top, -top, 0 * top, -0 * top))))
    return torch.where(row.abs() <= top, row, 0.0)


def test_a_value_below_a_middle_is_not_rounded_up(dev):
    s = 8388609 * 2.0**-149
    x = torch.tensor([[127 * s, 12582913 * 2.0**-149]])  # the second is 1.49999994 s
    q, sc = G.int8_empty(1, 2, device=dev)
    G.int8_quantize(x.to(dev), q, sc)
    assert float(sc) == s and q.tolist() == [[127, 1]]


@pytest.mark.parametrize("top", TOPS)
def test_quantize_next_to_the_middles(dev, top):
    row = _row(top)
    x = torch.stack((row, -row, row.flip(0)))
    want = R.quantize(x)
    q, sc = G.int8_empty(*x.shape, device=dev)
    G.int8_quantize(x.to(dev), q, sc)
    assert torch.equal(sc.cpu(), want[1]) and torch.equal(q.cpu(), want[0])
    for M in (1, 3, 9):  # and where a layer's rows are quantised on the way
        xm = row.repeat(M, 1)
        b = torch.eye(len(row), dtype=torch.int8)  # each value's integer by itself
        w, _ = G.int8_empty(*b.shape, device=dev)
        w.copy_(b)
        y = torch.full((M, len(row)), math.nan, device=dev)
        G.int8_linear(xm.to(dev), (w, None), y, alpha=2.0**100)
        qm, sm = R.quantize(xm)
        assert torch.equal(y.cpu(), qm.float() * (sm * 2.0**100)[:, None])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n", [8388609, 9000001, 12345679, 16777213])
def test_with_factors(dev, dtype, n):
    """The middles of the integers, as they are in either type, times factors that are the scale and its neighbours."""
    s = torch.tensor(n * 2.0**-149)
    x = torch.cat((torch.tensor([127.0]), torch.arange(-127, 127) + 0.5)).repeat(6).to(dtype)[None].repeat(3, 1)
    c = torch.stack((s, torch.nextafter(s, torch.tensor(math.inf)), torch.nextafter(s, torch.tensor(0.0))))
    c = c[torch.arange(x.shape[1]) % 3]
    c[::255] = s
    want = R.quantize(x, c)
    q, sc = G.int8_empty(*x.shape, device=dev)
    G.int8_quantize(x.to(dev), q, sc, col_scale=c.to(dev))
    assert torch.equal(sc.cpu(), want[1]) and torch.equal(q.cpu(), want[0])
