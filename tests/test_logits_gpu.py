"""Token log-probabilities, entropy, top alternatives and distillation on the GPU, forward and backward, against the
64-bit restatements of lowbit_ref.py. Bounds: z = x / T takes two roundings (2 half-steps of |z|); lse = m + ln s has s
from at most 64 additions on a thread and a tree (under 128 half-steps relative, so absolute in ln s), each
term's exponent |z - m| times 3 half-steps, weighed by its share (|d| e^d <= 0.37 per unit, |d| at most 2 max|z|), and one
rounding of the sum. Chosen columns have to be equal."""
import math

import pytest
import torch

import gonngpu as G
from tests import lowbit_ref as R

pytestmark = pytest.mark.gpu

E = 2.0**-24  # half a step of fp32


def _say(*a):
    print(*a, flush=True)


def _logits(rows, cols, dtype, seed, masked=0.0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * spread
    if masked:
        x[torch.rand((rows, cols), generator=g) < masked] = -math.inf
    return x.to(dtype)


def _biggest(x, temperature):
    z = x.double().abs() / temperature
    return torch.where(torch.isfinite(z), z, 0.0).amax(1)


def _close(got, ref, bound):
    got, ref = got.cpu().double(), ref.double()
    special = ~torch.isfinite(ref)
    assert torch.equal(torch.nan_to_num(got, nan=1e300)[special], torch.nan_to_num(ref, nan=1e300)[special])
    bad = ((got - ref).abs() > bound) & ~special
    assert not bool(bad.any()), (got[bad][:4], ref[bad][:4])
    assert torch.equal(torch.isfinite(got), ~special)


def _forward(dev, x, targets, k, temperature, everything=True):
    rows = x.shape[0]
    new = lambda *s, dtype=torch.float32: torch.full(s, -77, dtype=dtype, device=dev)  # noqa: E731
    lp, lse, h = new(rows), new(rows), new(rows)
    ids, tops = (new(rows, k, dtype=torch.int64), new(rows, k)) if k else (None, None)
    G.token_logprobs(x, targets, lp, lse=lse if everything else None, entropy=h if everything else None, top_ids=ids,
                     top_logprobs=tops, temperature=temperature)
    return lp, lse, h, ids, tops


def _check_forward(dev, x, targets, k, temperature, xd=None):
    lp, lse, h, ids, tops = _forward(dev, x.to(dev) if xd is None else xd, targets.to(dev), k, temperature)
    r = R.logprobs(x, targets, k, temperature)
    big = _biggest(x, temperature)
    tol = E * (8 * big + 128)
    _close(lse, r[1], tol)
    _close(lp, r[0], 2 * tol)
    _close(h, r[2], E * (256 + 16 * big) * (1 + torch.nan_to_num(r[2])))
    if k:
        assert torch.equal(ids.cpu(), r[3])
        _close(tops, r[4], 2 * tol[:, None])
    return lse, h


SHAPES = [(1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 64, 64), (4, 100, 20), (7, 257, 1), (2, 1000, 64), (33, 777, 8), (3, 4099, 20),
          (2, 8191, 64), (2, 8193, 20), (1, 16384, 33), (2, 32771, 7), (1, 50257, 20), (2, 70001, 64), (1, 131072, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,k", SHAPES)
def test_logprobs(dev, rows, cols, k, dtype):
    _say("logprobs", rows, cols, k, dtype)
    x = _logits(rows, cols, dtype, rows + cols)
    targets = torch.arange(rows) * 7919 % cols
    targets[rows // 2] = cols - 1
    _check_forward(dev, x, targets, k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("masked", [0.5, 0.99])
@pytest.mark.parametrize("temperature", [0.3, 5.0])
def test_logprobs_masked_with_temperature(dev, dtype, masked, temperature):
    """Fewer columns left than alternatives asked for: the rest are -inf, lowest columns first."""
    for rows, cols, k in ((6, 300, 30), (3, 9000, 64), (2, 40000, 20)):
        x = _logits(rows, cols, dtype, cols, masked)
        x[:, 17] = 1.0
        x[1, :] = -math.inf
        x[1, cols - 1] = -3.0  # one column left
        _check_forward(dev, x, torch.tensor([17, 3, 17, 0, 5, 299][:rows]), k, temperature)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("cols", [70, 5000, 33000])
def test_special_rows(dev, dtype, cols):
    """Rows of -inf, with NaN, with +inf, of equal values, of the lowest value, ordered both ways; targets that
    are absent or past the end."""
    top = torch.finfo(dtype).max
    x = _logits(12, cols, dtype, 5)
    x[0] = -math.inf
    x[1, cols // 2] = math.nan
    x[2, cols - 1] = math.inf
    x[3] = 0.25
    x[4] = -top
    x[5] = torch.linspace(-4, 4, cols).to(dtype)
    x[6] = torch.linspace(4, -4, cols).to(dtype)
    x[7, ::2], x[7, 1::2] = 0.0, -0.0
    x[8] = -math.inf
    x[8, 3] = math.nan
    x[9] = torch.where(torch.arange(cols) % 64 == 5, 3.0, -3.0).to(dtype)  # the best in one lane's places
    x[10] = -top
    x[10, 40] = 2.0
    targets = torch.tensor([4, 1, cols - 1, 0, cols - 1, 2, -1, -5, 3, cols, 40, 2**40])
    _check_forward(dev, x, targets, 20, 1.0)
    _check_forward(dev, x, targets, 64, 1.0)
    _check_forward(dev, x, targets, 0, 1.0)


def test_many_equal_and_clustered_values(dev):
    """Values in few steps, and the largest ones side by side: the lowest columns come first in each."""
    g = torch.Generator().manual_seed(6)
    for cols in (900, 20000):
        x = torch.randint(0, 4, (6, cols), generator=g).float()
        x[1, 100:400] += torch.rand(300, generator=g) + 5
        x[2, -300:] += torch.arange(300) / 100 + 5
        x[3, ::256] = 9.0
        x[4, ::4] = 9.0
        for k in (1, 20, 64):
            _check_forward(dev, x, torch.zeros(6, dtype=torch.int64), k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_many_segments(dev, dtype):
    """A row of more segments than the joining kernel takes at a time, its best entries anywhere, in one place, and equal."""
    g = torch.Generator().manual_seed(21)
    for rows, cols in ((1, 300000), (600, 17000), (1, 2**20 + 3)):
        x = torch.randn((rows, cols), generator=g).to(dtype)
        if rows == 1:
            x = torch.cat((x, x, x, x))
            x[1, 2 * cols // 3 : 2 * cols // 3 + 100] = 6.0 + torch.arange(100).to(dtype) / 64
            x[2] = torch.arange(cols).to(dtype) if dtype == torch.float32 else torch.arange(cols).float().div(cols).to(dtype)
            x[3] = 0.5
        xd = x.to(dev)
        for k in (1, 64):
            ids, tops = torch.empty((len(x), k), dtype=torch.int64, device=dev), torch.empty((len(x), k), device=dev)
            G.token_logprobs(xd, None, None, top_ids=ids, top_logprobs=tops)
            want = torch.sort(x.float(), dim=1, descending=True, stable=True)
            assert torch.equal(ids.cpu(), want.indices[:, :k])
            z = x.double()
            lp = want.values[:, :k].double() - torch.logsumexp(z, 1, keepdim=True)
            assert bool(((tops.cpu().double() - lp).abs() <= E * (512 + 16 * z.abs().amax())).all())


def test_strides_offsets_and_optional_outputs(dev):
    for dtype in (torch.float32, torch.float16):
        base = _logits(30, 1203, dtype, 7).to(dev)
        x = base[2:29:3, 5:1202]
        assert x.data_ptr() % 16
        t = torch.arange(9) * 100
        _check_forward(dev, x.cpu(), t, 10, 1.0, x)
        lp, lse, h, _, _ = _forward(dev, x, t.to(dev), 0, 1.0, everything=False)
        assert bool((lse == -77).all()) and bool((h == -77).all())
        ids, tops = torch.empty((9, 3), dtype=torch.int64, device=dev), torch.empty((9, 3), device=dev)
        G.token_logprobs(x, None, None, top_ids=ids, top_logprobs=tops)
        assert torch.equal(ids.cpu(), R.logprobs(x.cpu(), t, 3, 1.0)[3])
    e = torch.empty((0, 50), device=dev)
    G.token_logprobs(e, torch.empty(0, dtype=torch.int64, device=dev), e[:, 0])


def _grad_bound(ref, x, scale, temperature, dtype):
    """p's relative error is its exponent's absolute one (z, lse and their difference), times the size of what it is multiplied with."""
    z = x.double() / temperature
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    big = _biggest(x, temperature)[:, None]
    out = torch.finfo(dtype).eps / 2 * ref.abs() + (2.0**-25 if dtype == torch.float16 else 1e-44)
    return p * scale * E * (64 + 20 * big + 4 * lse.abs() + 256) * (1 + torch.where(p > 0, (z - lse).abs(), 0.0)) + 8 * E * ref.abs() + out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("exponent", [-2, -7, -12, -20, -100])
@pytest.mark.parametrize("cols", [50, 3000])
def test_small_temperatures(dev, cols, exponent, dtype):
    """Large logits over small temperatures: m / T is past what fp32 holds ln s beside, or past any use of it, and the
    log-probabilities are those of the differences to the maximum, which are exact here. Each has a few half-steps of its own, and
    ln s no more than 160."""
    x = _logits(4, cols, torch.float32, cols, spread=20.0).round()
    x[0] += 60000
    x[1] -= 50000
    x[2, cols // 2:] = x[2].amax()  # many equal ones
    x[3, 1] = x[3, cols - 1] = 65000  # two
    x = x.to(dtype)
    temperature, targets = 2.0**exponent, torch.tensor([0, 1, cols - 1, 1])
    lp, lse, h, ids, tops = _forward(dev, x.to(dev), targets.to(dev), 3, temperature)
    # 64 bits have no room either for ln s beside m / T (2^116 has steps of 2^63): of the differences, which are exact.
    m = x.double().amax(1)
    r = R.logprobs(x.double() - m[:, None], targets, 3, temperature)
    _close(lp, r[0], E * (4 * r[0].abs() + 160))
    _close(lse, m / temperature + r[1], E * (4 * (m / temperature + r[1]).abs() + 160))
    _close(h, r[2], E * 512 * (1 + r[2]))
    assert torch.equal(ids.cpu(), r[3])
    _close(tops, r[4], E * (4 * r[4].abs() + 160))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 3), (5, 100), (4, 1001), (3, 8192), (2, 40003)])
def test_logprobs_backward(dev, rows, cols, dtype):
    for temperature, masked in ((1.0, 0.0), (2.5, 0.6)):
        x = _logits(rows, cols, dtype, rows * cols, masked if cols > 50 else 0.0)
        targets = torch.arange(rows) * 31 % cols
        x[torch.arange(rows), targets] = 0.5
        if rows > 2:
            targets[2] = -1
        g = torch.Generator().manual_seed(8)
        gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
        lse, h = _check_forward(dev, x, targets, 0, temperature)
        xd = x.to(dev)
        dx = torch.full((rows, cols), 9.0, dtype=dtype, device=dev)
        G.token_logprobs_backward(xd, targets.to(dev), lse, gl.to(dev), dx, entropy=h, grad_entropy=gh.to(dev), temperature=temperature)
        entropy = torch.nan_to_num(h.cpu().double())[:, None]
        scale = (gl.abs() + gh.abs())[:, None].double() * (1 + entropy) / temperature

        def check(got, ref):  # the result's own rounding is relative to the result: a bound for each
            bound = _grad_bound(ref, x, scale, temperature, dtype)
            bound[torch.arange(rows), targets.clamp_min(0)] += 8 * E * gl.abs().double() / temperature
            _close(got, ref, bound)

        check(dx, R.logprobs_grad(x, targets, gl, gh, temperature))
        # one of the two gradients alone; in place
        G.token_logprobs_backward(xd, targets.to(dev), lse, gl.to(dev), dx, temperature=temperature)
        check(dx, R.logprobs_grad(x, targets, gl, 0 * gh, temperature))
        G.token_logprobs_backward(xd, None, lse, None, xd, entropy=h, grad_entropy=gh.to(dev), temperature=temperature)
        check(xd, R.logprobs_grad(x, -torch.ones(rows, dtype=torch.int64), gl, gh, temperature))


def test_logprobs_gradient_against_differences(dev):
    """d/dx of sum(gl logprob + gh entropy) by central differences of the 64-bit forward."""
    rows, cols, temperature = 3, 12, 1.7
    x = _logits(rows, cols, torch.float32, 9)
    t, g = torch.tensor([0, 11, 5]), torch.Generator().manual_seed(10)
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    lse, h = _check_forward(dev, x, t, 0, temperature)
    dx = torch.empty((rows, cols), device=dev)
    G.token_logprobs_backward(x.to(dev), t.to(dev), lse, gl.to(dev), dx, entropy=h, grad_entropy=gh.to(dev), temperature=temperature)

    def f(y):
        lp, _, hh, _, _ = R.logprobs(y, t, 0, temperature)
        return (gl * lp + gh * hh).sum()

    step = 1e-5  # the differences are off by step^2 times third derivatives of about 1, and 1e-16 / step
    for r in range(rows):
        for c in range(cols):
            d = torch.zeros(rows, cols, dtype=torch.float64)
            d[r, c] = step
            assert abs((f(x.double() + d) - f(x.double() - d)) / (2 * step) - dx[r, c].item()) < 1e-5


def test_backward_of_special_rows(dev):
    for cols in (60, 20000):
        x = _logits(8, cols, torch.float32, 11)
        x[0] = -math.inf
        x[1, 3] = math.nan
        x[2, 3] = math.inf
        x[4, 5] = math.nan
        t = torch.tensor([1, 1, 1, cols, 1, -1, 2, 3], device=dev)
        lp, lse, h, _, _ = _forward(dev, x.to(dev), t, 0, 1.0)
        gl = torch.tensor([1.0, 1, 1, 1, 0, 1, 1, 1], device=dev)
        dx = torch.empty((8, cols), device=dev)
        G.token_logprobs_backward(x.to(dev), t, lse, gl, dx)
        dx = dx.cpu()
        assert bool((dx[0] == 0).all()) and bool((dx[4] == 0).all()) and bool((dx[5] == 0).all())
        assert bool(torch.isnan(dx[1:4]).all())
        assert bool(torch.isfinite(dx[6:]).all()) and bool((dx[6:].abs().sum(1) > 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("cols", [100, 20000])
def test_rows_of_the_lowest_value(dev, cols, dtype):
    """A mask of the type's lowest value that leaves no column: the log-probabilities are those of equal logits (lse has
    no room for ln cols beside the lowest fp32 value), and the gradient does not take 1 for each p."""
    low = torch.finfo(dtype).min
    x = torch.full((2, cols), low, dtype=dtype)
    x[1, 7] = 1.0
    t = torch.tensor([3, 7], device=dev)
    lp, lse, h, ids, tops = _forward(dev, x.to(dev), t, 5, 1.0)
    ln = math.log(cols)
    # fp16: x - m and its product with T's reciprocal are exact here; ln s has the roundings of a sum and a logarithm
    assert abs(lp[0].item() + ln) <= 256 * E * (1 + ln) and abs(h[0].item() - ln) <= 512 * E * (1 + ln)
    assert abs(lp[1].item()) <= 256 * E and ids.tolist() == [[0, 1, 2, 3, 4], [7, 0, 1, 2, 3]]
    assert float((tops[0].cpu() + ln).abs().max()) <= 256 * E * (1 + ln)
    g, dx = torch.ones(2, device=dev), torch.empty((2, cols), dtype=dtype, device=dev)
    G.token_logprobs_backward(x.to(dev), t, lse, g, dx)
    if dtype == torch.float32:
        assert bool((dx[0] == 0).all())
    else:  # lse is off by half a step at 65504: 2^-9, and p by as much relatively
        want = torch.full((cols,), -1.0 / cols, dtype=torch.float64)
        want[3] += 1
        assert bool(((dx[0].cpu().double() - want).abs() <= 2.0**-8 / cols + 2.0**-11 * want.abs() + 2.0**-25).all())
    want = torch.zeros(cols, dtype=torch.float64)  # one column left: p = 1 there
    assert bool(((dx[1].cpu().double() - want).abs() <= 512 * E).all())
    loss = torch.empty(2, device=dev)
    ids, teacher = torch.tensor([[1, 2], [7, 7]], device=dev), torch.zeros((2, 2), device=dev)
    G.distill(x.to(dev), ids, teacher, loss, lse=lse)
    assert abs(loss[0].item() - (ln - math.log(2))) <= 512 * E * (1 + ln) and abs(loss[1].item() + math.log(2)) <= 512 * E
    G.distill_backward(x.to(dev), ids, teacher, lse, g, dx)
    if dtype == torch.float32:
        want[1:3] = -0.5
        assert bool((dx[0].cpu().double() == want).all())
    assert bool((dx[1].abs() <= 512 * E).all())


def _teacher(rows, cols, k, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(cols, generator=g)[:k] if k <= cols else torch.randint(0, cols, (k,), generator=g) for _ in range(rows)])
    return ids, torch.randn((rows, k), generator=g) * 2 + 5


def _check_distill(dev, x, ids, t, temperature, in_place=False):
    rows, cols = x.shape
    loss, lse = torch.full((rows,), -7.0, device=dev), torch.full((rows,), -7.0, device=dev)
    xd = x.to(dev)
    G.distill(xd, ids.to(dev), t.to(dev), loss, lse=lse, temperature=temperature)
    r = R.distill(x, ids, t, temperature)
    big = _biggest(x, temperature)
    tol = E * (8 * big + 128)
    _close(lse, r[1], tol)
    # sum of p (ln p - z + lse): p to 64 half-steps, the bracket to lse's and ln p's errors
    bracket = big + r[1].abs() + _biggest(t, temperature) * 2 + 8
    _close(loss, r[0], temperature**2 * (3 * tol + E * 300 * bracket))
    g = torch.linspace(-1.5, 2, rows)
    dx = xd if in_place else torch.full(x.shape, 3.0, dtype=x.dtype, device=dev)
    G.distill_backward(xd, ids.to(dev), t.to(dev), lse, g.to(dev), dx, temperature=temperature)
    ref = r[2] * g.double()[:, None]
    scale = (g.abs().double() * temperature)[:, None]
    w = torch.zeros(x.shape, dtype=torch.float64)
    w.scatter_add_(1, ids.clamp_min(0), torch.ones_like(ids).double())
    bound = _grad_bound(ref, x, scale, temperature, x.dtype) + (w > 0) * scale * E * (300 + 8 * _biggest(t, temperature))[:, None]
    _close(dx, ref, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (2, 5, 3), (3, 100, 64), (4, 1001, 256), (2, 8192, 20), (3, 8200, 1), (2, 50257, 64)])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_distill(dev, rows, cols, k, temperature, dtype):
    x = _logits(rows, cols, dtype, cols + k)
    _check_distill(dev, x, *_teacher(rows, cols, k, k), temperature)
    _check_distill(dev, x, *_teacher(rows, cols, k, k), temperature, in_place=True)


@pytest.mark.parametrize("exponent", [-2, -20, -100])
def test_distill_small_temperatures(dev, exponent):
    """Quotients that fp32 holds only as differences to the maximum; these are exact, each ln p has two roundings of its own and 160
    half-steps of ln s, and a term its p's 160 and a rounding."""
    T, x = 2.0**exponent, _logits(3, 500, torch.float16, 1, spread=30.0).round() + 40000
    ids, t = _teacher(3, 500, 6, 2)
    t = (t * 8).round() + 1e6
    loss = torch.empty(3, device=dev)
    G.distill(x.to(dev), ids.to(dev), t.to(dev), loss, temperature=T)
    t = t.double() - torch.where(ids >= 0, t, -math.inf).amax(1, keepdim=True).double()
    x = x.double() - x.double().amax(1, keepdim=True)
    size = T * T * ((t.abs() + torch.gather(x, 1, ids.clamp_min(0)).abs()) / T + 8).amax(1)
    _close(loss, R.distill(x, ids, t, T)[0], E * 6 * 400 * size)


def test_distill_absent_and_repeated_entries(dev):
    for cols in (40, 30000):
        x = _logits(6, cols, torch.float32, 12)
        ids, t = _teacher(6, cols, 9, 13)
        ids[0] = -1  # none present
        ids[1, 1:] = -1  # one
        ids[2, ::2] = -3
        t[3, 2] = -math.inf
        ids[4, :] = ids[4, 0]  # the same column throughout
        ids[5, 3] = ids[5, 7]
        t[0, 0] = math.nan  # an absent entry's logit is not looked at
        _check_distill(dev, x, ids, t, 1.5)
        _check_distill(dev, x, ids, t, 1.5, in_place=True)


def test_distill_special_rows(dev):
    for cols in (50, 30000):
        x = _logits(8, cols, torch.float32, 14)
        ids, t = _teacher(8, cols, 5, 15)
        x[0, ids[0, 1]] = -math.inf  # the student rules out what the teacher names
        x[1] = -math.inf
        x[2, 3] = math.nan
        ids[3, 2] = cols
        t[4, 1] = math.nan
        t[5, 0] = math.inf
        x[6, (ids[6, 0] + 1) % cols] = -math.inf if int((ids[6, 0] + 1) % cols) not in ids[6].tolist() else 0.0
        loss, lse = torch.empty(8, device=dev), torch.empty(8, device=dev)
        G.distill(x.to(dev), ids.to(dev), t.to(dev), loss, lse=lse)
        loss = loss.cpu()
        assert loss[0] == math.inf and loss[1] == math.inf
        assert bool(torch.isnan(loss[2:6]).all()) and bool(torch.isfinite(loss[6:]).all())
        dx, g = torch.empty((8, cols), device=dev), torch.ones(8, device=dev)
        g[5] = 0.0
        G.distill_backward(x.to(dev), ids.to(dev), t.to(dev), lse, g, dx)
        dx = dx.cpu()
        p = torch.softmax(t[1].double(), 0)
        assert bool(torch.isfinite(dx[0]).all())
        want = torch.zeros(cols, dtype=torch.float64).index_add_(0, ids[1], -p)  # q = 0
        assert bool(((dx[1].double() - want).abs() <= 64 * E).all())
        assert bool(torch.isnan(dx[2:5]).all()) and bool((dx[5] == 0).all()) and bool(torch.isfinite(dx[6:]).all())


def test_distill_gradient_against_differences(dev):
    rows, cols, k, temperature = 2, 11, 4, 1.3
    x = _logits(rows, cols, torch.float32, 16)
    ids, t = _teacher(rows, cols, k, 17)
    loss, lse, dx = torch.empty(rows, device=dev), torch.empty(rows, device=dev), torch.empty((rows, cols), device=dev)
    G.distill(x.to(dev), ids.to(dev), t.to(dev), loss, lse=lse, temperature=temperature)
    G.distill_backward(x.to(dev), ids.to(dev), t.to(dev), lse, torch.ones(rows, device=dev), dx, temperature=temperature)
    step = 1e-5
    for r in range(rows):
        for c in range(cols):
            d = torch.zeros(rows, cols, dtype=torch.float64)
            d[r, c] = step
            up, down = (R.distill(x.double() + s * d, ids, t, temperature)[0].sum() for s in (1, -1))
            assert abs((up - down) / (2 * step) - dx[r, c].item()) < 1e-5


def test_captured_and_replayed(dev):
    """Two graphs and eager calls over the same inputs keep out of each other's workspaces."""
    rows, cols, k = 3, 40001, 20
    x = _logits(rows, cols, torch.float32, 18).to(dev)
    t = torch.tensor([1, 2, 3], device=dev)
    ids, tl = (v.to(dev) for v in _teacher(rows, cols, 8, 19))
    new = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device=dev)  # noqa: E731

    def make():
        lp, lse, h, ti, tp, loss, lse2, dx, dx2 = new(rows), new(rows), new(rows), new(rows, k, dtype=torch.int64), new(rows, k), new(rows), new(rows), new(rows, cols), new(rows, cols)
        g = torch.ones(rows, device=dev)

        def step():
            G.token_logprobs(x, t, lp, lse=lse, entropy=h, top_ids=ti, top_logprobs=tp)
            G.token_logprobs_backward(x, t, lse, g, dx, entropy=h, grad_entropy=g)
            G.distill(x, ids, tl, loss, lse=lse2)
            G.distill_backward(x, ids, tl, lse2, g, dx2)

        return step, (lp, lse, h, ti, tp, loss, lse2, dx, dx2)

    (eager, want), (one, got1), (two, got2) = make(), make(), make()
    for f in (eager, one, two):
        f()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        one()
    with torch.cuda.graph(g2):
        two()
    for i in range(3):
        x.copy_(_logits(rows, cols, torch.float32, 40 + i))
        eager()
        for v in got1 + got2:
            v.fill_(0)
        g1.replay()
        eager()
        g2.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, got1, got2):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_streams(dev):
    x = _logits(2, 60000, torch.float16, 20).to(dev)
    t = torch.tensor([5, 59999], device=dev)
    want = _forward(dev, x, t, 20, 1.0)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    lp, ids, tops = torch.zeros(2, device=dev), torch.zeros((2, 20), dtype=torch.int64, device=dev), torch.zeros((2, 20), device=dev)
    torch.cuda.synchronize()
    G.token_logprobs(x, t, lp, top_ids=ids, top_logprobs=tops, stream_ptr=other.cuda_stream)
    other.synchronize()
    assert torch.equal(lp, want[0]) and torch.equal(ids, want[3]) and torch.equal(tops, want[4])
    # Calls on two streams at once, each with a workspace of its own stream's.
    x2 = _logits(2, 60000, torch.float16, 22).to(dev)
    want2 = _forward(dev, x2, t, 20, 1.0)
    lp2, ids2, tops2 = torch.zeros(2, device=dev), torch.zeros((2, 20), dtype=torch.int64, device=dev), torch.zeros((2, 20), device=dev)
    torch.cuda.synchronize()
    for _ in range(50):
        G.token_logprobs(x, t, lp, top_ids=ids, top_logprobs=tops, stream_ptr=other.cuda_stream)
        G.token_logprobs(x2, t, lp2, top_ids=ids2, top_logprobs=tops2)
    torch.cuda.synchronize()
    assert torch.equal(ids, want[3]) and torch.equal(tops, want[4]) and torch.equal(lp, want[0])
    assert torch.equal(ids2, want2[3]) and torch.equal(tops2, want2[4]) and torch.equal(lp2, want2[0])
    G.token_logprobs(x, t, lp, top_ids=ids, top_logprobs=tops, stream_ptr=0)  # the library's stream
    G.synchronize()
    assert torch.equal(ids, want[3]) and torch.equal(lp, want[0])
    lp.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.default_stream()):
        G.token_logprobs(x, t, lp, top_ids=ids, top_logprobs=tops)
        assert torch.equal(lp, want[0]) and torch.equal(ids, want[3])


def test_offsets_past_32_bits(dev):
    """More than 2^32 bytes and 2^31 values of logits, forward and backward."""
    rows, cols = 17000, 131072
    x = torch.empty((rows, cols), dtype=torch.float16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    t = (torch.arange(rows, device=dev) * 97) % cols
    lp, lse, h, ids, tops = _forward(dev, x, t, 5, 1.0)
    pick = torch.tensor([0, 1, 16383, 16384, 16999])
    xs = x[pick.to(dev)].cpu()
    r = R.logprobs(xs, t.cpu()[pick], 5, 1.0)
    tol = E * (8 * _biggest(xs, 1.0) + 128)
    _close(lse[pick.to(dev)], r[1], tol)
    _close(lp[pick.to(dev)], r[0], 2 * tol)
    assert torch.equal(ids[pick.to(dev)].cpu(), r[3])
    tid, tl = (v.to(dev) for v in (torch.randint(0, cols, (rows, 4)), torch.randn(rows, 4)))
    loss = torch.empty(rows, device=dev)
    G.distill(x, tid, tl, loss, lse=lse)
    _close(lse[pick.to(dev)], r[1], tol)
    gl = torch.full((rows,), 2048.0, device=dev)
    G.distill_backward(x, tid, tl, lse, gl, x)
    ref = R.distill(xs, tid.cpu()[pick], tl.cpu()[pick], 1.0)[2] * 2048.0
    scale = torch.full((5, 1), 2048.0, dtype=torch.float64)
    bound = _grad_bound(ref, xs, scale, 1.0, torch.float16)
    bound.scatter_add_(1, tid.cpu()[pick], torch.full((5, 4), 2048.0 * 400 * E, dtype=torch.float64))
    _close(x[pick.to(dev)], ref, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("cols", [1, 2, 64, 5000, 33000])
def test_nan_in_the_first_column(dev, cols, dtype):
    """NaN is the largest value in column 0 as in any other: alone, among numbers, beside other NaN, and where all are NaN. Every
    column named is one of the row's."""
    x = _logits(5, cols, dtype, 23)
    x[0, 0] = math.nan
    x[1] = math.nan
    x[2, 0] = x[2, cols // 2] = x[2, cols - 1] = math.nan
    x[3, 0], x[3, cols - 1] = -math.nan, math.inf
    targets = torch.tensor([0, cols - 1, 0, cols // 2, 0])
    for k in {1, min(cols, 5), min(cols, 64)}:
        _check_forward(dev, x, targets, k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_smallest_and_largest_temperatures(dev, dtype):
    """The ends of what is accepted: one column is left at the smallest, all are equally likely at the largest."""
    x = torch.tensor([[-3.0, 2.0, -5.0, 1.5, -math.inf], [-8.0, -4.0, -6.0, -4.5, -5.0]]).to(dtype)
    lp, lse, h, ids, tops = _forward(dev, x.to(dev), torch.tensor([1, 1], device=dev), 2, 4.3e-39)
    assert lp.tolist() == [0.0, 0.0] and h.tolist() == [0.0, 0.0] and ids.tolist() == [[1, 3], [1, 3]]
    assert tops[:, 0].tolist() == [0.0, 0.0] and bool((tops[:, 1] < -1e37).all())
    lp, lse, h, ids, tops = _forward(dev, x.to(dev), torch.tensor([1, 1], device=dev), 2, 3.4e38)
    for r, n in enumerate((4, 5)):
        assert abs(lp[r].item() + math.log(n)) <= 32 * E and abs(h[r].item() - math.log(n)) <= 64 * E


def test_infinite_loss_where_the_teacher_probability_underflows(dev):
    """A present entry whose logit the student rules out: +inf however small p is."""
    for cols in (40, 30000):
        for dtype in (torch.float32, torch.float16):
            x = _logits(4, cols, dtype, 24)
            ids, t = _teacher(4, cols, 3, 25)
            t[:, 0] = 0.0
            t[:3, 1] = torch.tensor([-200.0, -3e38, -100.0])
            x[0, ids[0, 1]] = x[1, ids[1, 1]] = x[2, ids[2, 1]] = -math.inf
            t[2, 1] = -math.inf  # absent: not looked at
            t[3, 1] = -200.0  # ruled out by nobody
            loss = torch.empty(4, device=dev)
            G.distill(x.to(dev), ids.to(dev), t.to(dev), loss)
            loss = loss.cpu()
            assert loss[0] == math.inf and loss[1] == math.inf
            r = R.distill(x[2:], ids[2:], t[2:], 1.0)[0]
            assert bool(((loss[2:].double() - r).abs() <= E * 2000 * (1 + r.abs())).all())


def _far_rows(rows, cols, dtype, seed):
    """Integers (so that differences to the maximum are exact) far from 0, on both sides of it."""
    x = _logits(rows, cols, torch.float32, seed, spread=20.0).round()
    x += torch.where(torch.arange(rows) % 2 == 0, 40000.0, -40000.0)[:, None]
    x[rows // 2, cols // 2:] = x[rows // 2].amax()  # many equal ones
    if cols > 10:
        x[:, 3:cols:7] = -math.inf
    return x.to(dtype)


def _far_bound(ref, x, scale, temperature, dtype):
    """p = 2^((x - m) c - log2 s) from the exact x - m: half-steps of c, of the product and of the subtraction (4 |z|), of ln s
    (160) and of the forward's entropy (512), and a few of the exponential's and the products'; p below 2^-126 is 0."""
    z = x / temperature
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = torch.where(torch.isneginf(z), 0.0, z - lse)
    p = torch.exp(z - lse)
    out = torch.finfo(dtype).eps / 2 * ref.abs() + (2.0**-25 if dtype == torch.float16 else 1e-44)
    return scale * (p * E * (800 + 4 * lp.abs()) * (1 + lp.abs()) + 2.0**-126 * 100) + 8 * E * ref.abs() + out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("exponent", [0, -2, -7, -12, -20, -100, -115, 3])
@pytest.mark.parametrize("rows,cols", [(2, 1), (4, 50), (3, 3000), (2, 70001), (600, 9000)])
def test_gradients_of_rows_far_from_zero(dev, rows, cols, exponent, dtype):
    """Large logits, small temperatures: lse has no room for ln s (at the last temperature it is infinite), and the gradients are
    those of the differences to the maximum, as the log-probabilities are. Both operators, in place too."""
    _say("far gradients", rows, cols, exponent, dtype)
    if rows == 600 and exponent not in (-7, -100):
        return
    x, temperature = _far_rows(rows, cols, dtype, cols + rows), 2.0**exponent
    d = x.double() - x.double().amax(1, keepdim=True)
    best = d.argmax(1)
    targets = torch.where(torch.arange(rows) % 3 == 1, (best + cols // 2) % cols, best)
    targets[-1] = -1
    g = torch.Generator().manual_seed(27)
    gl, gh = torch.randn(rows, generator=g) * temperature, torch.randn(rows, generator=g) * temperature
    xd, td = x.to(dev), targets.to(dev)
    lp, lse, h, _, _ = _forward(dev, xd, td, 0, temperature)
    assert bool((lse.abs() >= 4000).all())
    r = R.logprobs_grad(d, targets, gl, gh, temperature)
    scale = ((gl.abs() + gh.abs()).double() * (1 + R.logprobs(d, targets, 0, temperature)[2]) / temperature)[:, None] if rows < 600 else \
        ((gl.abs() + gh.abs()).double() * 11 / temperature)[:, None]  # an entropy of at most ln 9000
    bound = _far_bound(r, d, scale, temperature, dtype)
    at = torch.zeros_like(bound).scatter_(1, targets.clamp_min(0)[:, None], 1.0)
    bound += 16 * E * at * (gl.abs().double() / temperature)[:, None]
    dx = torch.full((rows, cols), 9.0, dtype=dtype, device=dev)
    G.token_logprobs_backward(xd, td, lse, gl.to(dev), dx, entropy=h, grad_entropy=gh.to(dev), temperature=temperature)
    _close(dx, r, bound)
    mine = xd.clone()
    G.token_logprobs_backward(mine, td, lse, gl.to(dev), mine, entropy=h, grad_entropy=gh.to(dev), temperature=temperature)
    assert torch.equal(mine, dx)

    k = min(cols, 5)
    ids = torch.stack([torch.randperm(cols, generator=g)[:k] for _ in range(rows)])
    ids[0, k - 1] = -1 if k > 1 else 0
    t = (torch.randn((rows, k), generator=g) * 2 * temperature).clamp(-1e30, 1e30)
    loss, gd = torch.empty(rows, device=dev), torch.linspace(-1.5, 2, rows) / temperature
    G.distill(xd, ids.to(dev), t.to(dev), loss, lse=lse, temperature=temperature)
    r = R.distill(d, ids, t, temperature)[2] * gd.double()[:, None]
    scale = (gd.abs().double() * temperature)[:, None]
    bound = _far_bound(r, d, scale, temperature, dtype)
    bound += 400 * E * scale * torch.zeros_like(bound).scatter_(1, ids.clamp_min(0), 1.0)
    G.distill_backward(xd, ids.to(dev), t.to(dev), lse, gd.to(dev), dx, temperature=temperature)
    _close(dx, r, bound)
    G.distill_backward(xd, ids.to(dev), t.to(dev), lse, gd.to(dev), xd, temperature=temperature)
    assert torch.equal(xd, dx)


def test_gradients_of_masked_rows_at_any_temperature(dev):
    """Rows of nothing but -inf or fp32's lowest value have gradient 0 (distillation: q = 0) whatever the temperature; NaN and +inf
    stay NaN, a row whose gradients are 0 is 0."""
    low = torch.finfo(torch.float32).min
    for cols in (60, 20000):
        x = torch.full((5, cols), low)
        x[1] = -math.inf
        x[2] = 40000.0
        x[2, 1] = math.nan
        x[3, 1] = math.inf
        x[4] = math.nan
        for temperature in (1.0, 1e-6, 1e10, 1e30):
            t = torch.tensor([3, 1, 2, 1, 0], device=dev)
            lp, lse, h, _, _ = _forward(dev, x.to(dev), t, 0, temperature)
            g = torch.tensor([1.0, 1, 1, 1, 0], device=dev)
            dx = torch.empty((5, cols), device=dev)
            G.token_logprobs_backward(x.to(dev), t, lse, g, dx, temperature=temperature)
            assert bool((dx[:2] == 0).all()) and bool(torch.isnan(dx[2:4]).all()) and bool((dx[4] == 0).all())
            ids, teacher = torch.tensor([[1, 2]] * 5, device=dev), torch.zeros((5, 2), device=dev)
            G.distill_backward(x.to(dev), ids, teacher, lse, g / temperature, dx, temperature=temperature)
            want = torch.zeros(cols)
            want[1:3] = -0.5
            dx = dx.cpu()
            assert bool(((dx[:2] - want).abs() <= 4 * E).all()) and bool(torch.isnan(dx[2:4]).all()) and bool((dx[4] == 0).all())


@pytest.mark.parametrize("cols", [300, 21000])
def test_far_rows_strided_repeated_and_captured(dev, cols):
    """Far rows and near ones side by side in a strided view at odd addresses, into one of another stride; repeated and absent
    entries; rows without a gradient; the same from a graph, replayed with other rows far."""
    rows, T = 20, 0.5
    g = torch.Generator().manual_seed(30)
    for dtype in (torch.float32, torch.float16):
        base, out = torch.zeros((2 * rows, cols + 7), dtype=dtype, device=dev), torch.full((rows, cols + 3), 7.0, dtype=dtype, device=dev)
        xd, dx = base[::2, 3:3 + cols], out[:, 1:1 + cols]
        ids = torch.randint(0, cols, (rows, 6), generator=g)
        ids[:, 4] = ids[:, 2]
        ids[1] = -1
        ids[2, 0] = -7
        t, gd = torch.randn((rows, 6), generator=g), torch.randn(rows, generator=g)
        gd[[3, 4]] = 0.0
        targets = torch.randint(0, cols, (rows,), generator=g)
        targets[5] = -1
        new = lambda: torch.empty(rows, device=dev)  # noqa: E731
        lse, lp, loss, l1, l2 = new(), new(), new(), torch.empty_like(dx), torch.empty_like(dx)
        td, idd, tld, gdd = targets.to(dev), ids.to(dev), t.to(dev), gd.to(dev)

        def step():
            G.token_logprobs(xd, td, lp, lse=lse, temperature=T)
            G.token_logprobs_backward(xd, td, lse, gdd, dx, temperature=T)
            l1.copy_(dx)
            G.distill(xd, idd, tld, loss, lse=lse, temperature=T)
            G.distill_backward(xd, idd, tld, lse, gdd, dx, temperature=T)
            l2.copy_(dx)

        def check(x):
            d = x.double() - x.double().amax(1, keepdim=True)
            none = torch.zeros(rows)
            scale = (gd.abs().double() / T)[:, None]
            hot = torch.zeros((rows, cols), dtype=torch.float64).scatter_(1, targets.clamp_min(0)[:, None], 1.0)
            r = R.logprobs_grad(d, targets, gd, none, T)
            # near rows: lse is off by half a step of 512
            near = 2.0**-16 * torch.softmax(d / T, 1)
            _close(l1, r, _far_bound(r, d, scale, T, dtype) + scale * (near + 16 * E * hot))
            r = R.distill(d, ids, t, T)[2] * gd.double()[:, None]
            hot = torch.zeros((rows, cols), dtype=torch.float64).scatter_(1, ids.clamp_min(0), 1.0)
            scale = (gd.abs().double() * T)[:, None]
            _close(l2, r, _far_bound(r, d, scale, T, dtype) + scale * (near + 1200 * E * hot))
            assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + cols:] == 7).all())

        def fill(first):
            x = _logits(rows, cols, dtype, 31 + first).round()
            x[first::3] = (x[first::3].float() + 2048).to(dtype)
            xd.copy_(x)
            return x

        x = fill(0)
        step()
        check(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for first in (1, 2, 0):
            x = fill(first)
            l1.zero_()
            l2.zero_()
            graph.replay()
            torch.cuda.synchronize()
            check(x)
            step()
