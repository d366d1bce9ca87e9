"""The operators together, as they are used: an int8 layer gives a batch's logits, they are adjusted by what was said so far
and what a grammar allows, the sampler's alternatives and the log-probabilities of its tokens are taken, and in training the
gradient goes back through all of it to the layer's inputs. Each step is compared with the definition on what the step before
it gave, bit for bit or with bounds from the roundings of its own sums; and the step's slope with differences in 64 bits."""
import math

import pytest
import torch

import gonngpu as G
from tests import int8_ref as I8
from tests import lowbit_ref as R
from tests.test_adjust_gpu import _same, _words

pytestmark = pytest.mark.gpu

E = 2.0**-24


@pytest.mark.parametrize("rows,inputs,vocab,h,k", [(1, 96, 500, 9, 5), (24, 320, 3001, 60, 20), (130, 256, 9000, 30, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_sampling_and_training_step_of_an_int8_layer(dev, rows, inputs, vocab, h, k, dtype):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((rows, inputs), generator=g).to(dtype)
    w = torch.randn((vocab, inputs), generator=g) * 3 / math.sqrt(inputs)
    new = lambda *s, dtype=torch.float32: torch.full(s, -5, dtype=dtype, device=dev)  # noqa: E731

    # The layer's weights in 8 bits, once as they are multiplied and once transposed for the gradient.
    wq, ws = G.int8_empty(vocab, inputs, device=dev)
    G.int8_quantize(w.to(dev), wq, ws)
    ref_w = I8.quantize(w)
    assert torch.equal(wq.cpu(), ref_w[0]) and torch.equal(ws.cpu(), ref_w[1])
    wt, _ = G.int8_empty(inputs, vocab, device=dev)
    wt.copy_(wq.t())

    logits = new(rows, vocab)
    G.int8_linear(x.to(dev), (wq, ws), logits)
    assert torch.equal(logits.cpu(), I8.product(*I8.quantize(x), *ref_w))

    # What the sampler sees.
    kw = dict(history=torch.randint(-1, vocab, (rows, h), generator=g), repetition=1.0 + torch.rand(rows, generator=g),
              mask=_words(rows, vocab, 0.7, 3))
    more = dict(prompt=torch.randint(0, h, (rows,), generator=g), frequency=torch.rand(rows, generator=g), presence=torch.rand(rows, generator=g),
                bias_ids=torch.randint(0, vocab, (rows, 7), generator=g), bias=torch.randn((rows, 7), generator=g))
    kwd, mored = ({a: t.to(dev) for a, t in d.items()} for d in (kw, more))
    seen = new(rows, vocab)
    G.adjust_logits(logits, seen, **kwd, **mored)
    assert _same(seen, I8.adjust(logits.cpu(), **kw, **more))

    temperature = 0.8
    ids, tops, lse, ent, lp = new(rows, k, dtype=torch.int64), new(rows, k), new(rows), new(rows), new(rows)
    targets = seen.argmax(1)
    G.token_logprobs(seen, targets, lp, lse=lse, entropy=ent, top_ids=ids, top_logprobs=tops, temperature=temperature)
    ref = R.logprobs(seen.cpu(), targets.cpu(), k, temperature)
    assert torch.equal(ids.cpu(), ref[3]) and torch.equal(ids[:, 0], targets)
    fine = seen.cpu()[torch.isfinite(seen.cpu())]
    big = float(fine.abs().max()) / temperature + 16
    for got, want in ((lp, ref[0]), (lse, ref[1]), (tops, ref[4])):
        assert bool(((got.cpu().double() - want).abs() <= 400 * E * big).all())

    # And back: to the adjusted logits, to the layer's outputs, to its inputs.
    gl = torch.randn(rows, generator=g)
    d_seen, d_logits, dx = new(rows, vocab), new(rows, vocab), new(rows, inputs)
    G.token_logprobs_backward(seen, targets, lse, gl.to(dev), d_seen, temperature=temperature)
    ref_d = R.logprobs_grad(seen.cpu(), targets.cpu(), gl, torch.zeros(rows), temperature)
    assert bool(((d_seen.cpu().double() - ref_d).abs() <= 800 * E * big * ref_d.abs().amax(1, keepdim=True)).all())
    G.adjust_logits_backward(logits, d_seen, d_logits, **kwd)
    assert _same(d_logits, I8.adjust_grad(logits.cpu(), d_seen.cpu(), **kw))
    assert bool((d_logits[torch.isneginf(seen)] == 0).all())
    G.int8_linear(d_logits, (wt, None), dx, col_scale=ws)
    assert torch.equal(dx.cpu(), I8.product(*I8.quantize(d_logits.cpu(), ref_w[1]), ref_w[0].t(), None))

    # The gradient of the layer's outputs is the slope of the log-probabilities: along a direction that keeps every sign, by
    # differences in 64 bits, whose error is of the third order in the step.
    v = torch.randn((rows, vocab), generator=g).double() * logits.cpu().double().abs()
    allowed = torch.isfinite(seen.cpu())
    factor = torch.where(allowed, I8.adjust_grad(logits.cpu(), torch.ones((rows, vocab)), **kw).double(), 0.0)

    def total(step):
        z = torch.where(allowed, (seen.cpu().double() + step * factor * v), -math.inf) / temperature
        return float((gl.double() * (z.gather(1, targets.cpu()[:, None])[:, 0] - torch.logsumexp(z, 1))).sum())

    step = 1e-4
    slope = (total(step) - total(-step)) / (2 * step)
    third = step**2 * float((gl.double().abs() * ((factor * v).abs().amax(1) / temperature) ** 3).sum())
    exact = float((ref_d * factor * v).sum())
    assert abs(slope - exact) <= third + 1e-9 * big * float(gl.abs().sum()) / step
    size = (ref_d.abs().amax(1, keepdim=True) * (factor * v).abs()).sum()
    assert abs(float((d_logits.cpu().double() * v).sum()) - exact) <= 900 * E * big * float(size)
