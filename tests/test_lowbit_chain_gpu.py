"""The operators together, as they are used: a teacher's layer names its best tokens, a student whose weights
are stored in MXFP4 answers, and is trained against them. The student's gradients reach its inputs through the
dequantised weights and its master weights straight through the rounding. Each step is compared
with 64 bits on what the step before it gave, with bounds from the roundings of its own sums."""
import math

import pytest
import torch

import gonngpu as G
from tests import lowbit_ref as R

pytestmark = pytest.mark.gpu

E = 2.0**-24


def _near(got, ref, bound):
    assert bool(((got.cpu().double() - ref).abs() <= bound).all()), float(((got.cpu().double() - ref).abs() - bound).max())


@pytest.mark.parametrize("rows,inputs,vocab,k", [(1, 96, 500, 5), (24, 320, 3001, 20), (130, 256, 9000, 64)])
@pytest.mark.parametrize("fp4_acts", [False, True])
def test_distillation_step_of_a_4_bit_layer(dev, rows, inputs, vocab, k, fp4_acts):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((rows, inputs), generator=g).half()
    w = torch.randn((vocab, inputs), generator=g) * 3 / math.sqrt(inputs)
    wt = (w + 0.3 * torch.randn((vocab, inputs), generator=g) / math.sqrt(inputs)).half()
    xd, wd = x.to(dev), w.to(dev)
    new = lambda *s, dtype=torch.float32: torch.full(s, -5, dtype=dtype, device=dev)  # noqa: E731

    # The teacher's logits, and its best tokens with their log-probabilities.
    t_logits, ids, tops = new(rows, vocab), new(rows, k, dtype=torch.int64), new(rows, k)
    G.gemm(xd, wt.to(dev), t_logits, transB=True)
    G.token_logprobs(t_logits, None, None, top_ids=ids, top_logprobs=tops)
    ref = R.logprobs(t_logits.cpu(), torch.zeros(rows, dtype=torch.int64), k, 1.0)
    assert torch.equal(ids.cpu(), ref[3])
    _near(tops, ref[4], 400 * E * (1 + ref[4].abs()))

    # The student's weights in 4 bits, and its logits.
    wq, logits = G.mxfp4_empty(vocab, inputs, device=dev), new(rows, vocab)
    G.mxfp4_quantize(wd, *wq)
    wv = R.values(*R.quantize(w), inputs)
    a = x.double()
    if fp4_acts:
        xq = G.mxfp4_empty(rows, inputs, device=dev)
        G.mxfp4_quantize(xd, *xq)
        a = R.values(*R.quantize(x), inputs)
        G.mxfp4_gemm(xq, wq, logits, K=inputs)
    else:
        G.mxfp4_gemm(xd, wq, logits)
    _near(logits, a @ wv.t(), 2 * E * (inputs + 8) * (a.abs() @ wv.abs().t()))

    # Loss and gradient of the student's logits.
    temperature = 2.0
    loss, lse, dl = new(rows), new(rows), new(rows, vocab)
    G.distill(logits, ids, tops, loss, lse=lse, temperature=temperature)
    G.distill_backward(logits, ids, tops, lse, torch.ones(rows, device=dev), dl, temperature=temperature)
    r_loss, r_lse, r_dl = R.distill(logits.cpu(), ids.cpu(), tops.cpu(), temperature)
    big = float(logits.abs().max()) + float(tops.abs().max()) + 8
    _near(loss, r_loss, 4 * 800 * E * big)
    _near(dl, r_dl, 800 * E * big * r_dl.abs() + 400 * E * temperature * torch.zeros_like(r_dl).scatter_(1, ids.cpu(), 1.0) + 1e-44)

    # Through the layer: to its inputs by the weights as they stand, to the master weights straight through.
    back, dx, dw = new(vocab, inputs), new(rows, inputs), new(vocab, inputs)
    G.mxfp4_dequantize(*wq, back)
    assert torch.equal(back.cpu(), wv.float())
    G.gemm(dl, back, dx)
    G.gemm(dl, xd.float(), dw, transA=True)
    d = dl.cpu().double()
    _near(dx, d @ wv, 2 * E * (vocab + 8) * (d.abs() @ wv.abs()))
    _near(dw, d.t() @ x.double(), 2 * E * (rows + 8) * (d.abs().t() @ x.double().abs()))

    # The loss falls along the gradient: its change over a small step of the logits is the gradient's.
    step = 1e-3
    moved = logits.cpu().double() - step * r_dl
    change = R.distill(moved, ids.cpu(), tops.cpu(), temperature)[0].sum() - r_loss.sum()
    slope = -step * (r_dl**2).sum()
    assert abs(change - slope) <= step**2 * 2 * float((r_dl**2).sum()) + 1e-12  # the curvature of the loss is at most 1

    # And the answer: the log-probability of the teacher's first choice.
    lp, h = new(rows), new(rows)
    G.token_logprobs(logits, ids[:, 0].contiguous(), lp, entropy=h)
    r = R.logprobs(logits.cpu(), ids.cpu()[:, 0], 0, 1.0)
    _near(lp, r[0], 400 * E * (1 + big))
    _near(h, r[2], 600 * E * (1 + big) * (1 + r[2]))
