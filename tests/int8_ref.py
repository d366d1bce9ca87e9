"""Plain restatements on the CPU of the int8 and logits-adjusting operators' definitions in include/gonngpu.h: in 64 bits,
or step by step in fp32 where the definition rounds there. Written for small sizes."""
import collections
import math

import torch


def quantize(x, col_scale=None):
    """(int8 values, fp32 scales) of a matrix's rows."""
    y = x.float() if col_scale is None else x.float() * col_scale
    rows, cols = y.shape
    finite = torch.isfinite(y).all(1)
    top = y.abs().amax(1) if cols else torch.zeros(rows)
    s = torch.clamp_min(top.double() / 127.0, 2.0**-126).float()
    t = y.double() / s.double()[:, None]
    q = torch.round(torch.where(finite[:, None], t, 0.0))  # half to even; 64 bits keep every quotient off the middles
    return q.to(torch.int8), torch.where(finite, s, math.nan)


def values(q, s):
    return q.float() * s[:, None]


def sums(a, b):
    """sum_k a b, exactly."""
    return a.double() @ b.double().t()


def product(a, sa, b, sb):
    """The scaled sums as defined: each step rounded to fp32. No infinities among the scales."""
    v = sums(a, b).float()
    if sb is not None:
        v = v * sb
    if sa is not None:
        v = v * sa[:, None]
    return v


def _at(ids, cols):
    return [int(t) for t in ids if 0 <= int(t) < cols]


def adjust(x, history=None, prompt=None, repetition=None, frequency=None, presence=None, bias_ids=None, bias=None, mask=None):
    """In fp32, a column at a time."""
    rows, cols = x.shape
    f = torch.float32
    out = x.clone()
    for r in range(rows):
        tokens = [] if history is None else history[r].tolist()
        first = 0 if prompt is None else max(0, int(prompt[r]))
        seen, answer = set(_at(tokens, cols)), collections.Counter(_at(tokens[first:], cols))
        touched = {}
        for c in seen:
            y = x[r, c].to(f)
            if repetition is not None:
                y = y / repetition[r] if y > 0 else y * repetition[r]
            n = torch.tensor(float(answer[c]), dtype=f)
            if n > 0:
                if frequency is not None:
                    y = y - frequency[r] * n
                if presence is not None:
                    y = y - presence[r]
            touched[c] = y
        if bias is not None:
            sums = {}
            for c, b in zip(bias_ids[r].tolist(), bias[r]):
                if 0 <= c < cols:
                    sums[c] = sums[c] + b if c in sums else b
            for c, b in sums.items():
                touched[c] = touched.get(c, x[r, c].to(f)) + b
        for c, y in touched.items():
            out[r, c] = y.to(x.dtype)
        if mask is not None:
            out[r, ~allowed(mask[r], cols)] = -math.inf
    return out


def allowed(words, cols):
    """The bits of a row of int32 words, as truth values."""
    at = torch.arange(cols)
    return (words.long()[at // 32] >> (at % 32)) & 1 == 1


def adjust_grad(x, g, history=None, repetition=None, mask=None):
    rows, cols = x.shape
    out = g.clone()
    for r in range(rows):
        if repetition is not None and history is not None:
            for c in set(_at(history[r].tolist(), cols)):
                d = g[r, c].float()
                out[r, c] = (d / repetition[r] if x[r, c] > 0 else d * repetition[r]).to(x.dtype)
        if mask is not None:
            out[r, ~allowed(mask[r], cols)] = 0.0
    return out
