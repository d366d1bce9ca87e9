"""Plain restatements, in 64 bits on the CPU, of the MXFP4 and logits operators' definitions in
include/gonngpu.h. Written for small sizes."""
import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x):
    """(codes, scale bytes) of a matrix, each row filled up to whole groups of 128 columns."""
    rows, cols = x.shape
    groups = -(-cols // 128)
    full = torch.zeros((rows, groups * 128), dtype=torch.float64)
    full[:, :cols] = x.double()
    b = full.view(rows, groups * 4, 32)
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    e = torch.frexp(torch.where(finite, top, 1.0)).exponent - 1 - 2
    byte = torch.where(top > 0, e.clamp(-127, 125) + 127, 127)
    y = b.abs() * torch.pow(torch.tensor(2.0, dtype=torch.float64), 127.0 - byte.double())[..., None]
    # nearest of the 8 magnitudes, the even code among equally near ones
    dist = (y[..., None] - MAGNITUDES).abs()
    near = dist == dist.amin(-1, keepdim=True)
    order = torch.tensor([8, 1, 7, 2, 6, 3, 5, 4])  # even codes 0, 2, 4, 6 before odd ones
    code = (near * order).argmax(-1)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(finite[..., None], code, 0)
    byte = torch.where(finite, byte, 255)
    code = code.view(rows, -1)
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), byte.to(torch.uint8)


def values(data, scales, cols):
    """The values that a stored matrix stands for."""
    code = torch.stack((data & 15, data >> 4), -1).view(data.shape[0], -1).long()
    v = MAGNITUDES[code & 7] * torch.where(code >= 8, -1.0, 1.0).double()
    unit = torch.where(scales == 255, math.nan, torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127))
    return (v * unit.repeat_interleave(32, 1))[:, :cols]


def act(y, code, alpha=0.0):
    if code == 0:
        return y.clamp_min(0)
    if code == 7:
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))
    if code == 4:
        return torch.where(y > 0, y, alpha * y)
    return y


def logprobs(x, targets, k, temperature):
    """(logprob, lse, entropy, top ids, top log-probabilities)."""
    z = x.double() / temperature
    lse = torch.logsumexp(z, 1)
    empty = torch.isneginf(lse)
    bad = torch.isnan(z).any(1) | torch.isposinf(z).any(1)
    lse = torch.where(bad, math.nan, lse)
    lp = torch.where(empty[:, None], -math.inf, z - lse[:, None])
    p = torch.exp(lp)
    h = -torch.where(p == 0, 0.0, p * lp).sum(1)
    lp = torch.where(bad[:, None], math.nan, lp)
    out = torch.zeros(len(x), dtype=torch.float64)
    ids = torch.zeros((len(x), k), dtype=torch.int64)
    for r in range(len(x)):
        t = int(targets[r])
        out[r] = 0.0 if t < 0 else math.nan if t >= x.shape[1] else lp[r, t]
        key = [(math.inf, 1) if math.isnan(v) else (v, 0) for v in x[r].double().tolist()]
        ids[r] = torch.tensor(sorted(range(x.shape[1]), key=lambda c: (-key[c][0], -key[c][1], c))[:k], dtype=torch.int64)
    return out, lse, h, ids, lp.gather(1, ids)


def logprobs_grad(x, targets, gl, gh, temperature):
    z = x.double() / temperature
    lse = torch.logsumexp(z, 1, keepdim=True)
    lp = z - lse
    p = torch.exp(lp)
    h = -torch.where(p == 0, 0.0, p * lp).sum(1, keepdim=True)
    gl = torch.where(targets >= 0, gl.double(), 0.0)[:, None]
    dz = -gl * p - gh.double()[:, None] * torch.where(p == 0, 0.0, p * (lp + h))
    for r in range(len(x)):
        if targets[r] >= 0:
            dz[r, targets[r]] += gl[r, 0]
    return torch.where(torch.isneginf(lse), 0.0, dz / temperature)


def distill(x, ids, teacher, temperature):
    """(loss, lse, gradient for a gradient of 1 of each loss)."""
    z = x.double() / temperature
    lse = torch.logsumexp(z, 1)
    loss, grad = torch.zeros(len(x), dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for r in range(len(x)):
        at = [i for i in range(ids.shape[1]) if ids[r, i] >= 0 and teacher[r, i] != -math.inf]
        if not at:
            continue
        logp = torch.log_softmax(teacher[r, at].double() / temperature, 0)  # finite where p itself underflows
        p = logp.exp()
        where = ids[r, at]
        loss[r] = temperature**2 * (p * (logp - (z[r, where] - lse[r]))).sum()
        grad[r] = temperature * torch.exp(z[r] - lse[r])
        grad[r].index_add_(0, where, -temperature * p)
    return loss, lse, grad
