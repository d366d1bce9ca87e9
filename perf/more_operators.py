"""What is measured: one pass of the operators around 8-bit integer layers and a sampler's logits.

Five kinds of pass, through the Python binding's public entry points where `own` is true and in
plain torch operations where it is not:

* quantize  a matrix brought to 8-bit integers with a scale for each row, and back to the values it
            then stands for;
* product   a product of two int8 matrices with scales for each token and output channel, bias and
            activation;
* linear    a linear layer with int8 weights (outputs x inputs): fp16 or fp32 activations are brought
            to 8 bits by token in the same pass;
* back      the gradient of such a layer's inputs: the outputs' gradient, times the weights' scales, brought
            to 8 bits by token, against the transposed weights;
* adjust    a batch's logits before sampling: repetition, frequency and presence penalties from
            the tokens so far, biases of listed tokens, a grammar's mask of allowed tokens; with "train" the
            gradient of the logits too.

Calls run on a torch stream of their own, as bench.py and a serving loop have it.
"""
import math
import os
import sys

import torch

own = False


def listed():
    return [
        # A few rows of fp32 activations of an odd width, to 8 bits and back: the smallest call.
        {"name": "quantize_f32_16", "kind": "quantize", "dtype": "f32", "rows": 16, "cols": 1000},
        # The benchmark's linear layer's weights on loading, fp16.
        {"name": "quantize_f16_weights", "kind": "quantize", "dtype": "f16", "rows": 11008, "cols": 4096},
        # Decode: one token through the benchmark's layer (4096 -> 11008); it reads its weights and little else.
        {"name": "linear_f16_1", "kind": "linear", "dtype": "f16", "act": "none", "rows": 1, "inputs": 4096, "outputs": 11008},
        # A batch of decoding sequences, and odd sizes throughout.
        {"name": "linear_f32_odd", "kind": "linear", "dtype": "f32", "act": "relu", "rows": 27, "inputs": 2027, "outputs": 4099},
        # Prefill of the benchmark's layer.
        {"name": "linear_f16_512", "kind": "linear", "dtype": "f16", "act": "gelu", "rows": 512, "inputs": 4096, "outputs": 11008},
        # Activations that several layers share, quantised once: one of these layers, a decoding batch.
        {"name": "product_64", "kind": "product", "act": "none", "rows": 64, "inputs": 4096, "outputs": 4096},
        # The benchmark's headline product (8192^3) in 8 bits: the largest call.
        {"name": "product_8192", "kind": "product", "act": "none", "rows": 8192, "inputs": 8192, "outputs": 8192},
        # Training in front of a frozen 8-bit layer: the gradient of its inputs, a small odd one and the benchmark's layer.
        {"name": "back_f16_odd", "kind": "back", "dtype": "f16", "rows": 130, "inputs": 1000, "outputs": 515},
        {"name": "back_f32_512", "kind": "back", "dtype": "f32", "rows": 512, "inputs": 4096, "outputs": 11008},
        # One decoding step of one sequence: penalties from the 300 tokens so far.
        {"name": "adjust_f32_1", "kind": "adjust", "dtype": "f32", "rows": 1, "cols": 131072, "history": 300, "biases": 0, "masked": 0.0, "train": False},
        # A batch of constrained decoding: fp16 logits, an odd vocabulary, long histories, biases, most tokens masked out.
        {"name": "adjust_f16_64", "kind": "adjust", "dtype": "f16", "rows": 64, "cols": 50257, "history": 2048, "biases": 64, "masked": 0.9, "train": False},
        # A training step on answers that were sampled so: the adjusted logits and, from theirs, the logits' gradient.
        {"name": "adjust_f32_train", "kind": "adjust", "dtype": "f32", "rows": 4096, "cols": 32768, "history": 512, "biases": 0, "masked": 0.1, "train": True},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of the larger ones multiples of 32."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v = v // 32 * 32
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["quantize", "product", "linear", "linear", "back", "adjust", "adjust", "adjust"])
    if kind == "quantize":
        return {"kind": kind, "dtype": rng.choice(["f32", "f16"]), "rows": _size(rng, 1, 11008), "cols": _size(rng, 32, 8192)}
    if kind != "adjust":
        c = {"kind": kind, "act": rng.choice(["none", "relu", "gelu"]), "rows": _size(rng, 1, 8192),
             "inputs": _size(rng, 32, 8192), "outputs": _size(rng, 32, 8192)}
        if kind != "product":
            c["dtype"] = rng.choice(["f32", "f16"])
        return c
    while True:
        c = {"kind": kind, "dtype": rng.choice(["f32", "f16"]), "rows": _size(rng, 1, 4096), "cols": _size(rng, 64, 131072)}
        c["history"], c["biases"] = _size(rng, 1, 4096), rng.choice([0, _size(rng, 1, 300)])
        if c["rows"] * max(c["cols"], 16 * c["history"]) > 4096 * 32768:
            continue
        c["masked"] = rng.choice([0.0, 0.1, 0.9])
        c["train"] = rng.random() < 0.4
        return c


# ------------------------------------------------------------------ inputs
_stream = None


def _use_stream():
    """Makes a stream of its own torch's current one (the default stream would be waited for around every call)."""
    global _stream
    if torch.cuda.current_stream().cuda_stream == 0:
        if _stream is None:
            _stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        torch.cuda.set_stream(_stream)


def _empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _bytes(rows, cols):
    """An int8 matrix whose rows start at multiples of 16 bytes."""
    return _empty(rows, -(-cols // 16) * 16, dtype=torch.int8)[:, :cols]


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _acts(g, rows, cols, dtype):
    """Activations: normal, with one channel in 64 (and the first of all) ten times as large."""
    x = _normal(g, rows, cols)
    loud = torch.rand((cols,), generator=g, device="cuda") < 1 / 64
    loud[0] = True
    x[:, loud] *= 10.0
    return x.half() if dtype == "f16" else x


def _stored(x):
    """A matrix as it is stored: int8 values and a scale for each row."""
    s = x.abs().amax(1) / 127.0
    q = _bytes(*x.shape)
    q.copy_(torch.round(x / s[:, None]).clamp_(-127, 127))
    return q, s


def _inputs(c, seed):
    kind, rows = c["kind"], c["rows"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "quantize":
        return {"x": _acts(g, rows, c["cols"], c["dtype"])}
    if kind == "back":  # gradients under a loss scale; the transposed weights carry no scale of their own, the outputs' go with dy
        q, s = _stored(_normal(g, c["inputs"], c["outputs"]).mul_(0.02))
        dy = _normal(g, rows, c["outputs"]).mul_(0.5)
        return {"x": dy.half() if c["dtype"] == "f16" else dy, "w": q, "ws": _normal(g, c["outputs"]).mul_(0.1).exp_().mul_(0.0006)}
    if kind != "adjust":
        s = {"b": _normal(g, c["outputs"]).mul_(0.01)}
        s["w"], s["ws"] = _stored(_normal(g, c["outputs"], c["inputs"]).mul_(0.02))
        if kind == "linear":
            s["x"] = _acts(g, rows, c["inputs"], c["dtype"])
        else:
            s["x"], s["xs"] = _stored(_acts(g, rows, c["inputs"], "f32"))
        return s
    cols, h, nb = c["cols"], c["history"], c["biases"]
    x = _normal(g, rows, cols).mul_(2.5)
    # The tokens so far: some of them often, as in a text; a row's last ones may be absent (shorter sequences in the batch).
    u = torch.rand((rows, h), generator=g, device="cuda")
    ids = (torch.exp(u * math.log(cols)).long() * 7919) % cols
    length = torch.randint((h + 1) // 2, h + 1, (rows, 1), generator=g, device="cuda")
    ids.masked_fill_(torch.arange(h, device="cuda") >= length, -1)
    s = {"x": x.half() if c["dtype"] == "f16" else x, "ids": ids, "prompt": (length[:, 0] // 3).contiguous()}
    s["rho"] = 1.0 + 0.3 * torch.rand((rows,), generator=g, device="cuda")
    s["freq"], s["pres"] = (0.5 * torch.rand((rows,), generator=g, device="cuda") for _ in range(2))
    if nb:
        s["bids"] = torch.randint(0, cols, (rows, nb), generator=g, device="cuda")
        s["bias"] = _normal(g, rows, nb).mul_(3.0)
    if c["masked"]:  # bit j % 32 of word j / 32: token j is allowed; one row in 64 has no token that is
        words = -(-cols // 32)
        w = torch.zeros((rows, words), dtype=torch.int64, device="cuda")
        for b in range(32):
            w |= (torch.rand((rows, words), generator=g, device="cuda") >= c["masked"]).long() << b
        w.masked_fill_((torch.arange(rows, device="cuda") % 64 == 63)[:, None], 0)
        s["mask"] = torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)
    if c["train"]:
        s["g"] = _normal(g, rows, cols).mul_(0.01).to(s["x"].dtype)
    return s


def prepare(case, seed):
    _use_stream()
    c, s = case, _inputs(case, seed)
    s["c"] = dict(c)
    kind, rows = c["kind"], c["rows"]
    if kind == "quantize":
        s["q"], s["qs"], s["y"] = _bytes(rows, c["cols"]), _empty(rows), torch.empty_like(s["x"])
    elif kind == "adjust":
        s["y"] = torch.empty_like(s["x"])
        s["dx"] = torch.empty_like(s["x"]) if c["train"] else None
    else:
        s["y"] = _empty(rows, c["inputs"] if kind == "back" else c["outputs"])
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    root = os.path.join(os.getcwd(), "go-nngpu_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gonngpu as G

    c = s["c"]
    kind = c["kind"]
    if kind == "quantize":
        G.int8_quantize(s["x"], s["q"], s["qs"])
        G.int8_dequantize(s["q"], s["qs"], s["y"])
        return s["y"]
    if kind == "adjust":
        G.adjust_logits(s["x"], s["y"], history=s["ids"], prompt=s["prompt"], repetition=s["rho"], frequency=s["freq"],
                        presence=s["pres"], bias_ids=s.get("bids"), bias=s.get("bias"), mask=s.get("mask"))
        if not c["train"]:
            return s["y"]
        G.adjust_logits_backward(s["x"], s["g"], s["dx"], history=s["ids"], repetition=s["rho"], mask=s.get("mask"))
        return {"logits": s["y"], "dx": s["dx"]}
    if kind == "back":
        G.int8_linear(s["x"], (s["w"], None), s["y"], col_scale=s["ws"])
        return s["y"]
    act = {"none": G.ACT_NONE, "relu": G.ACT_RELU, "gelu": G.ACT_GELU}[c["act"]]
    if kind == "linear":
        G.int8_linear(s["x"], (s["w"], s["ws"]), s["y"], bias=s["b"], act=act)
    else:
        G.int8_gemm((s["x"], s["xs"]), (s["w"], s["ws"]), s["y"], bias=s["b"], act=act)
    return s["y"]


def _plain_quantized(x):
    """int8 values, as fp32, and scales of x's rows. The quotients need 64 bits: a scale off by its last place, or a
    quotient rounded onto the middle of two integers, would change values by whole steps."""
    s = (x.abs().amax(1, keepdim=True).double() / 127.0).float().clamp_min(2.0**-126)
    return torch.round(x.double() / s.double()).float(), s


def _plain_act(x, act):
    if act == "relu":
        return x.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x


def _plain_counts(ids, first, cols):
    """How often each column is among ids[r, first[r]:], negative ones left out."""
    there = (ids >= 0) & (torch.arange(ids.shape[1], device=ids.device) >= first[:, None])
    n = torch.zeros((ids.shape[0], cols), device=ids.device)
    return n.scatter_add_(1, ids.clamp_min(0), there.float())


def _plain_allowed(mask, cols):
    bits = (mask[:, :, None] >> torch.arange(32, device=mask.device, dtype=torch.int32)) & 1
    return bits.reshape(mask.shape[0], -1)[:, :cols] != 0


def _run_plain(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "quantize":
        q, scale = _plain_quantized(s["x"].float())
        return (q * scale).to(s["x"].dtype)
    if kind == "adjust":
        x, cols, rho = s["x"].float(), c["cols"], s["rho"][:, None]
        seen = _plain_counts(s["ids"], torch.zeros_like(s["prompt"]), cols) > 0
        n = _plain_counts(s["ids"], s["prompt"], cols)
        y = torch.where(seen, torch.where(x > 0, x / rho, x * rho), x)
        y = y - s["freq"][:, None] * n - torch.where(n > 0, s["pres"][:, None], 0.0)
        if c["biases"]:
            y = y.scatter_add(1, s["bids"], s["bias"])
        if c["masked"]:
            allowed = _plain_allowed(s["mask"], cols)
            y = torch.where(allowed, y, -math.inf)
        y = y.to(s["x"].dtype)
        if not c["train"]:
            return y
        dx = s["g"].float()
        dx = torch.where(seen, torch.where(x > 0, dx / rho, dx * rho), dx)
        if c["masked"]:
            dx = torch.where(allowed, dx, 0.0)
        return {"logits": y, "dx": dx.to(s["x"].dtype)}
    if kind == "product":
        a, scale = s["x"].float(), s["xs"][:, None]
    else:
        a, scale = _plain_quantized(s["x"].float() * (s["ws"] if kind == "back" else 1.0))
    y = (a @ s["w"].float().t()) * scale
    return y if kind == "back" else _plain_act(y * s["ws"] + s["b"], c["act"])


def work(case):
    c = case
    kind, r = c["kind"], c["rows"]
    e = 2.0 if c.get("dtype") == "f16" else 4.0
    if kind == "quantize":
        return {"bytes": r * c["cols"] * (2 * e + 2.0) + 8.0 * r, "flops": 4.0 * r * c["cols"]}
    if kind == "adjust":
        back = 2 if c["train"] else 1
        per = r * (8.0 * c["history"] + 12.0 * c["biases"] + (c["cols"] / 8 if c["masked"] else 0) + 20.0)
        return {"bytes": r * 2 * e * c["cols"] * back + per * back, "flops": r * c["cols"] * 2.0 * back}
    k, n = (c["outputs"], c["inputs"]) if kind == "back" else (c["inputs"], c["outputs"])
    return {"bytes": r * k * (1.0 if kind == "product" else e) + float(n) * k + 4.0 * r * n + 8.0 * n, "flops": 2.0 * r * k * n}


# ------------------------------------------------------------------ the same in 64 bits
def _quantized64(x):
    """Whole numbers and scales (which are fp32 numbers by definition), both in fp64."""
    s = torch.maximum(x.max(1).values, -x.min(1).values).div(127.0).float().double().clamp_min(2.0**-126)[:, None]
    t = x / s
    low = torch.floor(t)
    up = (t - low > 0.5) | ((t - low == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return low + up.double(), s


def exact(case, seed):
    _use_stream()
    c, s = case, _inputs(case, seed)
    kind = c["kind"]
    if kind == "quantize":
        q, scale = _quantized64(s["x"].double())
        return q * scale
    if kind == "adjust":
        return _adjusted64(c, s)
    if kind == "product":
        a, scale = s["x"].double(), s["xs"].double()[:, None]
    elif kind == "linear":
        a, scale = _quantized64(s["x"].double())
    else:  # the factor is applied in fp32 by definition
        a, scale = _quantized64((s["x"].double() * s["ws"].double()).float().double())
    y = torch.empty((c["rows"], s["w"].shape[0]), dtype=torch.float64, device="cuda")
    for i in range(0, y.shape[1], 4096):
        y[:, i:i + 4096] = a @ s["w"][i:i + 4096].double().t().contiguous()
    y *= scale
    if kind == "back":
        return y
    y = y * s["ws"].double() + s["b"].double()
    if c["act"] == "relu":
        return y * (y > 0)
    if c["act"] == "gelu":
        return y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y**3))
    return y


def _adjusted64(c, s):
    cols = c["cols"]
    y = torch.empty((c["rows"], cols), dtype=torch.float64, device="cuda")
    dx = torch.empty_like(y) if c["train"] else None
    place = torch.arange(cols, device="cuda")
    for r in range(c["rows"]):
        ids = s["ids"][r]
        at = torch.arange(len(ids), device="cuda")
        kept = torch.bincount(torch.where(ids < 0, cols, ids), minlength=cols + 1)[:cols] > 0
        n = torch.bincount(torch.where((ids < 0) | (at < s["prompt"][r]), cols, ids), minlength=cols + 1)[:cols].double()
        x, rho = s["x"][r].double(), s["rho"][r].double()
        factor = torch.where(kept, torch.where(x > 0, 1.0 / rho, rho), 1.0)
        v = x * factor - n * s["freq"][r].double() - (n > 0).double() * s["pres"][r].double()
        if c["biases"]:
            v.index_put_((s["bids"][r],), s["bias"][r].double(), accumulate=True)
        if c["masked"]:
            off = (torch.div(s["mask"][r].long()[place // 32] % 2**32, 2 ** (place % 32), rounding_mode="floor") % 2) == 0
            v.masked_fill_(off, -math.inf)
            factor.masked_fill_(off, 0.0)
        y[r] = v
        if c["train"]:
            dx[r] = s["g"][r].double() * factor
    return {"logits": y, "dx": dx} if c["train"] else y
