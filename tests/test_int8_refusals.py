"""Refusals of the int8 and logits-adjusting entry points, before any device work: the arguments are checked first, so no GPU is
needed, and none of the addresses here is read."""
import pytest
import torch

import gonngpu as G

P = 1 << 20  # an aligned address that is never read
F32, F16, FP4 = G.GN_F32, G.GN_F16, G.GN_MXFP4
BIG = 1 << 61

QUANTIZE = dict(dtype=F32, x=P, rows=4, cols=100, ldx=100, cs=None, q=P, ldq=100, scales=P, stream=None)
DEQUANTIZE = dict(q=P, scales=P, rows=4, cols=100, ldq=100, dtype=F32, out=P, ldo=100, stream=None)
GEMM = dict(M=4, N=5, K=100, alpha=1.0, A=P, lda=112, sa=P, B=P, ldb=112, sb=P, beta=0.0, C=P, ldc=5, bias=None, act=G.ACT_NONE,
            act_alpha=0.0, stream=None)
LINEAR = dict(dtype=F32, M=4, N=5, K=100, alpha=1.0, x=P, ldx=100, cs=None, B=P, ldb=112, sb=P, beta=0.0, C=P, ldc=5, bias=None,
              act=G.ACT_NONE, act_alpha=0.0, ws=P, wsn=1 << 30, stream=None)
ADJUST = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, hist=P, h=7, prompt=P, rep=P, freq=P, pres=P, bids=P, bias=P, nb=3, mask=P,
              ldmask=4, out=P + 4096, ldo=100, stream=None)
ADJUST_GRAD = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, g=P, ldg=100, hist=P, h=7, rep=P, mask=P, ldmask=4, out=P + 4096, ldo=100,
                   stream=None)
PRODUCT = [("K of", dict(K=1 << 17)), ("negative", dict(M=-1)), ("negative", dict(N=-1)), ("negative", dict(K=-1)), ("activation", dict(act=3)),
           ("NULL C", dict(C=None)), ("leading", dict(ldc=4)), ("NULL B", dict(B=None)), ("leading", dict(ldb=96)),
           ("multiples", dict(B=P + 8)), ("multiples", dict(ldb=104)), ("too large", dict(ldb=(1 << 22) + 16)), ("aligned", dict(C=P + 2)),
           ("aligned", dict(bias=P + 1)), ("aligned", dict(sb=P + 2)), ("too large", dict(M=1, N=(1 << 25) + 1, ldc=1 << 26)),
           ("too large", dict(M=(1 << 25) + 1, N=1, ldc=1)), ("too large", dict(M=1 << 20, N=1 << 20, ldc=1 << 20))]
CASES = [
    ("gn_int8_quantize", QUANTIZE, [
        ("dtype", dict(dtype=FP4)), ("size", dict(rows=-1)), ("size", dict(cols=-1)), ("leading", dict(ldx=99)), ("leading", dict(ldq=99)),
        ("NULL", dict(x=None)), ("NULL", dict(q=None)), ("NULL", dict(scales=None)), ("aligned", dict(x=P + 2)), ("aligned", dict(scales=P + 2)),
        ("aligned", dict(cs=P + 1)), ("aligned", dict(dtype=F16, x=P + 1)), ("size", dict(rows=BIG)), ("too large", dict(rows=1 << 22)),
        ("too large", dict(cols=65535 * 2048 + 1, ldx=1 << 30, ldq=1 << 30))]),
    ("gn_int8_dequantize", DEQUANTIZE, [
        ("dtype", dict(dtype=7)), ("size", dict(rows=-1)), ("leading", dict(ldo=99)), ("leading", dict(ldq=99)), ("NULL", dict(out=None)),
        ("NULL", dict(q=None)), ("NULL", dict(scales=None)), ("aligned", dict(out=P + 2)), ("too large", dict(rows=1 << 22))]),
    ("gn_int8_gemm", GEMM, PRODUCT + [
        ("NULL A", dict(A=None)), ("leading", dict(lda=96)), ("multiples", dict(A=P + 4)), ("multiples", dict(lda=101)),
        ("too large", dict(lda=(1 << 22) + 16)), ("aligned", dict(sa=P + 3))]),
    ("gn_int8_linear", LINEAR, PRODUCT + [
        ("dtype", dict(dtype=FP4)), ("leading", dict(ldx=99)), ("NULL", dict(x=None)), ("aligned", dict(x=P + 2)), ("aligned", dict(cs=P + 2)),
        ("too large", dict(M=1 << 22))]),
    ("gn_adjust_logits", ADJUST, [
        ("dtype", dict(dtype=FP4)), ("size", dict(rows=-1)), ("size", dict(cols=0)), ("size", dict(cols=1 << 31, ld=1 << 31, ldo=1 << 31, ldmask=1 << 27)),
        ("too large", dict(rows=BIG)), ("too large", dict(rows=1 << 24)), ("too large", dict(rows=1 << 22, h=2048)),
        ("leading", dict(ld=99)), ("leading", dict(ldo=99)), ("NULL", dict(x=None)), ("NULL", dict(out=None)),
        ("aligned", dict(x=P + 2)), ("aligned", dict(out=P + 2)), ("aligned", dict(dtype=F16, x=P + 1)), ("in place", dict(out=P, ldo=101)),
        ("history", dict(h=-1)), ("history", dict(h=1 << 29)), ("NULL history", dict(hist=None)), ("history", dict(hist=P + 4)),
        ("aligned", dict(prompt=P + 4)), ("aligned", dict(rep=P + 2)), ("aligned", dict(freq=P + 1)),
        ("aligned", dict(pres=P + 2)), ("biases", dict(nb=-1)), ("biases", dict(nb=1025)), ("NULL biases", dict(bids=None)),
        ("NULL biases", dict(bias=None)), ("aligned", dict(bids=P + 4)), ("aligned", dict(bias=P + 2)), ("words", dict(ldmask=3)),
        ("mask", dict(mask=P + 2))]),
    ("gn_adjust_logits_backward", ADJUST_GRAD, [
        ("dtype", dict(dtype=9)), ("size", dict(cols=0)), ("leading", dict(ld=99)), ("leading", dict(ldg=99)), ("leading", dict(ldo=99)),
        ("NULL logits", dict(x=None)), ("NULL grad_out", dict(g=None)), ("NULL grad_logits", dict(out=None)), ("in place", dict(out=P, x=P + 8192, ldo=101)),
        ("logits' place", dict(out=P + 8192, x=P + 8192, ldo=101)), ("history", dict(h=-1)), ("NULL history", dict(hist=None)),
        ("aligned", dict(rep=P + 2)), ("words", dict(ldmask=3)), ("aligned", dict(out=P + 2))]),
]


@pytest.mark.parametrize("name,good,word,change", [(n, g, w, c) for n, g, cs in CASES for w, c in cs],
                         ids=lambda v: v if isinstance(v, str) else ",".join(f"{k}={x}" for k, x in v.items()) if len(v) < 5 else "")
def test_refused(name, good, word, change):
    rc, msg = G.call_rc(name, *{**good, **change}.values())
    assert rc == -1 and word in msg, (rc, msg)


def test_workspace_needed_is_checked():
    for M in (1, 4, 40, 400):
        need = G.load().gn_int8_linear_workspace(M, 5, 100)
        if need:
            for change in (dict(wsn=need - 1), dict(ws=None), dict(ws=P + 8)):
                rc, msg = G.call_rc("gn_int8_linear", *{**LINEAR, "M": M, **change}.values())
                assert rc == -1 and "workspace" in msg
    assert G.load().gn_int8_linear_workspace(400, 5, 100) >= 400 * 104
    for bad in ((-1, 5, 5), (5, -1, 5), (5, 5, -1), (0, 5, 5), (5, 5, 0), (5, 5, 1 << 17), ((1 << 63) - 1, 5, 100000)):
        assert G.load().gn_int8_linear_workspace(*bad) == 0


# ------------------------------------------------------------------ the Python binding's own checks
def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def _q(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def _m(rows, cols):
    return G.int8_empty(rows, cols, device="cpu")


I64, I32, H = torch.int64, torch.int32, torch.float16
BINDING = [
    ("float32 or float16", lambda: G.int8_quantize(_t(4, 8, dtype=torch.float64), *_m(4, 8))),
    ("dense rows", lambda: G.int8_quantize(_t(8, 4).t(), *_m(4, 8))),
    ("dense rows", lambda: G.int8_quantize(_t(4, 8), _q(8, 4).t(), _t(4))),
    ("dense rows", lambda: G.int8_quantize(_t(4, 8), _q(1, 8).expand(4, 8), _t(4))),
    ("int8 is needed", lambda: G.int8_quantize(_t(4, 8), _t(4, 8, dtype=torch.uint8), _t(4))),
    ("values", lambda: G.int8_quantize(_t(4, 8), *_m(4, 9))),
    ("scales", lambda: G.int8_quantize(_t(4, 8), _q(4, 8), _t(5))),
    ("scales", lambda: G.int8_quantize(_t(4, 8), _q(4, 8), _t(4, dtype=H))),
    ("col_scale", lambda: G.int8_quantize(_t(4, 8), *_m(4, 8), col_scale=_t(4))),
    ("current GPU", lambda: G.int8_quantize(_t(4, 8), *_m(4, 8))),
    ("integers", lambda: G.int8_dequantize(*_m(4, 8), _t(3, 8))),
    ("scales", lambda: G.int8_dequantize(_q(4, 8), _t(3), _t(4, 8))),
    ("C is float32", lambda: G.int8_gemm(_m(2, 8), _m(3, 8), _t(2, 3, dtype=H))),
    ("int8 is needed", lambda: G.int8_gemm((_t(2, 8), None), _m(3, 8), _t(2, 3))),
    ("is not", lambda: G.int8_gemm(_m(2, 8), _m(3, 9), _t(2, 3))),
    ("is not", lambda: G.int8_gemm(_m(2, 8), _m(4, 8), _t(2, 3))),
    ("is not", lambda: G.int8_gemm(_m(3, 8), _m(3, 8), _t(2, 3))),
    ("scales of A", lambda: G.int8_gemm((_q(2, 8), _t(3)), _m(3, 8), _t(2, 3))),
    ("scales of B", lambda: G.int8_gemm(_m(2, 8), (_q(3, 8), _t(2)), _t(2, 3))),
    ("bias", lambda: G.int8_gemm(_m(2, 8), _m(3, 8), _t(2, 3), bias=_t(2))),
    ("current GPU", lambda: G.int8_gemm(_m(2, 8), _m(3, 8), _t(2, 3))),
    ("float32 or float16", lambda: G.int8_linear(_q(2, 8), _m(3, 8), _t(2, 3))),
    ("is not", lambda: G.int8_linear(_t(2, 8), _m(3, 9), _t(2, 3))),
    ("col_scale", lambda: G.int8_linear(_t(2, 8), _m(3, 8), _t(2, 3), col_scale=_t(3))),
    ("bias", lambda: G.int8_linear(_t(2, 8), _m(3, 8), _t(2, 3), bias=_t(2))),
    ("current GPU", lambda: G.int8_linear(_t(2, 8), _m(3, 8), _t(2, 3))),
    ("type and shape", lambda: G.adjust_logits(_t(2, 8), _t(2, 8, dtype=H))),
    ("type and shape", lambda: G.adjust_logits(_t(2, 8), _t(2, 9))),
    ("together", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), bias=_t(2, 3))),
    ("need a history", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), repetition=_t(2))),
    ("need a history", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), prompt=_t(2, dtype=I64))),
    ("history", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), history=_t(2, 5))),
    ("history", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), history=_t(3, 5, dtype=I64))),
    ("history", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), history=_t(2, dtype=I64))),
    ("prompt", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), history=_t(2, 5, dtype=I64), prompt=_t(2, dtype=I32))),
    ("frequency", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), history=_t(2, 5, dtype=I64), frequency=_t(3))),
    ("bias_ids", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), bias_ids=_t(2, 4, dtype=I64), bias=_t(2, 3))),
    ("bias", lambda: G.adjust_logits(_t(2, 8), _t(2, 8), bias_ids=_t(2, 3, dtype=I64), bias=_t(2, 3, dtype=H))),
    ("mask", lambda: G.adjust_logits(_t(2, 40), _t(2, 40), mask=_t(2, 1, dtype=I32))),
    ("mask", lambda: G.adjust_logits(_t(2, 40), _t(2, 40), mask=_t(1, 2, dtype=I32))),
    ("mask", lambda: G.adjust_logits(_t(2, 40), _t(2, 40), mask=_t(1, 2, dtype=I32).expand(2, 2))),
    ("mask", lambda: G.adjust_logits(_t(2, 40), _t(2, 40), mask=_t(2, 2, dtype=I64))),
    ("current GPU", lambda: G.adjust_logits(_t(2, 8), _t(2, 8))),
    ("grad_out has", lambda: G.adjust_logits_backward(_t(2, 8), _t(2, 9), _t(2, 8))),
    ("grad_logits has", lambda: G.adjust_logits_backward(_t(2, 8), _t(2, 8), _t(2, 8, dtype=H))),
    ("needs a history", lambda: G.adjust_logits_backward(_t(2, 8), _t(2, 8), _t(2, 8), repetition=_t(2))),
    ("current GPU", lambda: G.adjust_logits_backward(_t(2, 8), _t(2, 8), _t(2, 8))),
]


@pytest.mark.parametrize("i", range(len(BINDING)))
def test_binding_refuses(i):
    word, call = BINDING[i]
    with pytest.raises(G.GonngpuError, match=word):
        call()


def test_int8_empty_rows_start_at_multiples_of_16_bytes():
    for cols in (1, 15, 16, 17, 100):
        q, s = G.int8_empty(3, cols, device="cpu")
        assert q.shape == (3, cols) and q.stride(0) % 16 == 0 and q.stride(0) - cols < 16 and s.shape == (3,)
