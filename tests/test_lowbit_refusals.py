"""Refusals of the MXFP4 and logits entry points, before any device work: the arguments are checked
first, so no GPU is needed, and none of the addresses here is read."""
import ctypes

import pytest
import torch

import gonngpu as G

P = 1 << 20  # an aligned address that is never read
F32, F16, FP4 = G.GN_F32, G.GN_F16, G.GN_MXFP4
BIG = 1 << 61


def _size(rows, cols):
    d, s = ctypes.c_size_t(), ctypes.c_size_t()
    rc, msg = G.call_rc("gn_mxfp4_size", rows, cols, ctypes.byref(d), ctypes.byref(s))
    return rc, d.value, s.value


def test_mxfp4_size():
    assert _size(0, 5) == (0, 0, 0)
    assert _size(3, 1) == (0, 192, 12)
    assert _size(2, 128) == (0, 128, 8)
    assert _size(2, 129) == (0, 256, 16)
    assert _size(140000, 32768) == (0, 140000 * 16384, 140000 * 1024)
    for bad in ((-1, 4), (4, -1), (BIG, 4096), (1, (1 << 63) - 1)):
        assert _size(*bad)[0] == -1
    assert G.call_rc("gn_mxfp4_size", 1, 1, None, None)[0] == -1


def _refused(word, name, *args):
    rc, msg = G.call_rc(name, *args)
    assert rc == -1 and word in msg, (rc, msg)


QUANTIZE = dict(dtype=F32, x=P, rows=4, cols=100, ldx=100, data=P, scales=P, stream=None)
DEQUANTIZE = dict(data=P, scales=P, rows=4, cols=100, dtype=F32, out=P, ldo=100, stream=None)
GEMM = dict(a=F16, M=4, N=5, K=100, alpha=1.0, A=P, lda=100, asc=None, B=P, bsc=P, beta=0.0, C=P, ldc=5, bias=None,
            act=G.ACT_NONE, act_alpha=0.0, stream=None)
LOGPROBS = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, temp=1.0, targets=P, logprob=P, lse=P, entropy=P, k=5, ids=P,
                tops=P, ws=P, wsn=1 << 30, stream=None)
LOGPROBS_GRAD = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, temp=1.0, targets=P, lse=P, entropy=P, gl=P, gh=P, g=P + 4096,
                     ldg=100, stream=None)
DISTILL = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, temp=1.0, ids=P, teacher=P, k=5, loss=P, lse=P, ws=P, wsn=1 << 30,
               stream=None)
DISTILL_GRAD = dict(dtype=F32, x=P, rows=4, cols=100, ld=100, temp=1.0, ids=P, teacher=P, k=5, lse=P, gl=P, g=P + 4096, ldg=100,
                    stream=None)
INF, NAN = float("inf"), float("nan")
CASES = [
    ("gn_mxfp4_quantize", QUANTIZE, [
        ("dtype", dict(dtype=FP4)), ("size", dict(rows=-1)), ("size", dict(cols=-1)), ("leading", dict(ldx=99)), ("NULL", dict(x=None)),
        ("NULL", dict(data=None)), ("NULL", dict(scales=None)), ("multiple", dict(data=P + 8)), ("multiple", dict(scales=P + 2)),
        ("aligned", dict(x=P + 2)), ("aligned", dict(dtype=F16, x=P + 1)), ("size", dict(rows=BIG)), ("too large", dict(rows=(1 << 25) + 1)),
        ("too large", dict(cols=65535 * 2048 + 1, ldx=1 << 30))]),
    ("gn_mxfp4_dequantize", DEQUANTIZE, [
        ("dtype", dict(dtype=7)), ("size", dict(rows=-1)), ("leading", dict(ldo=99)), ("NULL", dict(out=None)), ("NULL", dict(data=None)),
        ("multiple", dict(data=P + 4)), ("multiple", dict(scales=P + 1)), ("aligned", dict(out=P + 2)), ("too large", dict(rows=(1 << 25) + 1))]),
    ("gn_mxfp4_gemm", GEMM, [
        ("dtype", dict(a=F32)), ("negative", dict(M=-1)), ("negative", dict(K=-1)), ("activation", dict(act=3)), ("NULL C", dict(C=None)),
        ("leading", dict(ldc=4)), ("leading", dict(lda=99)), ("NULL", dict(A=None)), ("NULL", dict(B=None)), ("NULL", dict(bsc=None)),
        ("multiple", dict(B=P + 8)), ("multiple", dict(bsc=P + 2)), ("scales given", dict(asc=P)), ("NULL", dict(a=FP4)),
        ("multiple", dict(a=FP4, A=P + 8, asc=P)), ("aligned", dict(A=P + 1)), ("aligned", dict(C=P + 2)), ("aligned", dict(bias=P + 1)),
        ("too large", dict(M=1 << 33, N=1 << 33, ldc=1 << 33)), ("too large", dict(M=1, N=(1 << 25) + 1, ldc=1 << 26)),
        ("too large", dict(M=(1 << 25) + 1, N=1, ldc=1)), ("too large", dict(M=1 << 20, N=1 << 20, ldc=1 << 20))]),
    ("gn_token_logprobs", LOGPROBS, [
        ("dtype", dict(dtype=FP4)), ("size", dict(rows=-1)), ("size", dict(cols=0)), ("size", dict(cols=1 << 31, ld=1 << 31)),
        ("temperature", dict(temp=0.0)), ("temperature", dict(temp=-1.0)), ("temperature", dict(temp=NAN)), ("temperature", dict(temp=INF)),
        ("temperature", dict(temp=1e-44)), ("leading", dict(ld=99)), ("NULL", dict(x=None)), ("aligned", dict(x=P + 2)), ("alternatives", dict(k=65)),
        ("alternatives", dict(k=-1)), ("alternatives", dict(cols=4, ld=4)), ("together", dict(targets=None)), ("together", dict(logprob=None)),
        ("NULL", dict(ids=None)), ("NULL", dict(tops=None)), ("too large", dict(rows=BIG))]),
    ("gn_token_logprobs_backward", LOGPROBS_GRAD, [
        ("dtype", dict(dtype=9)), ("size", dict(cols=0)), ("temperature", dict(temp=0.0)), ("leading", dict(ldg=99)), ("NULL", dict(lse=None)),
        ("NULL", dict(g=None)), ("together", dict(targets=None)), ("together", dict(gl=None)), ("together", dict(entropy=None)),
        ("together", dict(gh=None)), ("aligned", dict(g=P + 2)), ("in place", dict(g=P, ldg=101))]),
    ("gn_distill_forward", DISTILL, [
        ("dtype", dict(dtype=FP4)), ("size", dict(rows=-1)), ("temperature", dict(temp=NAN)), ("entries", dict(k=0)), ("entries", dict(k=257)),
        ("NULL", dict(ids=None)), ("NULL", dict(teacher=None)), ("NULL", dict(loss=None)), ("leading", dict(ld=3))]),
    ("gn_distill_backward", DISTILL_GRAD, [
        ("dtype", dict(dtype=FP4)), ("entries", dict(k=0)), ("leading", dict(ldg=99)), ("NULL", dict(lse=None)), ("NULL", dict(gl=None)),
        ("NULL", dict(g=None)), ("NULL", dict(ids=None)), ("in place", dict(g=P, ldg=101))]),
]


@pytest.mark.parametrize("name,good,word,change", [(n, g, w, c) for n, g, cs in CASES for w, c in cs],
                         ids=lambda v: v if isinstance(v, str) else ",".join(f"{k}={x}" for k, x in v.items()) if len(v) < 5 else "")
def test_refused(name, good, word, change):
    _refused(word, name, *{**good, **change}.values())


def test_workspace_needed_is_checked():
    need = G.load().gn_logits_workspace(1, 1 << 20, 20)
    if need:
        wide = dict(LOGPROBS, rows=1, cols=1 << 20, ld=1 << 20, k=20)
        _refused("workspace", "gn_token_logprobs", *{**wide, "wsn": need - 1}.values())
        _refused("workspace", "gn_token_logprobs", *{**wide, "ws": None}.values())
        _refused("workspace", "gn_token_logprobs", *{**wide, "ws": P + 8}.values())
        need = G.load().gn_logits_workspace(1, 1 << 20, 0)
        _refused("workspace", "gn_distill_forward", *{**DISTILL, "rows": 1, "cols": 1 << 20, "ld": 1 << 20, "wsn": need - 1}.values())
    assert G.load().gn_logits_workspace(-1, 5, 0) == 0


# ------------------------------------------------------------------ the Python binding's own checks
def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def _pair(rows, cols):
    return G.mxfp4_empty(rows, cols, device="cpu")


I64, H = torch.int64, torch.float16
BINDING = [
    ("float32 or float16", lambda: G.mxfp4_quantize(_t(4, 8, dtype=torch.float64), *_pair(4, 8))),
    ("dense rows", lambda: G.mxfp4_quantize(_t(8, 4).t(), *_pair(4, 8))),
    ("dense rows", lambda: G.mxfp4_quantize(_t(1, 8).expand(4, 8), *_pair(4, 8))),
    ("values", lambda: G.mxfp4_quantize(_t(4, 129), *_pair(4, 128))),
    ("values", lambda: G.mxfp4_quantize(_t(4, 8), *_pair(5, 8))),
    ("values", lambda: G.mxfp4_quantize(_t(4, 8), _pair(4, 8)[0], _t(4, 4))),
    ("values", lambda: G.mxfp4_quantize(_t(4, 8), _pair(8, 8)[0][::2], _pair(4, 8)[1])),
    ("gemm: A", lambda: G.mxfp4_gemm(_pair(3, 8), _pair(3, 8), _t(2, 3), K=8)),
    ("current GPU", lambda: G.mxfp4_quantize(_t(4, 8), *_pair(4, 8))),
    ("values", lambda: G.mxfp4_dequantize(*_pair(4, 8), _t(3, 8))),
    ("C is float32", lambda: G.mxfp4_gemm(_t(2, 8, dtype=H), _pair(3, 8), _t(2, 3, dtype=H))),
    ("A is float16", lambda: G.mxfp4_gemm(_t(2, 8), _pair(3, 8), _t(2, 3))),
    ("A is float16", lambda: G.mxfp4_gemm(_t(2, 8, dtype=H), _pair(3, 8), _t(2, 3), K=9)),
    ("rows of A", lambda: G.mxfp4_gemm(_t(4, 8, dtype=H), _pair(3, 8), _t(2, 3))),
    ("gemm: B", lambda: G.mxfp4_gemm(_t(2, 8, dtype=H), _pair(4, 8), _t(2, 3))),
    ("gemm: B", lambda: G.mxfp4_gemm(_pair(2, 129), _pair(3, 128), _t(2, 3), K=129)),
    # as many values, other rows
    ("gemm: A", lambda: G.mxfp4_gemm(_pair(3, 256), _pair(3, 128), _t(6, 3), K=128)),
    ("gemm: B", lambda: G.mxfp4_gemm(_t(2, 128, dtype=H), _pair(3, 256), _t(2, 6))),
    ("bias", lambda: G.mxfp4_gemm(_t(2, 8, dtype=H), _pair(3, 8), _t(2, 3), bias=_t(2))),
    ("together", lambda: G.token_logprobs(_t(2, 8), _t(2, dtype=I64), None)),
    ("together", lambda: G.token_logprobs(_t(2, 8), None, None, top_ids=_t(2, 3, dtype=I64))),
    ("targets", lambda: G.token_logprobs(_t(2, 8), _t(2, dtype=torch.int32), _t(2))),
    ("targets", lambda: G.token_logprobs(_t(2, 8), _t(3, dtype=I64), _t(2))),
    ("top_logprobs", lambda: G.token_logprobs(_t(2, 8), None, None, top_ids=_t(2, 3, dtype=I64), top_logprobs=_t(2, 4))),
    ("lse", lambda: G.token_logprobs(_t(2, 8), None, None, lse=_t(2, dtype=H))),
    ("type and shape", lambda: G.token_logprobs_backward(_t(2, 8), None, _t(2), None, _t(2, 8, dtype=H))),
    ("together", lambda: G.token_logprobs_backward(_t(2, 8), None, _t(2), None, _t(2, 8), entropy=_t(2))),
    ("ids", lambda: G.distill(_t(2, 8), _t(2, 3), _t(2, 3), _t(2))),
    ("teacher", lambda: G.distill(_t(2, 8), _t(2, 3, dtype=I64), _t(2, 4), _t(2))),
    ("teacher", lambda: G.distill(_t(2, 8), _t(2, 3, dtype=I64), _t(3, 2), _t(2))),
    ("loss", lambda: G.distill(_t(2, 8), _t(2, 3, dtype=I64), _t(2, 3), _t(3))),
    ("type and shape", lambda: G.distill_backward(_t(2, 8), _t(2, 3, dtype=I64), _t(2, 3), _t(2), _t(2), _t(2, 9))),
    ("grad_loss", lambda: G.distill_backward(_t(2, 8), _t(2, 3, dtype=I64), _t(2, 3), _t(2), _t(2, dtype=H), _t(2, 8))),
    ("current GPU", lambda: G.distill(_t(2, 8), _t(2, 3, dtype=I64), _t(2, 3), _t(2))),
]


@pytest.mark.parametrize("i", range(len(BINDING)))
def test_binding_refuses(i):
    word, call = BINDING[i]
    with pytest.raises(G.GonngpuError, match=word):
        call()


@pytest.mark.parametrize("name,good", [("gn_token_logprobs", LOGPROBS), ("gn_token_logprobs_backward", LOGPROBS_GRAD),
                                       ("gn_distill_forward", DISTILL), ("gn_distill_backward", DISTILL_GRAD)])
@pytest.mark.parametrize("temperature", [1e-45, 2.9e-39, 2.95e-39, 3.5e-39, 4.23e-39])
def test_temperature_whose_exponents_would_be_infinite(name, good, temperature):
    """The reciprocal may be finite, but not its product with log2(e), which the exponents are multiplied with."""
    _refused("temperature", name, *{**good, "temp": temperature}.values())
