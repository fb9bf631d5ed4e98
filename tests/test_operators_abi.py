"""Host-side validation of the row, 8-bit and log-probability entry points: each refusal comes
before any CUDA call, with its documented status (runs without a GPU)."""
import ctypes
import math

import pytest
import torch

from race_attention_b200 import _lib
from test_abi import status_codes

P = ctypes.c_void_p(256)  # never dereferenced: validation fails first
OFF = ctypes.c_void_p(264)
F32, BF16 = _lib.RACE_F32, _lib.RACE_BF16
BAD = 7


def _code(rc):
    return {v: k for k, v in status_codes().items()}[rc]


def norm_fwd(x=P, xs=64, r=P, rs=64, dt=F32, w=P, wd=F32, y=P, h=P, rstd=P, rows=4, K=64):
    return _code(_lib.load().race_rms_norm_fwd(x, xs, r, rs, dt, w, wd, y, h, rstd, rows, K, 1e-5, None))


def norm_int8(x=P, xs=64, r=P, rs=64, dt=F32, w=P, wd=F32, q=P, qs=64, s=P, h=P, rows=4, K=64):
    return _code(_lib.load().race_rms_norm_int8(x, xs, r, rs, dt, w, wd, q, qs, s, h, rows, K, 1e-5, None))


def norm_bwd(dy=P, h=P, rstd=P, dt=F32, w=P, wd=F32, dx=P, dw=P, rows=4, K=64, ws=P, nb=1 << 30):
    return _code(_lib.load().race_rms_norm_bwd(dy, None, h, rstd, dt, w, wd, dx, dw, rows, K, ws, nb, None))


def quant(x=P, xs=64, dt=F32, q=P, qs=64, s=P, rows=4, K=64):
    return _code(_lib.load().race_quant_int8(x, xs, dt, q, qs, s, rows, K, None))


def swiglu(x=P, xs=128, dt=F32, q=P, qs=64, s=P, rows=4, F=64):
    return _code(_lib.load().race_swiglu_int8(x, xs, dt, q, qs, s, rows, F, None))


def dequant(q=P, qs=64, s=P, o=P, dt=F32, rows=4, K=64):
    return _code(_lib.load().race_dequant_int8(q, qs, s, o, dt, rows, K, None))


def linear(x=P, xs=64, s=P, w=P, ws=64, t=P, b=None, y=P, dt=F32, M=4, N=8, K=64):
    return _code(_lib.load().race_int8_linear(x, xs, s, w, ws, t, b, y, dt, M, N, K, None))


def logp_fwd(l=P, st=100, dt=F32, t=P, temp=1.0, n=2, lp=P, e=P, lse=P, ids=P, top=P, rows=4, V=100):
    return _code(_lib.load().race_token_logprobs_fwd(l, st, dt, t, -100, temp, n, lp, e, lse, ids, top, rows, V, None))


def logp_bwd(l=P, st=100, dt=F32, t=P, temp=1.0, lse=P, e=P, d=P, rows=4, V=100):
    return _code(_lib.load().race_token_logprobs_bwd(l, st, dt, t, -100, temp, lse, e, P, P, d, rows, V, None))


@pytest.mark.parametrize("call,bad", [
    (norm_fwd, [dict(x=None), dict(y=None), dict(h=None)]),
    (norm_int8, [dict(x=None), dict(q=None), dict(s=None), dict(h=None)]),
    (norm_bwd, [dict(dy=None), dict(h=None), dict(rstd=None), dict(dx=None)]),
    (quant, [dict(x=None), dict(q=None), dict(s=None)]),
    (swiglu, [dict(x=None), dict(q=None), dict(s=None)]),
    (dequant, [dict(q=None), dict(s=None), dict(o=None)]),
    (linear, [dict(x=None), dict(s=None), dict(w=None), dict(t=None), dict(y=None)]),
    (logp_fwd, [dict(l=None), dict(t=None), dict(lp=None), dict(e=None), dict(ids=None), dict(top=None)]),
    (logp_bwd, [dict(l=None), dict(t=None), dict(lse=None), dict(e=None), dict(d=None)]),
])
def test_null_pointers_and_dtypes(call, bad):
    for kw in bad:
        assert call(**kw) == "RACE_ERR_ARG", kw
        assert "null" in _lib.load().race_last_error().decode()
    assert call(dt=BAD) == "RACE_ERR_DTYPE"


@pytest.mark.parametrize("call,width", [(norm_fwd, "K"), (norm_int8, "K"), (norm_bwd, "K"), (quant, "K"), (swiglu, "F"),
                                        (dequant, "K"), (logp_fwd, "V"), (logp_bwd, "V")])
def test_sizes(call, width):
    for kw in (dict(rows=0), dict(rows=1 << 31), {width: 0}, {width: 1 << 31}):
        assert call(**kw) == "RACE_ERR_SHAPE", kw


def test_strides_and_weights():
    assert norm_fwd(xs=63) == norm_fwd(rs=63) == norm_int8(qs=63) == quant(xs=63) == quant(qs=63) == "RACE_ERR_SHAPE"
    assert swiglu(xs=127) == swiglu(qs=63) == dequant(qs=63) == logp_fwd(st=99) == logp_bwd(st=99) == "RACE_ERR_SHAPE"
    assert norm_fwd(wd=BAD) == norm_int8(wd=BAD) == norm_bwd(wd=BAD) == "RACE_ERR_DTYPE"
    need = _lib.load().race_rms_norm_bwd_workspace_bytes(4, 64)
    assert need > 0 and _lib.load().race_rms_norm_bwd_workspace_bytes(0, 64) == 0
    assert norm_bwd(ws=None) == norm_bwd(nb=need - 1) == "RACE_ERR_WORKSPACE"


def _at(n):
    return ctypes.c_void_p(256 + n)


@pytest.mark.parametrize("call,arrays", [
    (norm_fwd, dict(x=4, r=4, w=4, y=4, h=4, rstd=4)), (norm_int8, dict(x=4, r=4, w=4, s=4, h=4)),
    (norm_bwd, dict(dy=4, h=4, rstd=4, w=4, dx=4, dw=4, ws=4)), (quant, dict(x=4, s=4)), (swiglu, dict(x=4, s=4)),
    (dequant, dict(s=4, o=4)), (linear, dict(s=4, t=4, b=4, y=4)),
    (logp_fwd, dict(l=4, t=8, lp=4, e=4, lse=8, ids=8, top=4)), (logp_bwd, dict(l=4, t=8, lse=8, e=4, d=4)),
])
def test_arrays_that_start_inside_a_value(call, arrays):
    for name, size in arrays.items():
        for n in (1, size // 2):
            assert call(**{name: _at(n)}) == "RACE_ERR_ALIGN", (name, n)


def test_arrays_of_bf16_that_start_inside_a_value():
    for call, names in ((norm_fwd, "x r y h"), (norm_int8, "x r h"), (norm_bwd, "dy h dx"), (quant, "x"), (swiglu, "x"),
                        (dequant, "o"), (linear, "y"), (logp_fwd, "l"), (logp_bwd, "l d")):
        for name in names.split():
            assert call(dt=BF16, **{name: _at(1)}) == "RACE_ERR_ALIGN", name
    for call in (norm_fwd, norm_int8, norm_bwd):
        assert call(w=_at(1), wd=BF16) == "RACE_ERR_ALIGN"
    assert norm_bwd(w=None, dw=_at(1), wd=BF16) == "RACE_ERR_ALIGN"


def test_linear():
    assert linear(M=0) == linear(N=0) == linear(K=0) == linear(K=131072) == linear(M=1 << 31) == "RACE_ERR_SHAPE"
    assert linear(xs=48) == linear(ws=48) == "RACE_ERR_SHAPE"
    assert linear(x=OFF) == linear(w=OFF) == linear(xs=72) == linear(ws=72) == "RACE_ERR_ALIGN"
    assert linear(s=ctypes.c_void_p(258)) == linear(b=ctypes.c_void_p(257)) == "RACE_ERR_ALIGN"


def test_logprobs():
    assert logp_fwd(n=-1) == logp_fwd(n=33) == logp_fwd(n=3, V=2) == "RACE_ERR_SHAPE"
    for temp in (0.0, -1.0, math.inf, math.nan, 1e-39):
        assert logp_fwd(temp=temp) == logp_bwd(temp=temp) == "RACE_ERR_ARG"
    assert logp_fwd(lse=ctypes.c_void_p(260)) == logp_bwd(lse=ctypes.c_void_p(260)) == "RACE_ERR_ALIGN"


def test_host_tensors_are_refused():
    import race_attention_b200 as rb
    x, s = torch.zeros(2, 64), torch.zeros(2)
    rows = rb.Int8Rows(torch.zeros(2, 64, dtype=torch.int8), s)
    for call in (lambda: rb.add_rms_norm(x), lambda: rb.add_rms_norm_int8(x), lambda: rb.quant_int8(x),
                 lambda: rb.swiglu_int8(x), lambda: rows.dequant(), lambda: rb.int8_linear(rows, rows),
                 lambda: rb.token_logprobs(x, torch.zeros(2, dtype=torch.int64)),
                 lambda: rb.add_rms_norm(x.requires_grad_(True))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
