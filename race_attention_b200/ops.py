"""Torch-level calls into the C ABI (no autograd here; see race_causal_cuda.py).

Each function validates its tensors the way the reference extension does
(CUDA-only, dtype, rank -> RuntimeError, kernels/gpu/forward_kernel.cu:112-114,
kernels/gpu/backward_kernels.cu:176-179), allocates outputs and workspace with
torch on the inputs' device, and launches on torch's current stream under a
device guard.  torch is only plumbing here: memory, streams and devices.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_DT = {torch.float32: _lib.RACE_F32, torch.bfloat16: _lib.RACE_BF16}


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(dev):
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _check_cuda(*ts):
    dev, index = None, -1
    for t in ts:
        if t is None:
            continue
        i = t.get_device()  # -1: not on a GPU
        if i < 0:
            raise RuntimeError("CUDA only")
        if dev is None:
            dev, index = t.device, i
        elif i != index:
            raise RuntimeError("all tensors must be on the same CUDA device")
    return dev


def _dtype_code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise RuntimeError(f"unsupported dtype {t.dtype} (float32 or bfloat16)") from None


def _dtype_code_of(dtype):
    try:
        return _DT[dtype]
    except KeyError:
        raise RuntimeError(f"unsupported dtype {dtype} (float32 or bfloat16)") from None


def _workspace(op, N, T, S, D, L, P, dtype, dev):
    lib = _lib.load()
    nbytes = ctypes.c_size_t(0)
    _lib.check(lib.race_workspace_bytes(op, N, T, S, D, L, P, dtype, 0, ctypes.byref(nbytes)),
               "race_workspace_bytes")
    n = int(nbytes.value)
    return torch.empty(max(n, 1), dtype=torch.uint8, device=dev), n


def _as_ntd(x, name):
    if x.dim() == 4:
        x = x.reshape(-1, x.shape[2], x.shape[3])
    if x.dim() != 3:
        raise RuntimeError(f"{name} must be [N,T,D] or [B,H,T,D]")
    return x.contiguous()


def _opt_state(A, B, N, S, D, dev):
    if A is None and B is None:
        return None, None
    if A is None or B is None:
        raise RuntimeError("state A and B must be given together")
    A = A.to(device=dev, dtype=torch.float32).reshape(N, S).contiguous()
    B = B.to(device=dev, dtype=torch.float32).reshape(N, S, D).contiguous()
    return A, B


def fast_path(dtype, D, L, P) -> bool:
    """Whether the library runs the tcgen05 kernels for this configuration
    (same rule as csrc/fast_host.cuh: bf16, D=64, P=4, L in {8,16})."""
    return dtype == torch.bfloat16 and D == 64 and P == 4 and L in (8, 16)


def default_logit_scale(D: int) -> float:
    """The reference divides tanh(proj) by sqrt(D) (scaling/race_common.py:46,68)."""
    return 1.0 / math.sqrt(D)


# ---------------------------------------------------------------------------
# probability-level (reference extension surface)
def race_fused_fwd(probsK, probsQ, V2, eps, chunk=0, return_state=False):
    """out[N,T,D] = causal RACE forward (kernels/gpu/forward_kernel.cu:110 semantics)."""
    dev = _check_cuda(probsK, probsQ, V2)
    if probsK.dtype != torch.float32 or probsQ.dtype != torch.float32 or V2.dtype != torch.float32:
        raise RuntimeError("fp32 only")
    if probsK.dim() != 3 or probsQ.dim() != 3 or V2.dim() != 3:
        raise RuntimeError("shapes [N,T,S],[N,T,S],[N,T,D]")
    probsK, probsQ, V2 = probsK.contiguous(), probsQ.contiguous(), V2.contiguous()
    N, T, S = probsK.shape
    D = V2.shape[2]
    if probsQ.shape != probsK.shape or V2.shape[:2] != probsK.shape[:2]:
        raise RuntimeError("shapes [N,T,S],[N,T,S],[N,T,D]")
    out = torch.empty((N, T, D), dtype=torch.float32, device=dev)
    Af = torch.empty((N, S), dtype=torch.float32, device=dev) if return_state else None
    Bf = torch.empty((N, S, D), dtype=torch.float32, device=dev) if return_state else None
    if T == 0:
        if return_state:
            Af.zero_()
            Bf.zero_()
        return (out, Af, Bf) if return_state else out
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_FWD_PROBS, N, T, S, D, 0, 0, 0, dev)
        _lib.check(lib.race_fwd_probs(_ptr(probsK), _ptr(probsQ), _ptr(V2), _ptr(out), _ptr(Af), _ptr(Bf),
                                      N, T, S, D, float(eps), int(chunk), _ptr(ws), nb, _stream(dev)),
                   "race_fwd_probs")
    return (out, Af, Bf) if return_state else out


def race_backward(probsK, probsQ, V2, grad_out, eps, chunk=0):
    """[gradProbsK, gradProbsQ, gradV] (kernels/gpu/backward_kernels.cu:174 semantics)."""
    dev = _check_cuda(probsK, probsQ, V2, grad_out)
    for t in (probsK, probsQ, V2, grad_out):
        if t.dtype != torch.float32:
            raise RuntimeError("fp32 only")
    probsK, probsQ, V2, grad_out = (t.contiguous() for t in (probsK, probsQ, V2, grad_out))
    N, T, S = probsK.shape
    D = V2.shape[2]
    if S > 1024:
        raise RuntimeError("S must be <= 1024")
    gpk = torch.empty_like(probsK)
    gpq = torch.empty_like(probsQ)
    gv = torch.empty_like(V2)
    if T == 0:
        return [gpk, gpq, gv]
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_BWD_PROBS, N, T, S, D, 0, 0, 0, dev)
        _lib.check(lib.race_bwd_probs(_ptr(probsK), _ptr(probsQ), _ptr(V2), _ptr(grad_out), _ptr(gpk), _ptr(gpq),
                                      _ptr(gv), N, T, S, D, float(eps), int(chunk), _ptr(ws), nb, _stream(dev)),
                   "race_bwd_probs")
    return [gpk, gpq, gv]


# ---------------------------------------------------------------------------
# soft hash
def soft_hash(X, planes_T, L, P, logit_scale=None):
    """probs[N,T,L*2^P] fp32 of X [N,T,D] (bf16 or fp32)."""
    dev = _check_cuda(X, planes_T)
    X = _as_ntd(X, "X")
    N, T, D = X.shape
    S = L << P
    planes_T = planes_T.to(torch.float32).contiguous()
    if planes_T.shape != (D, L * P):
        raise RuntimeError(f"planes_T must be [D, L*P] = [{D}, {L * P}]")
    scale = default_logit_scale(D) if logit_scale is None else float(logit_scale)
    probs = torch.empty((N, T, S), dtype=torch.float32, device=dev)
    if N * T == 0:
        return probs
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.race_soft_hash(_ptr(X), _dtype_code(X), _ptr(planes_T), _ptr(probs), N, T, D, L, P, scale,
                                      _stream(dev)), "race_soft_hash")
    return probs


def soft_hash_bwd(X, planes_T, dprobs, L, P, logit_scale=None):
    dev = _check_cuda(X, planes_T, dprobs)
    X = _as_ntd(X, "X")
    N, T, D = X.shape
    planes_T = planes_T.to(torch.float32).contiguous()
    dprobs = dprobs.to(torch.float32).reshape(N, T, L << P).contiguous()
    scale = default_logit_scale(D) if logit_scale is None else float(logit_scale)
    dX = torch.empty_like(X)
    if N * T == 0:
        return dX
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.race_soft_hash_bwd(_ptr(X), _dtype_code(X), _ptr(planes_T), _ptr(dprobs), _ptr(dX), N, T, D,
                                          L, P, scale, _stream(dev)), "race_soft_hash_bwd")
    return dX


# ---------------------------------------------------------------------------
# fused layer
def _qkv_common(Q, K, V, planes_T, L, P, logit_scale):
    dev = _check_cuda(Q, K, V, planes_T)
    Q, K, V = _as_ntd(Q, "Q"), _as_ntd(K, "K"), _as_ntd(V, "V")
    if not (Q.shape == K.shape == V.shape):
        raise RuntimeError("Q, K, V must have the same shape")
    if not (Q.dtype == K.dtype == V.dtype):
        raise RuntimeError("Q, K, V must have the same dtype")
    N, T, D = Q.shape
    planes_T = planes_T.to(torch.float32).contiguous()
    if planes_T.shape != (D, L * P):
        raise RuntimeError(f"planes_T must be [D, L*P] = [{D}, {L * P}]")
    scale = default_logit_scale(D) if logit_scale is None else float(logit_scale)
    return dev, Q, K, V, planes_T, N, T, D, L << P, scale


def saved_bytes(N, T, D, L, P, dtype) -> int:
    """Size of the chunk-state buffer a saving forward keeps for the backward (0: not used)."""
    nb = ctypes.c_size_t(0)
    _lib.check(_lib.load().race_saved_bytes(N, T, D, L, P, _dtype_code_of(dtype), ctypes.byref(nb)),
               "race_saved_bytes")
    return int(nb.value)


def fwd_qkv(Q, K, V, planes_T, L, P, eps=1e-6, logit_scale=None, A0=None, B0=None, return_state=False,
            save=False):
    """Fused soft hash + causal scan + readout; out has Q's dtype and [N,T,D] shape.
    save=True also returns the chunk-state buffer for bwd_qkv(saved=...) (None when unused)."""
    dev, Q, K, V, planes_T, N, T, D, S, scale = _qkv_common(Q, K, V, planes_T, L, P, logit_scale)
    A0, B0 = _opt_state(A0, B0, N, S, D, dev)
    out = torch.empty_like(Q)
    Af = torch.empty((N, S), dtype=torch.float32, device=dev) if return_state else None
    Bf = torch.empty((N, S, D), dtype=torch.float32, device=dev) if return_state else None
    lib = _lib.load()
    saved = None
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_FWD_QKV, N, T, S, D, L, P, _dtype_code(Q), dev)
        sb = saved_bytes(N, T, D, L, P, Q.dtype) if save else 0
        if sb:
            saved = torch.empty(sb, dtype=torch.uint8, device=dev)
        _lib.check(lib.race_fwd_qkv_save(_ptr(Q), _ptr(K), _ptr(V), _dtype_code(Q), _ptr(planes_T), _ptr(out),
                                         _ptr(A0), _ptr(B0), _ptr(Af), _ptr(Bf), _ptr(saved), sb, N, T, D, L, P,
                                         float(eps), scale, _ptr(ws), nb, _stream(dev)), "race_fwd_qkv")
    res = (out, Af, Bf) if return_state else (out,)
    if save:
        res = res + (saved,)
    return res if len(res) > 1 else res[0]


def bwd_qkv(Q, K, V, dO, planes_T, L, P, eps=1e-6, logit_scale=None, A0=None, B0=None, gA=None, gB=None,
            return_state_grad=False, saved=None):
    """(dQ, dK, dV[, dA0, dB0]) of the fused layer.  saved: the buffer of fwd_qkv(save=True) on the
    same inputs (skips rebuilding the forward's chunk states)."""
    dev, Q, K, V, planes_T, N, T, D, S, scale = _qkv_common(Q, K, V, planes_T, L, P, logit_scale)
    dO = _as_ntd(dO, "dO").to(Q.dtype)
    A0, B0 = _opt_state(A0, B0, N, S, D, dev)
    gA, gB = _opt_state(gA, gB, N, S, D, dev)
    dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
    dA0 = torch.empty((N, S), dtype=torch.float32, device=dev) if return_state_grad else None
    dB0 = torch.empty((N, S, D), dtype=torch.float32, device=dev) if return_state_grad else None
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_BWD_QKV, N, T, S, D, L, P, _dtype_code(Q), dev)
        sb = saved.numel() if saved is not None else 0
        _lib.check(lib.race_bwd_qkv_saved(_ptr(Q), _ptr(K), _ptr(V), _ptr(dO), _dtype_code(Q), _ptr(planes_T),
                                          _ptr(saved), sb, _ptr(dQ), _ptr(dK), _ptr(dV), _ptr(A0), _ptr(B0),
                                          _ptr(gA), _ptr(gB), _ptr(dA0), _ptr(dB0), N, T, D, L, P, float(eps), scale,
                                          _ptr(ws), nb, _stream(dev)), "race_bwd_qkv")
    return (dQ, dK, dV, dA0, dB0) if return_state_grad else (dQ, dK, dV)


def _bthd_common(Q, K, V, planes_T, L, P, logit_scale):
    dev = _check_cuda(Q, K, V, planes_T)
    if Q.dim() != 4 or not (Q.shape == K.shape == V.shape):
        raise RuntimeError("Q, K, V must have the same [B,T,H,D] shape")
    if not (Q.dtype == K.dtype == V.dtype):
        raise RuntimeError("Q, K, V must have the same dtype")
    Bn, T, H, D = Q.shape
    if not fast_path(Q.dtype, D, L, P):
        raise RuntimeError("the [B,T,H,D] layout needs bf16, D=64, P=4, L in {8,16}")
    planes_T = planes_T.to(torch.float32).contiguous()
    if planes_T.shape != (D, L * P):
        raise RuntimeError(f"planes_T must be [D, L*P] = [{D}, {L * P}]")
    scale = default_logit_scale(D) if logit_scale is None else float(logit_scale)
    return dev, Q.contiguous(), K.contiguous(), V.contiguous(), planes_T, Bn, T, H, D, L << P, scale


def fwd_bthd(Q, K, V, planes_T, L, P, eps=1e-6, logit_scale=None):
    """Fused layer on [B,T,H,D] activations (no transposes): (out [B,T,H,D], saved chunk states)."""
    dev, Q, K, V, planes_T, Bn, T, H, D, S, scale = _bthd_common(Q, K, V, planes_T, L, P, logit_scale)
    N = Bn * H
    out = torch.empty_like(Q)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_FWD_QKV, N, T, S, D, L, P, _dtype_code(Q), dev)
        sb = saved_bytes(N, T, D, L, P, Q.dtype)
        saved = torch.empty(max(sb, 1), dtype=torch.uint8, device=dev)
        _lib.check(lib.race_fwd_bthd(_ptr(Q), _ptr(K), _ptr(V), _dtype_code(Q), _ptr(planes_T), _ptr(out), _ptr(saved),
                                     sb, Bn, T, H, D, L, P, float(eps), scale, _ptr(ws), nb, _stream(dev)),
                   "race_fwd_bthd")
    return out, saved


def bwd_bthd(Q, K, V, dO, planes_T, L, P, saved, eps=1e-6, logit_scale=None):
    """(dQ, dK, dV) [B,T,H,D] of fwd_bthd, reusing its saved chunk states."""
    dev, Q, K, V, planes_T, Bn, T, H, D, S, scale = _bthd_common(Q, K, V, planes_T, L, P, logit_scale)
    N = Bn * H
    dO = dO.to(Q.dtype).contiguous()
    dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_BWD_QKV, N, T, S, D, L, P, _dtype_code(Q), dev)
        _lib.check(lib.race_bwd_bthd(_ptr(Q), _ptr(K), _ptr(V), _ptr(dO), _dtype_code(Q), _ptr(planes_T), _ptr(saved),
                                     saved.numel(), _ptr(dQ), _ptr(dK), _ptr(dV), Bn, T, H, D, L, P, float(eps), scale,
                                     _ptr(ws), nb, _stream(dev)), "race_bwd_bthd")
    return dQ, dK, dV


def state_from_prefill(K, V, planes_T, L, P, logit_scale=None, A0=None, B0=None):
    """(A[N,S], B[N,S,D]) fp32 state after the prefill tokens K, V [N,T,D]."""
    dev, K, _, V, planes_T, N, T, D, S, scale = _qkv_common(K, K, V, planes_T, L, P, logit_scale)
    A0, B0 = _opt_state(A0, B0, N, S, D, dev)
    A = torch.empty((N, S), dtype=torch.float32, device=dev)
    B = torch.empty((N, S, D), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_STATE, N, T, S, D, L, P, _dtype_code(K), dev)
        _lib.check(lib.race_state_from_prefill(_ptr(K), _ptr(V), _dtype_code(K), _ptr(planes_T), _ptr(A0), _ptr(B0),
                                               _ptr(A), _ptr(B), N, T, D, L, P, scale, _ptr(ws), nb, _stream(dev)),
                   "race_state_from_prefill")
    return A, B


def ace_fwd(Q, K, V, planes_T, L, P, eps=1e-6, logit_scale=None):
    """Non-causal RACE forward on [N,T,D] (tcgen05 path only: bf16, D=64, P=4, L in {8,16}):
    (out [N,T,D], A [N,S], B [N,S,D]); A and B are the bucket summaries the backward takes."""
    dev, Q, K, V, planes_T, N, T, D, S, scale = _qkv_common(Q, K, V, planes_T, L, P, logit_scale)
    if not fast_path(Q.dtype, D, L, P):
        raise RuntimeError("race_ace_fwd: bf16, D=64, P=4, L in {8,16} only")
    out = torch.empty_like(Q)
    A = torch.empty((N, S), dtype=torch.float32, device=dev)
    B = torch.empty((N, S, D), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_ACE_FWD, N, T, S, D, L, P, _dtype_code(Q), dev)
        _lib.check(lib.race_ace_fwd(_ptr(Q), _ptr(K), _ptr(V), _dtype_code(Q), _ptr(planes_T), _ptr(out), _ptr(A),
                                    _ptr(B), N, T, D, L, P, float(eps), scale, _ptr(ws), nb, _stream(dev)),
                   "race_ace_fwd")
    return out, A, B


def ace_bwd(Q, K, V, dO, planes_T, A, B, L, P, eps=1e-6, logit_scale=None):
    """(dQ, dK, dV) [N,T,D] of ace_fwd, from its summaries A, B."""
    dev, Q, K, V, planes_T, N, T, D, S, scale = _qkv_common(Q, K, V, planes_T, L, P, logit_scale)
    if not fast_path(Q.dtype, D, L, P):
        raise RuntimeError("race_ace_bwd: bf16, D=64, P=4, L in {8,16} only")
    dO = _as_ntd(dO, "dO").to(Q.dtype)
    _check_cuda(Q, dO, A, B)
    A = A.float().reshape(N, S).contiguous()
    B = B.float().reshape(N, S, D).contiguous()
    dQ, dK, dV = torch.empty_like(Q), torch.empty_like(K), torch.empty_like(V)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_ACE_BWD, N, T, S, D, L, P, _dtype_code(Q), dev)
        _lib.check(lib.race_ace_bwd(_ptr(Q), _ptr(K), _ptr(V), _ptr(dO), _dtype_code(Q), _ptr(planes_T), _ptr(A),
                                    _ptr(B), _ptr(dQ), _ptr(dK), _ptr(dV), N, T, D, L, P, float(eps), scale,
                                    _ptr(ws), nb, _stream(dev)),
                   "race_ace_bwd")
    return dQ, dK, dV


class FwdSplit:
    """What race_fwd_local leaves for race_fwd_finish: K, V and the workspace."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def fwd_local(K, V, planes_T, L, P, logit_scale=None):
    """First half of a shard's forward: (A_tot[N,S], B_tot[N,S,D], handle) -- this shard's state
    totals; the handle (holding its segment prefixes) goes to fwd_finish."""
    dev, K, _, V, planes_T, N, T, D, S, scale = _qkv_common(K, K, V, planes_T, L, P, logit_scale)
    A = torch.empty((N, S), dtype=torch.float32, device=dev)
    B = torch.empty((N, S, D), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_FWD_SPLIT, N, T, S, D, L, P, _dtype_code(K), dev)
        _lib.check(lib.race_fwd_local(_ptr(K), _ptr(V), _dtype_code(K), _ptr(planes_T), _ptr(A), _ptr(B), N, T, D,
                                      L, P, scale, _ptr(ws), nb, _stream(dev)), "race_fwd_local")
    return A, B, FwdSplit(K=K, V=V, planes_T=planes_T, L=L, P=P, scale=scale, ws=ws, nb=nb, dev=dev)


def fwd_finish(h, Q, A0=None, B0=None, eps=1e-6, save=False):
    """Second half: out (and, with save=True, the chunk-state buffer for bwd_local/bwd_qkv, None when
    unused) given A0/B0 = the sum of the totals of all earlier shards."""
    dev, Q, K, V, planes_T, N, T, D, S, _ = _qkv_common(Q, h.K, h.V, h.planes_T, h.L, h.P, h.scale)
    A0, B0 = _opt_state(A0, B0, N, S, D, dev)
    out = torch.empty_like(Q)
    lib = _lib.load()
    saved = None
    with torch.cuda.device(dev):
        sb = saved_bytes(N, T, D, h.L, h.P, Q.dtype) if save else 0
        if sb:
            saved = torch.empty(sb, dtype=torch.uint8, device=dev)
        _lib.check(lib.race_fwd_finish(_ptr(Q), _ptr(K), _ptr(V), _dtype_code(Q), _ptr(planes_T), _ptr(out),
                                       _ptr(saved), sb, _ptr(A0), _ptr(B0), N, T, D, h.L, h.P, float(eps), h.scale,
                                       _ptr(h.ws), h.nb, _stream(dev)), "race_fwd_finish")
    return (out, saved) if save else out


class BwdSplit:
    """What race_bwd_local leaves for race_bwd_finish: the inputs and the workspace."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def bwd_local(Q, K, V, dO, planes_T, L, P, eps=1e-6, logit_scale=None, A0=None, B0=None, saved=None):
    """First half of a shard's backward: (gA_tot[N,S], gB_tot[N,S,D], handle) -- this shard's
    gradient totals for its start state; the handle goes to bwd_finish."""
    dev, Q, K, V, planes_T, N, T, D, S, scale = _qkv_common(Q, K, V, planes_T, L, P, logit_scale)
    dO = _as_ntd(dO, "dO").to(Q.dtype)
    A0, B0 = _opt_state(A0, B0, N, S, D, dev)
    gA = torch.empty((N, S), dtype=torch.float32, device=dev)
    gB = torch.empty((N, S, D), dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws, nb = _workspace(_lib.OP_BWD_SPLIT, N, T, S, D, L, P, _dtype_code(Q), dev)
        sb = saved.numel() if saved is not None else 0
        _lib.check(lib.race_bwd_local(_ptr(Q), _ptr(K), _ptr(V), _ptr(dO), _dtype_code(Q), _ptr(planes_T),
                                      _ptr(saved), sb, _ptr(A0), _ptr(B0), _ptr(gA), _ptr(gB), N, T, D, L, P,
                                      float(eps), scale, _ptr(ws), nb, _stream(dev)), "race_bwd_local")
    h = BwdSplit(Q=Q, K=K, V=V, dO=dO, planes_T=planes_T, L=L, P=P, eps=eps, scale=scale, A0=A0, B0=B0,
                 saved=saved, ws=ws, nb=nb, dev=dev)
    return gA, gB, h


def bwd_finish(h, gA=None, gB=None):
    """Second half: (dQ, dK, dV) given gA/gB = the sum of the totals of all later shards."""
    N, T, D = h.Q.shape
    S = h.L << h.P
    gA, gB = _opt_state(gA, gB, N, S, D, h.dev)
    dQ, dK, dV = torch.empty_like(h.Q), torch.empty_like(h.K), torch.empty_like(h.V)
    lib = _lib.load()
    with torch.cuda.device(h.dev):
        sb = h.saved.numel() if h.saved is not None else 0
        _lib.check(lib.race_bwd_finish(_ptr(h.Q), _ptr(h.K), _ptr(h.V), _ptr(h.dO), _dtype_code(h.Q),
                                       _ptr(h.planes_T), _ptr(h.saved), sb, _ptr(h.A0), _ptr(h.B0), _ptr(gA),
                                       _ptr(gB), _ptr(dQ), _ptr(dK), _ptr(dV), N, T, D, h.L, h.P, float(h.eps),
                                       h.scale, _ptr(h.ws), h.nb, _stream(h.dev)), "race_bwd_finish")
    return dQ, dK, dV


def decode_step(q, k, v, planes_T, A, B, L, P, eps=1e-6, logit_scale=None):
    """One decode token.  q [Nq,D], k/v [Nkv,D] (Nq = group*Nkv); updates A/B in place; returns out [Nq,D]."""
    dev = _check_cuda(q, k, v, planes_T, A, B)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if not (q.dtype == k.dtype == v.dtype):
        raise RuntimeError("q, k, v must have the same dtype")
    Nq, D = q.shape
    Nkv = k.shape[0]
    S = L << P
    if A.dtype != torch.float32 or B.dtype != torch.float32 or not A.is_contiguous() or not B.is_contiguous():
        raise RuntimeError("decode state A/B must be contiguous float32")
    if A.shape != (Nkv, S) or B.shape != (Nkv, S, D):
        raise RuntimeError(f"decode state must be A[{Nkv},{S}], B[{Nkv},{S},{D}]")
    planes_T = planes_T.to(torch.float32).contiguous()
    scale = default_logit_scale(D) if logit_scale is None else float(logit_scale)
    out = torch.empty_like(q)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.race_decode_step(_ptr(q), _ptr(k), _ptr(v), _dtype_code(q), _ptr(planes_T), _ptr(A), _ptr(B),
                                        _ptr(out), Nq, Nkv, D, L, P, float(eps), scale, _stream(dev)),
                   "race_decode_step")
    return out


def gqa_decode_splits(B, Hkv, t_max, device) -> int:
    """Key ranges per (batch row, kv head) for gqa_decode_attention: about 16 waves of
    two CTAs per SM over the whole grid, at least 512 cache slots per range, at most 64."""
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    want = -(-16 * 2 * sms // max(1, B * Hkv))
    return int(max(1, min(64, want, max(1, t_max // 512))))


def gqa_decode_workspace(B, Hq, Hkv, n_splits, device):
    """Zero-filled workspace for gqa_decode_attention (reused as is across calls)."""
    nbytes = int(_lib.load().race_gqa_decode_workspace_bytes(B, Hq, Hkv, int(n_splits)))
    if nbytes == 0:
        raise RuntimeError("invalid gqa_decode_attention workspace shape")
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def gqa_decode_attention(q, k_new, v_new, k_cache, v_cache, length, workspace, n_splits, softmax_scale=None):
    """Softmax GQA attention of one decode token over a bf16 KV cache (the softmax layers
    of a hybrid decoder).  q [B,Hq,64], k_new/v_new [B,Hkv,64], caches [B,Hkv,Tmax,64],
    length = int32 device tensor [1] holding the tokens already cached.  Stores k_new/v_new
    at position length, returns out [B,Hq,64]; length itself is not advanced."""
    dev = _check_cuda(q, k_new, v_new, k_cache, v_cache, length, workspace)
    for name, t in (("q", q), ("k_new", k_new), ("v_new", v_new), ("k_cache", k_cache), ("v_cache", v_cache)):
        if t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous bfloat16")
    if length.dtype != torch.int32 or length.numel() != 1:
        raise RuntimeError("length must be an int32 tensor with one element")
    B, Hq, D = q.shape
    Hkv, Tmax = k_cache.shape[1], k_cache.shape[2]
    if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D) or k_cache.shape != (B, Hkv, Tmax, D) \
            or v_cache.shape != k_cache.shape:
        raise RuntimeError("gqa_decode_attention: inconsistent shapes")
    lib = _lib.load()
    need = int(lib.race_gqa_decode_workspace_bytes(B, Hq, Hkv, int(n_splits)))
    if workspace.numel() * workspace.element_size() < need:
        raise RuntimeError(f"gqa_decode_attention workspace needs {need} bytes")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    out = torch.empty_like(q)
    with torch.cuda.device(dev):
        _lib.check(lib.race_gqa_decode_attn(_ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache),
                                            _ptr(length), _ptr(out), _ptr(workspace), B, Hq, Hkv, Tmax, D,
                                            int(n_splits), scale, _stream(dev)), "race_gqa_decode_attn")
    return out


# ---------------------------------------------------------------------------
# operators around the layer: residual RMS norm, 8-bit rows and products, token log
# probabilities.  Some of them run for a few microseconds on a decode step, so their checks
# are single passes over attributes and they launch without entering a device context where
# the tensors' device is current.  (None with a torch that has no CUDA: nothing is launched there.)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _launch(dev, name, *args):
    """Call C entry point `name` with args and the current stream of `dev`."""
    fn = getattr(_lib.load(), name)
    index = dev.index
    if index == _current_device():
        rc = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _current_stream(index))
    if rc:
        _lib.check(rc, name)


def _rows(x, name):
    """x [..., K] as (rows with unit stride inside a row, row stride, rows, K): a view where
    the rows are evenly spaced, else a copy."""
    shape = x.shape
    if not shape or not shape[-1]:
        raise RuntimeError(f"{name} must have rows of at least one value")
    K = shape[-1]
    if x.is_contiguous():
        return x, K, x.numel() // K, K
    if len(shape) != 2:
        x = x.reshape(-1, K)
    rows, stride = x.shape[0], x.stride(0)
    if x.stride(1) != 1 or (stride < K and rows > 1):  # strided or overlapping (expanded) rows
        x, stride = x.contiguous(), K
    return x, max(stride, K), rows, K


def _weight_code(weight, K):
    if weight is None:
        return _lib.RACE_F32
    if weight.shape != (K,) or not weight.is_contiguous():
        raise RuntimeError(f"weight must be a contiguous [{K}] tensor")
    return _dtype_code(weight)


def _norm_inputs(x, residual, weight):
    dev = _check_cuda(x, residual, weight)
    code = _dtype_code(x)
    xr, xs, rows, K = _rows(x, "x")
    rr, rs = None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise RuntimeError("residual must have x's shape and dtype")
        rr, rs, _, _ = _rows(residual, "residual")
    return dev, code, xr, xs, rr, rs, rows, K, _weight_code(weight, K)


def _ptr_of(t):
    return None if t is None else t.data_ptr()


def _dense_like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)


def rms_norm_fwd(x, residual=None, weight=None, eps=1e-5, return_rstd=False):
    """(y, h[, rstd]): h = x + residual in x's dtype (x itself without a residual),
    y = h * rsqrt(mean(h^2) + eps) * weight; x [..., K]."""
    dev, code, xr, xs, rr, rs, rows, K, wc = _norm_inputs(x, residual, weight)
    y = _dense_like(x)
    h = x if residual is None else _dense_like(x)
    rstd = x.new_empty(rows, dtype=torch.float32) if return_rstd else None
    if rows:
        _launch(dev, "race_rms_norm_fwd", xr.data_ptr(), xs, _ptr_of(rr), rs, code, _ptr_of(weight), wc, y.data_ptr(),
                None if residual is None else h.data_ptr(), _ptr_of(rstd), rows, K, eps)
    return (y, h, rstd) if return_rstd else (y, h)


def rms_norm_bwd(dy, dh, h, rstd, weight=None, weight_grad=True):
    """(dx, dw) of rms_norm_fwd for the gradients dy of y and dh of h (None: zero); dx is the
    gradient of x and of the residual alike, dw (None unless weight_grad) has weight's dtype."""
    _check_cuda(dy, dh, h, rstd, weight)
    if dy.shape != h.shape or dy.dtype != h.dtype or (dh is not None and (dh.shape != h.shape or dh.dtype != h.dtype)):
        raise RuntimeError("dy and dh must have h's shape and dtype")
    if rstd.dtype != torch.float32 or rstd.numel() * h.shape[-1] != h.numel():
        raise RuntimeError(f"rstd must hold {h.numel() // h.shape[-1]} float32 values")
    _weight_code(weight, h.shape[-1])
    return rms_norm_bwd_unchecked(dy, dh, h.contiguous(), rstd.contiguous(), weight, weight_grad)


def rms_norm_bwd_unchecked(dy, dh, h, rstd, weight, weight_grad):
    """rms_norm_bwd for what autograd saved and checked (h and rstd dense)."""
    K = h.shape[-1]
    rows = h.numel() // K
    dy = dy.contiguous()
    dx = torch.empty_like(h)
    dw = ws = None
    nb = 0
    if weight_grad:
        dw = h.new_empty(K, dtype=torch.float32) if weight is None else torch.empty_like(weight)
        if not rows:
            dw.zero_()
        else:
            nb = _lib.load().race_rms_norm_bwd_workspace_bytes(rows, K)
            ws = h.new_empty(nb, dtype=torch.uint8)
    if rows:
        dh = None if dh is None else dh.contiguous()
        _launch(h.device, "race_rms_norm_bwd", dy.data_ptr(), _ptr_of(dh), h.data_ptr(), rstd.data_ptr(), _dtype_code(h),
                _ptr_of(weight), _lib.RACE_F32 if weight is None else _dtype_code(weight), dx.data_ptr(), _ptr_of(dw),
                rows, K, _ptr_of(ws), nb)
    return dx, dw


def _int8_out(x, K):
    """8-bit rows [..., K] (for x [..., *]) that start at multiples of 16 bytes, as the 8-bit
    product's tile loads need, their row stride, and their scales [...]."""
    shape = x.shape
    lead = shape[:-1]
    scale = x.new_empty(lead, dtype=torch.float32)
    if K % 16 == 0:
        if K == shape[-1] and x.is_contiguous():
            return torch.empty_like(x, dtype=torch.int8), K, scale
        return x.new_empty(lead + (K,), dtype=torch.int8), K, scale
    stride = -(-K // 16) * 16
    return x.new_empty(lead + (stride,), dtype=torch.int8)[..., :K], stride, scale


def rms_norm_int8(x, residual=None, weight=None, eps=1e-5):
    """(q, scale, h): the y of rms_norm_fwd as 8-bit rows (not rounded in between), and h."""
    dev, code, xr, xs, rr, rs, rows, K, wc = _norm_inputs(x, residual, weight)
    q, qs, scale = _int8_out(x, K)
    h = x if residual is None else _dense_like(x)
    if rows:
        _launch(dev, "race_rms_norm_int8", xr.data_ptr(), xs, _ptr_of(rr), rs, code, _ptr_of(weight), wc, q.data_ptr(),
                qs, scale.data_ptr(), None if residual is None else h.data_ptr(), rows, K, eps)
    return q, scale, h


def quant_int8(x):
    """(q, scale): x [..., K] as 8-bit rows."""
    dev = _check_cuda(x)
    code = _dtype_code(x)
    xr, xs, rows, K = _rows(x, "x")
    q, qs, scale = _int8_out(x, K)
    if rows:
        _launch(dev, "race_quant_int8", xr.data_ptr(), xs, code, q.data_ptr(), qs, scale.data_ptr(), rows, K)
    return q, scale


def swiglu_int8(gate_up):
    """(q, scale): silu(gate) * up of gate_up [..., 2 F] = [gate | up] as 8-bit rows [..., F]."""
    dev = _check_cuda(gate_up)
    code = _dtype_code(gate_up)
    xr, xs, rows, K2 = _rows(gate_up, "gate_up")
    if K2 % 2:
        raise RuntimeError("gate_up must hold an even number of values per row")
    q, qs, scale = _int8_out(gate_up, K2 // 2)
    if rows:
        _launch(dev, "race_swiglu_int8", xr.data_ptr(), xs, code, q.data_ptr(), qs, scale.data_ptr(), rows, K2 // 2)
    return q, scale


def _int8_rows(q, scale, name):
    if q.dtype != torch.int8 or scale.dtype != torch.float32 or scale.shape != q.shape[:-1]:
        raise RuntimeError(f"{name} must be int8 rows [..., K] with float32 scales [...]")
    return *_rows(q, name), scale.contiguous()


def dequant_int8(q, scale, dtype=torch.bfloat16):
    """q * scale, rounded to dtype."""
    dev = _check_cuda(q, scale)
    qr, qs, rows, K, scale = _int8_rows(q, scale, "q")
    out = torch.empty_like(q, dtype=dtype, memory_format=torch.contiguous_format)
    if rows:
        _launch(dev, "race_dequant_int8", qr.data_ptr(), qs, scale.data_ptr(), out.data_ptr(), _dtype_code(out), rows, K)
    return out


def _aligned_rows(q, rows, K):
    """8-bit rows whose starts are multiples of 16 bytes, and their stride: a padded copy of q, or
    q itself where it is a single row that starts at one."""
    stride = -(-K // 16) * 16
    if rows == 1 and q.data_ptr() % 16 == 0:
        return q, stride
    p = q.new_empty((rows, stride))[:, :K]
    p.copy_(q.reshape(rows, K))
    return p, stride


def int8_linear(xq, x_scale, wq, w_scale, bias=None, dtype=torch.bfloat16):
    """(xq . wq^T) * x_scale * w_scale + bias: xq int8 [..., K], wq int8 [N, K], scales and bias
    float32 -> [..., N] of dtype.  Rows that start at multiples of 16 bytes (as the quantisers
    here lay them out) are read in place; others are copied first."""
    dev = _check_cuda(xq, x_scale, wq, w_scale, bias)
    xr, xs, M, K, x_scale = _int8_rows(xq, x_scale, "x")
    wr, ws, N, Kw, w_scale = _int8_rows(wq, w_scale, "w")
    if Kw != K or wq.dim() != 2:
        raise RuntimeError(f"w must be int8 [N, {K}]")
    if bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32 or not bias.is_contiguous()):
        raise RuntimeError(f"bias must be a contiguous float32 [{N}] tensor")
    code = _dtype_code_of(dtype)
    y = xq.new_empty((M, N) if xq.dim() == 2 else xq.shape[:-1] + (N,), dtype=dtype)
    if M and N:
        if xs % 16 or xr.data_ptr() % 16:
            xr, xs = _aligned_rows(xr, M, K)
        if ws % 16 or wr.data_ptr() % 16:
            wr, ws = _aligned_rows(wr, N, K)
        _launch(dev, "race_int8_linear", xr.data_ptr(), xs, x_scale.data_ptr(), wr.data_ptr(), ws, w_scale.data_ptr(),
                None if bias is None else bias.data_ptr(), y.data_ptr(), code, M, N, K)
    return y


def _logit_rows(logits, tokens):
    dev = _check_cuda(logits, tokens)
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
        raise RuntimeError("tokens must be int64 of the logits' shape without its last dimension")
    return dev, _dtype_code(logits), *_rows(logits, "logits"), tokens.contiguous()


def token_logprobs_fwd(logits, tokens, temperature=1.0, n_top=0, ignore_index=-100, keep_lse=True):
    """(logp, entropy, lse, top_ids, top_logp) of logits [..., V] at tokens [...]; the last two are
    [..., n_top], lse [..., 2] is for the backward (None unless keep_lse).  See race_token_logprobs_fwd in include/race_b200.h for masked and ignored rows."""
    dev, code, lr, ls, rows, V, tokens = _logit_rows(logits, tokens)
    n_top = int(n_top)
    shape = tokens.shape
    logp = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logp)
    lse = logp.new_empty(shape + (2,)) if keep_lse else None
    top_logp = logp.new_empty(shape + (max(n_top, 0),))
    top_ids = torch.empty_like(top_logp, dtype=torch.int64)
    if rows:
        _launch(dev, "race_token_logprobs_fwd", lr.data_ptr(), ls, code, tokens.data_ptr(), int(ignore_index),
                float(temperature), n_top, logp.data_ptr(), entropy.data_ptr(), _ptr_of(lse), top_ids.data_ptr(),
                top_logp.data_ptr(), rows, V)
    return logp, entropy, lse, top_ids, top_logp


def token_logprobs_bwd(logits, tokens, lse, entropy, g_logp, g_entropy, temperature=1.0, ignore_index=-100):
    """dlogits of token_logprobs_fwd for the gradients g_logp, g_entropy (None: zero)."""
    _logit_rows(logits, tokens)
    _check_cuda(logits, lse, entropy, g_logp, g_entropy)
    rows = tokens.numel()
    if lse.numel() != 2 * rows or entropy.numel() != rows or (g_logp is not None and g_logp.numel() != rows) \
            or (g_entropy is not None and g_entropy.numel() != rows):
        raise RuntimeError(f"lse must hold {2 * rows} values, entropy and the gradients {rows}")
    return token_logprobs_bwd_unchecked(logits, tokens.contiguous(), lse.float().contiguous(), entropy.float().contiguous(),
                                        g_logp, g_entropy, temperature, ignore_index)


def token_logprobs_bwd_unchecked(logits, tokens, lse, entropy, g_logp, g_entropy, temperature, ignore_index):
    """token_logprobs_bwd for what autograd saved and checked (dense but for the logits)."""
    lr, ls, rows, V = _rows(logits, "logits")
    g_logp = None if g_logp is None else g_logp.float().contiguous()
    g_entropy = None if g_entropy is None else g_entropy.float().contiguous()
    d = _dense_like(logits)
    if rows:
        _launch(logits.device, "race_token_logprobs_bwd", lr.data_ptr(), ls, _dtype_code(logits), tokens.data_ptr(),
                int(ignore_index), float(temperature), lse.data_ptr(), entropy.data_ptr(), _ptr_of(g_logp),
                _ptr_of(g_entropy), d.data_ptr(), rows, V)
    return d
