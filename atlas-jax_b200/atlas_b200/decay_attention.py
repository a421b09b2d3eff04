"""Decay attention (include/atlas_decay.h): causal linear attention whose state decays by
a factor of its own in each head,

    S_t = exp(log_decay_h) S_{t-1} + k_t v_t^T,    y_t = scale * q_t^T S_t.

``decay_attention`` is the differentiable whole-sequence form, ``decay_attention_forward`` /
``decay_attention_backward`` are its two halves, and ``decay_attention_step`` advances
states by one or a few tokens (generation).  Every computation runs in libatlas_scan.so.
"""

import ctypes

import torch

from . import _lib as L
from .scan import _WS, _ptr, _stream


class AtlasDecayParams(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("abi_version", "B", "T", "H", "D", "act_dtype")] +
                [("scale", ctypes.c_float), ("reserved", ctypes.c_int32)] +
                [(n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride")])


_P = ctypes.c_void_p
_bound = False


def _lib():
    global _bound
    lib = L.load()
    if not _bound:
        pp = ctypes.POINTER(AtlasDecayParams)
        for n in ("atlas_decay_saved_bytes", "atlas_decay_workspace_bytes"):
            getattr(lib, n).restype = ctypes.c_size_t
            getattr(lib, n).argtypes = [pp]
        lib.atlas_decay_fwd.restype = ctypes.c_int
        lib.atlas_decay_fwd.argtypes = [pp] + [_P] * 9 + [ctypes.c_size_t, _P]
        lib.atlas_decay_bwd.restype = ctypes.c_int
        lib.atlas_decay_bwd.argtypes = [pp] + [_P] * 13 + [ctypes.c_size_t, _P]
        lib.atlas_decay_step.restype = ctypes.c_int
        lib.atlas_decay_step.argtypes = [pp] + [_P] * 6 + [ctypes.c_int32] + [_P] * 3
        _bound = True
    return lib


def _check(q, k, v, log_decay):
    """Shapes, types and devices; returns q, k, v with contiguous channels."""
    if q.dim() != 4:
        raise ValueError(f"q: expected (B, T, H, D), got {tuple(q.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"q: expected float32 or bfloat16, got {q.dtype}")
    for n, x in (("q", q), ("k", k), ("v", v)):
        if x.dtype != q.dtype or x.shape != q.shape or not x.is_cuda or x.device != q.device:
            raise ValueError(f"{n}: expected CUDA {q.dtype} {tuple(q.shape)}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    _need(log_decay, (q.shape[2],), "log_decay", q.device)
    return [x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous() for x in (q, k, v)]


def _need(x, shape, name, device):
    if x.dtype != torch.float32 or tuple(x.shape) != tuple(shape) or not x.is_contiguous() or x.device != device:
        raise ValueError(f"{name}: expected contiguous CUDA float32 {tuple(shape)}, got {x.dtype} {tuple(x.shape)} on {x.device}")


def _params(q, k, v, scale):
    B, T, H, D = q.shape
    s = [(ctypes.c_int64 * 3)(*x.stride()[:3]) for x in (q, k, v)]
    return AtlasDecayParams(L.ATLAS_ABI_VERSION, B, T, H, D, L.ATLAS_BF16 if q.dtype == torch.bfloat16 else L.ATLAS_F32,
                            D ** -0.5 if scale is None else scale, 0, *s)


def _size(n):
    """A size query's answer; 0 is an error only when it left a message."""
    if n == 0 and L.load().atlas_last_error_string():
        raise L.AtlasError(L.ATLAS_ERR_INVALID_ARGUMENT, L.load().atlas_last_error_string().decode())
    return n


def decay_attention_forward(q, k, v, log_decay, state=None, scale=None, need_saved=True, workspace=None):
    """q, k, v: (B, T, H, D) float32 or bf16, any strides with contiguous channels; log_decay
    (H,) float32; state (B, H, D, D) float32 or None (zeros); scale defaults to D^-0.5.
    Returns (y, state after the last token, saved for the backward or None)."""
    lib = _lib()
    q, k, v = _check(q, k, v, log_decay)
    B, T, H, D = q.shape
    dev = q.device
    if state is not None:
        _need(state, (B, H, D, D), "state", dev)
    with torch.cuda.device(dev):
        p = _params(q, k, v, scale)
        y = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
        out = torch.empty(B, H, D, D, device=dev)
        nbytes = _size(lib.atlas_decay_saved_bytes(ctypes.byref(p)))
        saved = torch.empty(nbytes, dtype=torch.uint8, device=dev) if need_saved else None
        ws, wsb = (None, 0) if need_saved else (workspace or _WS).get(nbytes, dev)
        L.check(lib.atlas_decay_fwd(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _ptr(state), _ptr(y),
                                    _ptr(out), _ptr(saved), _ptr(ws), wsb, _stream(dev)))
    return y, out, saved


def decay_attention_backward(q, k, v, log_decay, saved, dy, dstate=None, scale=None, workspace=None):
    """VJP of ``decay_attention_forward``: (dq, dk, dv, dlog_decay, dstate_in)."""
    lib = _lib()
    q, k, v = _check(q, k, v, log_decay)
    B, T, H, D = q.shape
    dev = q.device
    if dy.dtype != q.dtype or dy.shape != q.shape or dy.device != dev:
        raise ValueError(f"dy: expected CUDA {q.dtype} {tuple(q.shape)}, got {dy.dtype} {tuple(dy.shape)} on {dy.device}")
    dy = dy.contiguous()
    if dstate is not None:
        _need(dstate, (B, H, D, D), "dstate", dev)
    with torch.cuda.device(dev):
        p = _params(q, k, v, scale)
        if saved.numel() * saved.element_size() < _size(lib.atlas_decay_saved_bytes(ctypes.byref(p))):
            raise ValueError("saved: not what decay_attention_forward saved for these inputs")
        dq, dk, dv = (torch.empty(B, T, H, D, dtype=q.dtype, device=dev) for _ in range(3))
        dg, dstate_in = torch.empty(H, device=dev), torch.empty(B, H, D, D, device=dev)
        ws, wsb = (workspace or _WS).get(_size(lib.atlas_decay_workspace_bytes(ctypes.byref(p))), dev)
        L.check(lib.atlas_decay_bwd(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _ptr(saved), _ptr(dy),
                                    _ptr(dstate), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dg), _ptr(dstate_in), _ptr(ws), wsb,
                                    _stream(dev)))
    return dq, dk, dv, dg, dstate_in


def decay_attention_step(q, k, v, log_decay, state, slots=None, scale=None, out=None):
    """The recurrent form, for the tokens of one generation step.

    q, k, v: (B, T, H, D), T usually 1; state: (B, H, D, D) float32, or with ``slots`` (B,)
    int32 a pool (n, H, D, D) in which sequence b uses row slots[b] (every running
    sequence a row of its own; a slot outside the pool marks an idle sequence, whose y is
    0).  The new states are written to ``out`` (a buffer like ``state``; default: in place).
    Returns (y, out)."""
    lib = _lib()
    q, k, v = _check(q, k, v, log_decay)
    B, T, H, D = q.shape
    dev = q.device
    n = B if slots is None else state.shape[0]
    _need(state, (n, H, D, D), "state", dev)
    out = state if out is None else out
    _need(out, (n, H, D, D), "out", dev)
    if slots is not None and (slots.dtype != torch.int32 or tuple(slots.shape) != (B,) or not slots.is_contiguous()
                              or slots.device != dev):
        raise ValueError(f"slots: expected contiguous CUDA int32 ({B},), got {slots.dtype} {tuple(slots.shape)} on {slots.device}")
    with torch.cuda.device(dev):
        p = _params(q, k, v, scale)
        y = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
        L.check(lib.atlas_decay_step(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _ptr(state), _ptr(slots),
                                     n, _ptr(y), _ptr(out), _stream(dev)))
    return y, out


class DecayAttention(torch.autograd.Function):
    """Autograd pairing of the forward and backward kernels."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, scale):
        need = any(ctx.needs_input_grad[:5])
        y, out, saved = decay_attention_forward(q, k, v, log_decay, state, scale, need_saved=need)
        ctx.scale, ctx.has_state = scale, state is not None
        if need:
            ctx.save_for_backward(q, k, v, log_decay, saved)
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    def backward(ctx, dy, dstate):
        q, k, v, log_decay, saved = ctx.saved_tensors
        dy = torch.zeros_like(q) if dy is None else dy.to(q.dtype)
        dstate = None if dstate is None else dstate.float().contiguous()
        dq, dk, dv, dg, dstate_in = decay_attention_backward(q, k, v, log_decay, saved, dy, dstate, ctx.scale)
        return dq, dk, dv, dg, dstate_in if ctx.has_state else None, None


def decay_attention(q, k, v, log_decay, state=None, scale=None):
    """Differentiable decay attention: returns (y, state after the last token)."""
    return DecayAttention.apply(q, k, v, log_decay, state, scale)
