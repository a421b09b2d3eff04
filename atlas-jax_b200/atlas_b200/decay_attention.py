"""Decay attention (include/atlas_decay.h): causal linear attention whose state decays by
a factor of its own in each head,

    S_t = exp(log_decay_h) S_{t-1} + k_t v_t^T,    y_t = scale * q_t^T S_t.

``decay_attention`` is the differentiable whole-sequence form, ``decay_attention_forward`` /
``decay_attention_backward`` are its two halves, and ``decay_attention_step`` advances
states by one or a few tokens (generation).  Every computation runs in libatlas_scan.so.
"""

import ctypes
import functools

import torch
from torch.autograd.graph import increment_version

from . import _lib as L
from .scan import _WS, addr, away, empty_like, first_derivatives, stream_of


class AtlasDecayParams(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("abi_version", "B", "T", "H", "D", "act_dtype")] +
                [("scale", ctypes.c_float), ("aligned16", ctypes.c_int32)] +
                [(n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride")])


_P = ctypes.c_void_p
_bound = False


def _lib():
    global _bound
    lib = L.load()
    if not _bound:
        pp = ctypes.POINTER(AtlasDecayParams)
        for n in ("atlas_decay_saved_bytes", "atlas_decay_fwd_workspace_bytes",
                  "atlas_decay_saved_workspace_bytes", "atlas_decay_bwd_workspace_bytes"):
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


class _Plan:
    """What a call needs that depends on shapes, strides and types alone."""

    def __init__(self, q, k, v, g, scale, aligned):
        (shape, st, dtype, dev) = q
        if len(shape) != 4:
            raise ValueError(f"q: expected (B, T, H, D), got {tuple(shape)}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"q: expected float32 or bfloat16, got {dtype}")
        for n, x in (("q", q), ("k", k), ("v", v)):
            if x[0] != shape or x[2] != dtype or x[3] != dev or dev < 0:
                raise ValueError(f"{n}: expected CUDA {dtype} {tuple(shape)} on the device of q, got {x[2]} {tuple(x[0])}")
        B, T, H, D = shape
        if max(shape) >= 1 << 31:  # (a c_int32 field would keep the lower half)
            raise L.AtlasError(L.ATLAS_ERR_UNSUPPORTED, f"decay attention: sizes must be below 2^31, got {tuple(shape)}")
        if g[0] != (H,) or g[2] != torch.float32 or g[3] != dev or (g[1] != (1,) and H > 1):
            raise ValueError(f"log_decay: expected contiguous CUDA float32 {(H,)}, got {g[2]} {tuple(g[0])}")
        # contiguous channels; bf16 on the tensor cores also has no broadcast (stride 0) axes.  Strides of
        # empty tensors say nothing, and contiguous() keeps them.
        fast = dtype == torch.bfloat16 and D % 8 == 0
        self.packed = 0 in shape or all(
            (x[1][3] == 1 or D == 1) and not (fast and any(s == 0 and n > 1 for s, n in zip(x[1], shape))) for x in (q, k, v))
        strides = [(ctypes.c_int64 * 3)(*x[1][:3]) for x in (q, k, v)]
        self.params = AtlasDecayParams(L.ATLAS_ABI_VERSION, B, T, H, D,
                                       L.ATLAS_BF16 if dtype == torch.bfloat16 else L.ATLAS_F32,
                                       max(D, 1) ** -0.5 if scale is None else scale, int(aligned), *strides)
        self.lib, self.ref = _lib(), ctypes.byref(self.params)
        self.shape, self.dtype = tuple(shape), dtype
        self.B, self.state_shape = B, (B, H, D, D)
        self.saved_bytes = self._size(self.lib.atlas_decay_saved_bytes)
        self.fwd_workspace_bytes = self._size(self.lib.atlas_decay_fwd_workspace_bytes)
        self.saved_workspace_bytes = self._size(self.lib.atlas_decay_saved_workspace_bytes)
        self.bwd_workspace_bytes = self._size(self.lib.atlas_decay_bwd_workspace_bytes)

    def _size(self, query):
        """A size query's answer; 0 is an error only when it left a message."""
        n = query(self.ref)
        if n == 0 and L.load().atlas_last_error_string():
            raise L.AtlasError(L.ATLAS_ERR_INVALID_ARGUMENT, L.load().atlas_last_error_string().decode())
        return n


_plans = functools.lru_cache(maxsize=512)(_Plan)


def _plan(q, k, v, log_decay, scale):
    """Checks the inputs; returns their plan and q, k, v with contiguous channels."""
    scale = None if scale is None else float(scale)  # (a tensor would be a key by its identity)
    aligned = (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 == 0
    p = _plans(*[(x.shape, x.stride(), x.dtype, x.get_device()) for x in (q, k, v, log_decay)], scale, aligned)
    if not p.packed:
        return _plan(q.contiguous(), k.contiguous(), v.contiguous(), log_decay, scale)
    return p, q, k, v


def _aligned(x):
    """x, or a copy of it where it starts off the 16-byte grid."""
    return x if x is None or x.data_ptr() & 15 == 0 else x.clone()


def _need(x, shape, name, q):
    if x.dtype != torch.float32 or x.shape != shape or not x.is_contiguous() or x.get_device() != q.get_device():
        raise ValueError(f"{name}: expected contiguous float32 {tuple(shape)} on {q.device}, "
                         f"got {x.dtype} {tuple(x.shape)} on {x.device}")


def decay_attention_forward(q, k, v, log_decay, state=None, scale=None, need_saved=True, workspace=None):
    """q, k, v: (B, T, H, D) float32 or bf16, any strides with contiguous channels; log_decay
    (H,) float32; state (B, H, D, D) float32 or None (zeros); scale defaults to D^-0.5.
    Returns (y, state after the last token, saved for the backward or None)."""
    p, q, k, v = _plan(q, k, v, log_decay, scale)
    dev = q.device
    if state is not None:
        _need(state, p.state_shape, "state", q)
        state = _aligned(state)
    if away(dev):
        with torch.cuda.device(dev):
            return decay_attention_forward(q, k, v, log_decay, state, scale, need_saved, workspace)
    y = empty_like(q)
    out = torch.empty(*p.state_shape, dtype=torch.float32, device=dev) if state is None else torch.empty_like(state)
    saved, need = None, p.fwd_workspace_bytes
    if need_saved:
        saved, need = torch.empty(p.saved_bytes // 4, dtype=torch.float32, device=dev), p.saved_workspace_bytes
    ws, wsb = (workspace or _WS).get(need, dev)
    rc = p.lib.atlas_decay_fwd(p.ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), addr(state),
                               y.data_ptr(), out.data_ptr(), addr(saved), addr(ws), wsb, stream_of(dev))
    if rc:
        L.check(rc)
    return y, out, saved


def decay_attention_backward(q, k, v, log_decay, saved, dy, dstate=None, scale=None, workspace=None):
    """VJP of ``decay_attention_forward``: (dq, dk, dv, dlog_decay, dstate_in)."""
    p, q, k, v = _plan(q, k, v, log_decay, scale)
    dev = q.device
    if dy.dtype != p.dtype or dy.shape != p.shape or dy.get_device() != q.get_device():
        raise ValueError(f"dy: expected {p.dtype} {p.shape} on {dev}, got {dy.dtype} {tuple(dy.shape)} on {dy.device}")
    dy = _aligned(dy.contiguous())
    if dstate is not None:
        _need(dstate, p.state_shape, "dstate", q)
        dstate = _aligned(dstate)
    if saved.numel() * saved.element_size() != p.saved_bytes or not saved.is_contiguous() \
            or saved.get_device() != q.get_device():
        raise ValueError("saved: not what decay_attention_forward saved for these inputs")
    if away(dev):
        with torch.cuda.device(dev):
            return decay_attention_backward(q, k, v, log_decay, saved, dy, dstate, scale, workspace)
    dq, dk, dv = empty_like(q), empty_like(q), empty_like(q)
    dg, dstate_in = torch.empty_like(log_decay), torch.empty(*p.state_shape, dtype=torch.float32, device=dev)
    ws, wsb = (workspace or _WS).get(p.bwd_workspace_bytes, dev)
    rc = p.lib.atlas_decay_bwd(p.ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), saved.data_ptr(),
                               dy.data_ptr(), addr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
                               dstate_in.data_ptr(), addr(ws), wsb, stream_of(dev))
    if rc:
        L.check(rc)
    return dq, dk, dv, dg, dstate_in


def decay_attention_step(q, k, v, log_decay, state, slots=None, scale=None, out=None):
    """The recurrent form, for the tokens of one generation step.

    q, k, v: (B, T, H, D), T usually 1; state: (B, H, D, D) float32, or with ``slots`` (B,)
    int32 a pool (n, H, D, D) in which sequence b uses row slots[b] (every running
    sequence a row of its own; a slot outside the pool marks an idle sequence, whose y is
    0).  The new states are written to ``out`` (a buffer like ``state``; default: in place).
    There is no backward: inputs that require gradients are for torch.no_grad().
    Returns (y, out)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad or (out is not None and out.requires_grad)):
        raise ValueError("decay_attention_step has no backward: call it under torch.no_grad(), or use decay_attention")
    p, q, k, v = _plan(q, k, v, log_decay, scale)
    dev = q.device
    n = p.B if slots is None else state.shape[0]
    if n >= 1 << 31:
        raise ValueError(f"state: expected fewer than 2^31 rows, got {n}")
    shape = p.state_shape if n == p.B else (n,) + p.state_shape[1:]
    _need(state, shape, "state", q)
    if out is None:
        out = state
    else:
        _need(out, shape, "out", q)
    if slots is not None and (slots.dtype != torch.int32 or slots.shape != (p.B,) or not slots.is_contiguous()
                              or slots.get_device() != q.get_device()):
        raise ValueError(f"slots: expected contiguous int32 ({p.B},) on {dev}, got {slots.dtype} {tuple(slots.shape)} on {slots.device}")
    if away(dev):
        with torch.cuda.device(dev):
            return decay_attention_step(q, k, v, log_decay, state, slots, scale, out)
    y = empty_like(q)
    rc = p.lib.atlas_decay_step(p.ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), state.data_ptr(),
                                addr(slots), n, y.data_ptr(), out.data_ptr(), stream_of(dev))
    if rc:
        L.check(rc)
    increment_version(out)  # written behind autograd's back
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
    @first_derivatives
    def backward(ctx, dy, dstate):
        q, k, v, log_decay, saved = ctx.saved_tensors
        dy = torch.zeros_like(q) if dy is None else dy.to(q.dtype)
        dstate = None if dstate is None else dstate.float().contiguous()
        dq, dk, dv, dg, dstate_in = decay_attention_backward(q, k, v, log_decay, saved, dy, dstate, ctx.scale)
        return dq, dk, dv, dg, dstate_in if ctx.has_state else None, None


def decay_attention(q, k, v, log_decay, state=None, scale=None):
    """Differentiable decay attention: returns (y, state after the last token).  First
    derivatives only: differentiating a gradient again raises."""
    return DecayAttention.apply(q, k, v, log_decay, state, scale)
