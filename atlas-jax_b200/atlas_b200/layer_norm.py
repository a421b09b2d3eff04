"""Layer norm with an optional fused residual add and per-group weights
(include/atlas_norm.h): ``layer_norm`` is differentiable, ``layer_norm_forward`` /
``layer_norm_backward`` are its two halves.  Every computation runs in libatlas_scan.so.

x is (..., N) with weight and bias (N,), or (..., G, N) with weight and bias (G, N), one
for each group (the heads of an attention output)."""

import ctypes
import functools

import torch

from . import _lib as L
from .scan import _WS, addr, away, first_derivatives, stream_of


class AtlasNormParams(ctypes.Structure):
    _fields_ = [("abi_version", ctypes.c_int32), ("act_dtype", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("G", ctypes.c_int32), ("N", ctypes.c_int32), ("eps", ctypes.c_float), ("reserved", ctypes.c_int32)]


_P = ctypes.c_void_p
_bound = False


def _lib():
    global _bound
    lib = L.load()
    if not _bound:
        pp = ctypes.POINTER(AtlasNormParams)
        lib.atlas_layernorm_workspace_bytes.restype = ctypes.c_size_t
        lib.atlas_layernorm_workspace_bytes.argtypes = [pp]
        lib.atlas_layernorm_fwd.restype = ctypes.c_int
        lib.atlas_layernorm_fwd.argtypes = [pp] + [_P] * 8
        lib.atlas_layernorm_bwd.restype = ctypes.c_int
        lib.atlas_layernorm_bwd.argtypes = [pp] + [_P] * 9 + [ctypes.c_size_t, _P]
        _bound = True
    return lib


class _Plan:
    """What a call needs that depends on shapes and types alone.  x: (shape, type, device);
    params: the same with contiguity for weight and bias, or None."""

    def __init__(self, x, weight, bias, eps):
        shape, dtype, dev = x
        if dtype not in (torch.float32, torch.bfloat16) or dev < 0 or len(shape) < 1:
            raise ValueError(f"x: expected a CUDA float32 or bfloat16 (..., N) tensor, got {dtype} {tuple(shape)}")
        p = None
        for n, w in (("weight", weight), ("bias", bias)):
            if w is None:
                continue
            if p is None:
                p = tuple(w[0])
                if len(p) not in (1, 2) or len(shape) < len(p) or tuple(shape[-len(p):]) != p:
                    raise ValueError(f"{n}: {p} are not the last one or two axes of x {tuple(shape)}")
            if w[1] != torch.float32 or tuple(w[0]) != p or w[2] != dev or not w[3]:
                raise ValueError(f"{n}: expected contiguous float32 {p} on the device of x, got {w[1]} {tuple(w[0])}")
        self.param_shape = p or (shape[-1],)
        G, N = (1, shape[-1]) if len(self.param_shape) == 1 else self.param_shape
        if G >= 1 << 31 or N >= 1 << 31:  # (a c_int32 field would keep the lower half)
            raise L.AtlasError(L.ATLAS_ERR_UNSUPPORTED, f"layer norm: G * N must be at most 2^20, got {G} * {N}")
        rows = shape.numel() // (G * N) if G * N else 0
        self.params = AtlasNormParams(L.ATLAS_ABI_VERSION, L.ATLAS_BF16 if dtype == torch.bfloat16 else L.ATLAS_F32,
                                      rows, G, N, eps, 0)
        self.lib, self.ref, self.vecs = _lib(), ctypes.byref(self.params), rows * G
        self.workspace_bytes = self.lib.atlas_layernorm_workspace_bytes(self.ref)
        if self.workspace_bytes == 0:
            raise L.AtlasError(L.ATLAS_ERR_INVALID_ARGUMENT, L.load().atlas_last_error_string().decode())


_plans = functools.lru_cache(maxsize=512)(_Plan)


def _key(w):
    return None if w is None else (w.shape, w.dtype, w.get_device(), w.is_contiguous())


def _plan(x, weight, bias, eps):
    return _plans((x.shape, x.dtype, x.get_device()), _key(weight), _key(bias), float(eps))  # (a tensor: its value)


def _like(x, ref, name):
    if x.dtype != ref.dtype or x.shape != ref.shape or x.get_device() != ref.get_device():
        raise ValueError(f"{name}: expected {ref.dtype} {tuple(ref.shape)} on {ref.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.contiguous()


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Returns (y, h, stats): h = x + residual (x itself without a residual), y its layer
    norm, stats (vectors, 2) float32 what the backward needs of the statistics of h."""
    p = _plan(x, weight, bias, eps)
    x = x.contiguous()
    dev = x.device
    if away(dev):
        with torch.cuda.device(dev):
            return layer_norm_forward(x, weight, bias, eps, residual)
    y, stats = torch.empty_like(x), torch.empty(p.vecs, 2, dtype=torch.float32, device=dev)
    h, hp = x, None
    if residual is not None:
        residual, h = _like(residual, x, "residual"), torch.empty_like(x)
        hp = h.data_ptr()
    rc = p.lib.atlas_layernorm_fwd(p.ref, x.data_ptr(), addr(residual), addr(weight), addr(bias), y.data_ptr(), hp,
                                   stats.data_ptr(), stream_of(dev))
    if rc:
        L.check(rc)
    return y, h, stats


def layer_norm_backward(dy, h, weight, stats, dh=None, need_params=True, shape=None, workspace=None):
    """VJP of ``layer_norm_forward``: (dx, dweight, dbias).  dx is the cotangent of x and of
    residual; dh the cotangent of h (None: zeros); the parameter gradients have the shape
    of ``weight`` (or ``shape``, for a norm with a bias alone) and are None with
    need_params=False."""
    if weight is None and shape is not None:  # a plan for parameters of that shape
        p = _plans((h.shape, h.dtype, h.get_device()), (tuple(shape), torch.float32, h.get_device(), True), None, 0.0)
    else:
        p = _plan(h, weight, None, 0.0)
    h = h.contiguous()
    dy = _like(dy, h, "dy")
    if dh is not None:
        dh = _like(dh, h, "dh")
    dev = h.device
    if stats.dtype != torch.float32 or stats.shape != (p.vecs, 2) or not stats.is_contiguous() \
            or stats.get_device() != h.get_device():
        raise ValueError(f"stats: expected contiguous float32 {(p.vecs, 2)} on {dev}, got {stats.dtype} {tuple(stats.shape)}")
    if away(dev):
        with torch.cuda.device(dev):
            return layer_norm_backward(dy, h, weight, stats, dh, need_params, shape, workspace)
    dx = torch.empty_like(h)
    dw = db = ws = None
    wsb = 0
    if need_params:
        dw = torch.empty(*p.param_shape, dtype=torch.float32, device=dev) if weight is None else torch.empty_like(weight)
        db = torch.empty_like(dw)
        ws, wsb = (workspace or _WS).get(p.workspace_bytes, dev)
    rc = p.lib.atlas_layernorm_bwd(p.ref, dy.data_ptr(), h.data_ptr(), addr(weight), stats.data_ptr(), addr(dh),
                                   dx.data_ptr(), addr(dw), addr(db), addr(ws), wsb, stream_of(dev))
    if rc:
        L.check(rc)
    return dx, dw, db


class LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        y, h, stats = layer_norm_forward(x, weight, bias, eps, residual)
        ctx.save_for_backward(h, weight, stats)
        ctx.has_residual, ctx.shape = residual is not None, None if bias is None else tuple(bias.shape)
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @first_derivatives
    def backward(ctx, dy, dh=None):
        h, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = torch.zeros_like(h) if dy is None else dy.to(h.dtype)
        dx, dw, db = layer_norm_backward(dy, h, weight, stats, None if dh is None else dh.to(h.dtype), need[1] or need[2],
                                         ctx.shape)
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, \
            dx if ctx.has_residual and need[4] else None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Differentiable layer norm of x, or with ``residual`` (y, h) of h = x + residual.  First
    derivatives only: differentiating a gradient again raises."""
    return LayerNorm.apply(x, weight, bias, eps, residual)
