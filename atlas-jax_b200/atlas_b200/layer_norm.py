"""Layer norm with an optional fused residual add and per-group weights
(include/atlas_norm.h): ``layer_norm`` is differentiable, ``layer_norm_forward`` /
``layer_norm_backward`` are its two halves.  Every computation runs in libatlas_scan.so.

x is (..., N) with weight and bias (N,), or (..., G, N) with weight and bias (G, N), one
for each group (the heads of an attention output)."""

import ctypes

import torch

from . import _lib as L
from .scan import _WS, _ptr, _stream


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


def _group(x, weight, bias):
    """(G, N) of the parameters, checked against x."""
    if x.dtype not in (torch.float32, torch.bfloat16) or not x.is_cuda or x.dim() < 1:
        raise ValueError(f"x: expected a CUDA float32 or bfloat16 (..., N) tensor, got {x.dtype} {tuple(x.shape)} on {x.device}")
    shape = None
    for n, w in (("weight", weight), ("bias", bias)):
        if w is None:
            continue
        if shape is None:
            shape = tuple(w.shape)
            if len(shape) not in (1, 2) or x.dim() < len(shape) or tuple(x.shape[-len(shape):]) != shape:
                raise ValueError(f"{n}: {shape} are not the last one or two axes of x {tuple(x.shape)}")
        if w.dtype != torch.float32 or tuple(w.shape) != shape or not w.is_contiguous() or w.device != x.device:
            raise ValueError(f"{n}: expected contiguous float32 {shape} on {x.device}, got {w.dtype} {tuple(w.shape)} on {w.device}")
    return (1, x.shape[-1]) if shape is None or len(shape) == 1 else shape


def _params(x, G, N, eps):
    rows = x.numel() // (G * N) if G * N else 0
    return AtlasNormParams(L.ATLAS_ABI_VERSION, L.ATLAS_BF16 if x.dtype == torch.bfloat16 else L.ATLAS_F32, rows, G, N,
                           eps, 0)


def _like(x, ref, name):
    if x.dtype != ref.dtype or x.shape != ref.shape or x.device != ref.device:
        raise ValueError(f"{name}: expected {ref.dtype} {tuple(ref.shape)} on {ref.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.contiguous()


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Returns (y, h, stats): h = x + residual (x itself without a residual), y its layer
    norm, stats (vectors, 2) float32 the means and reciprocal deviations of h."""
    lib = _lib()
    G, N = _group(x, weight, bias)
    x = x.contiguous()
    residual = None if residual is None else _like(residual, x, "residual")
    with torch.cuda.device(x.device):
        p = _params(x, G, N, eps)
        y = torch.empty_like(x)
        h = x if residual is None else torch.empty_like(x)
        stats = torch.empty(p.rows * G, 2, device=x.device)
        L.check(lib.atlas_layernorm_fwd(ctypes.byref(p), _ptr(x), _ptr(residual), _ptr(weight), _ptr(bias), _ptr(y),
                                        None if residual is None else _ptr(h), _ptr(stats), _stream(x.device)))
    return y, h, stats


def layer_norm_backward(dy, h, weight, stats, dh=None, need_params=True, shape=None, workspace=None):
    """VJP of ``layer_norm_forward``: (dx, dweight, dbias).  dx is the cotangent of x and of
    residual; dh the cotangent of h (None: zeros); the parameter gradients have the shape
    of ``weight`` (or ``shape``, for a norm with a bias alone) and are None with
    need_params=False."""
    lib = _lib()
    G, N = _group(h, weight, None)
    shape = tuple(weight.shape) if weight is not None else (h.shape[-1],) if shape is None else tuple(shape)
    if weight is None and len(shape) == 2:
        G = shape[0]
    h = h.contiguous()
    dy = _like(dy, h, "dy")
    dh = None if dh is None else _like(dh, h, "dh")
    dev = h.device
    with torch.cuda.device(dev):
        p = _params(h, G, N, 0.0)
        if stats.dtype != torch.float32 or tuple(stats.shape) != (p.rows * G, 2) or not stats.is_contiguous() \
                or stats.device != dev:
            raise ValueError(f"stats: expected contiguous float32 {(p.rows * G, 2)} on {dev}, got {stats.dtype} {tuple(stats.shape)}")
        dx = torch.empty_like(h)
        dw, db = (torch.empty(shape, device=dev), torch.empty(shape, device=dev)) if need_params else (None, None)
        ws, wsb = (workspace or _WS).get(lib.atlas_layernorm_workspace_bytes(ctypes.byref(p)), dev)
        L.check(lib.atlas_layernorm_bwd(ctypes.byref(p), _ptr(dy), _ptr(h), _ptr(weight), _ptr(stats), _ptr(dh), _ptr(dx),
                                        _ptr(dw), _ptr(db), _ptr(ws), wsb, _stream(dev)))
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
    def backward(ctx, dy, dh=None):
        h, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = torch.zeros_like(h) if dy is None else dy.to(h.dtype)
        dx, dw, db = layer_norm_backward(dy, h, weight, stats, None if dh is None else dh.to(h.dtype), need[1] or need[2],
                                         ctx.shape)
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, \
            dx if ctx.has_residual and need[4] else None


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Differentiable layer norm of x, or with ``residual`` (y, h) of h = x + residual."""
    return LayerNorm.apply(x, weight, bias, eps, residual)
