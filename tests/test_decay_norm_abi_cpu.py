"""CPU checks of the decay attention and layer norm entry points: sizes, and refusals that
come before any device work."""
import ctypes
import os
import re

from atlas_b200 import _lib as L


def _decay(**kw):
    from atlas_b200.decay_attention import AtlasDecayParams
    b = dict(abi=L.ATLAS_ABI_VERSION, B=2, T=300, H=3, D=64, dt=L.ATLAS_BF16, scale=0.125, aligned=1, stride=(300 * 192, 192, 64))
    b.update(kw)
    s = [(ctypes.c_int64 * 3)(*b["stride"]) for _ in range(3)]
    return AtlasDecayParams(b["abi"], b["B"], b["T"], b["H"], b["D"], b["dt"], b["scale"], b["aligned"], *s)


def _norm(**kw):
    from atlas_b200.layer_norm import AtlasNormParams
    b = dict(abi=L.ATLAS_ABI_VERSION, dt=L.ATLAS_BF16, rows=100, G=1, N=768, eps=1e-5)
    b.update(kw)
    return AtlasNormParams(b["abi"], b["dt"], b["rows"], b["G"], b["N"], b["eps"], 0)


def test_prototypes_match_the_headers():
    from atlas_b200 import decay_attention, layer_norm
    inc = os.path.dirname(L.HEADER)
    for header, lib in (("atlas_decay.h", decay_attention._lib()), ("atlas_norm.h", layer_norm._lib())):
        txt = open(os.path.join(inc, header)).read()
        decls = re.findall(r"^(?:int|size_t) (atlas_\w+)\(([^;]*)\);", txt, re.M)
        assert len(decls) >= 3
        for name, args in decls:
            assert len(getattr(lib, name).argtypes) == args.count(",") + 1, name


def test_decay_sizes():
    from atlas_b200.decay_attention import _lib
    lib = _lib()
    p = _decay()
    # the state entering each of ceil(300 / 64) chunks
    assert lib.atlas_decay_saved_bytes(ctypes.byref(p)) == 2 * 3 * 5 * 64 * 64 * 4
    assert lib.atlas_decay_bwd_workspace_bytes(ctypes.byref(p)) >= 2 * 3 * 5 * 64 * 64 * 4
    # without 16-byte alignment the forward keeps every chunk's state
    assert lib.atlas_decay_fwd_workspace_bytes(ctypes.byref(_decay(aligned=0))) == 2 * 3 * 5 * 64 * 64 * 4
    assert lib.atlas_decay_saved_bytes(ctypes.byref(_decay(T=0))) == 0 and lib.atlas_last_error_string() == b""


def test_decay_refusals():
    from atlas_b200.decay_attention import _lib
    lib = _lib()
    for kw, code, word in ((dict(abi=9), L.ATLAS_ERR_INVALID_ARGUMENT, b"abi"), (dict(B=-1), L.ATLAS_ERR_INVALID_ARGUMENT, b"B, T"),
                           (dict(D=0), L.ATLAS_ERR_INVALID_ARGUMENT, b"positive"), (dict(D=129), L.ATLAS_ERR_UNSUPPORTED, b"128"),
                           (dict(dt=7), L.ATLAS_ERR_INVALID_ARGUMENT, b"act_dtype"),
                           (dict(scale=float("inf")), L.ATLAS_ERR_INVALID_ARGUMENT, b"scale"),
                           (dict(stride=(1, -1, 1)), L.ATLAS_ERR_INVALID_ARGUMENT, b"strides"),
                           (dict(T=(1 << 30) + 1), L.ATLAS_ERR_UNSUPPORTED, b"2^30"),
                           (dict(B=1 << 20, H=1 << 10), L.ATLAS_ERR_UNSUPPORTED, b"too large")):
        p = _decay(**kw)
        assert lib.atlas_decay_saved_bytes(ctypes.byref(p)) == 0
        for rc in (lib.atlas_decay_fwd(ctypes.byref(p), *[None] * 9, 0, None),
                   lib.atlas_decay_bwd(ctypes.byref(p), *[None] * 13, 0, None),
                   lib.atlas_decay_step(ctypes.byref(p), *[None] * 6, 0, *[None] * 3)):
            assert rc == code and word in lib.atlas_last_error_string(), kw
    p = _decay()
    x = ctypes.c_void_p(16)
    assert lib.atlas_decay_fwd(ctypes.byref(p), *[None] * 9, 0, None) == L.ATLAS_ERR_INVALID_ARGUMENT
    assert lib.atlas_decay_fwd(ctypes.byref(_decay(aligned=0)), *[x] * 7, None, x, 16, None) == L.ATLAS_ERR_WORKSPACE
    odd = ctypes.c_void_p(20)
    assert lib.atlas_decay_fwd(ctypes.byref(p), x, odd, *[x] * 5, x, None, 0, None) == L.ATLAS_ERR_INVALID_ARGUMENT
    assert b"aligned" in lib.atlas_last_error_string()
    assert lib.atlas_decay_bwd(ctypes.byref(p), *[x] * 13, 16, None) == L.ATLAS_ERR_WORKSPACE
    assert lib.atlas_decay_step(ctypes.byref(p), *[x] * 6, -1, x, x, None) == L.ATLAS_ERR_INVALID_ARGUMENT
    assert lib.atlas_decay_fwd(None, *[None] * 9, 0, None) == L.ATLAS_ERR_INVALID_ARGUMENT


def test_norm_sizes_and_refusals():
    from atlas_b200.layer_norm import _lib
    lib = _lib()
    assert lib.atlas_layernorm_workspace_bytes(ctypes.byref(_norm())) >= 2 * 768 * 4
    for kw, code, word in ((dict(abi=9), L.ATLAS_ERR_INVALID_ARGUMENT, b"abi"), (dict(rows=-1), L.ATLAS_ERR_INVALID_ARGUMENT, b"rows"),
                           (dict(N=0), L.ATLAS_ERR_INVALID_ARGUMENT, b"positive"), (dict(dt=2), L.ATLAS_ERR_INVALID_ARGUMENT, b"act"),
                           (dict(N=(1 << 20) + 1), L.ATLAS_ERR_UNSUPPORTED, b"2^20"), (dict(G=1 << 11, N=1 << 10), L.ATLAS_ERR_UNSUPPORTED, b"2^20"),
                           (dict(rows=1 << 60), L.ATLAS_ERR_UNSUPPORTED, b"2^50"), (dict(eps=-1.0), L.ATLAS_ERR_INVALID_ARGUMENT, b"eps"),
                           (dict(eps=float("nan")), L.ATLAS_ERR_INVALID_ARGUMENT, b"eps")):
        p = _norm(**kw)
        assert lib.atlas_layernorm_workspace_bytes(ctypes.byref(p)) == 0
        for rc in (lib.atlas_layernorm_fwd(ctypes.byref(p), *[None] * 8), lib.atlas_layernorm_bwd(ctypes.byref(p), *[None] * 9, 0, None)):
            assert rc == code and word in lib.atlas_last_error_string(), kw
    p = _norm()
    x = ctypes.c_void_p(16)
    assert lib.atlas_layernorm_fwd(ctypes.byref(p), *[None] * 8) == L.ATLAS_ERR_INVALID_ARGUMENT
    assert lib.atlas_layernorm_fwd(ctypes.byref(p), x, x, x, x, x, None, x, None) == L.ATLAS_ERR_INVALID_ARGUMENT
    assert lib.atlas_layernorm_bwd(ctypes.byref(p), *[x] * 9, 16, None) == L.ATLAS_ERR_WORKSPACE
    odd = ctypes.c_void_p(20)
    assert lib.atlas_layernorm_fwd(ctypes.byref(p), x, None, x, x, x, None, odd, None) == L.ATLAS_ERR_INVALID_ARGUMENT
