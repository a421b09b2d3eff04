"""CPU checks of the Python side of decay attention and layer norm, with the library and the
device queries replaced: what buffers a call makes, which calls it refuses, and what autograd
is told."""
import ast
import glob
import os
import types

import pytest
import torch

from atlas_b200 import scan


@pytest.fixture
def host(monkeypatch):
    """No device: CPU tensors count as device 0's, launches are noted in ``host.calls``, and the
    one stream captures while ``host.capturing`` is set."""
    from atlas_b200 import decay_attention, layer_norm
    h = types.SimpleNamespace(capturing=False, calls=[])

    class Library:
        def __getattr__(self, name):
            return lambda *a: h.calls.append((name, a)) or 0

    def planned(module):
        real = module._Plan

        def plan(*keys):
            dev0 = [k if not isinstance(k, tuple) else tuple(0 if type(i) is int and i < 0 else i for i in k) for k in keys]
            p = real(*dev0)
            p.lib = Library()
            return p
        monkeypatch.setattr(module, "_plans", plan)
    planned(decay_attention)
    planned(layer_norm)
    for m in (scan, decay_attention, layer_norm):
        monkeypatch.setattr(m, "away", lambda dev: False)
        monkeypatch.setattr(m, "stream_of", lambda dev: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: h.capturing)
    return h


def test_captured_scratch_is_the_graphs_own(host):
    """A captured call's address is replayed for as long as the graph lives: its scratch is neither
    a buffer that a later, larger call replaces nor one that another call or graph uses."""
    ws, dev = scan.Workspace(), torch.device("cpu")
    eager, _ = ws.get(100, dev)
    host.capturing = True
    a, n = ws.get(50, dev)
    b, _ = ws.get(50, dev)
    assert n >= 50 and a.numel() >= 50
    assert len({x.data_ptr() for x in (eager, a, b)}) == 3
    assert ws.get(0, dev) == (None, 0)
    host.capturing = False
    assert ws.get(80, dev)[0] is eager
    larger, n = ws.get(200, dev)
    assert n >= 200 and larger is not eager and ws.get(200, dev)[0] is larger


def _decay_inputs(B=2, T=70, H=3, D=16, dtype=torch.bfloat16):
    q, k, v = (torch.zeros(B, T, H, D, dtype=dtype) for _ in range(3))
    return q, k, v, torch.zeros(H, dtype=torch.float32)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_buffers_are_float32_under_any_default_type(host, default):
    """The kernels write float32 states, statistics and parameter gradients whatever type torch makes
    by default: half as many bytes would be written past their end."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    torch.set_default_dtype(default)
    try:
        q, k, v, g = _decay_inputs()
        y, out, saved = decay_attention_forward(q, k, v, g)
        assert out.dtype == torch.float32 and out.shape == (2, 3, 16, 16)
        assert saved.numel() * saved.element_size() == 2 * 3 * 2 * 16 * 16 * 4  # two chunks of 64 tokens
        dq, dk, dv, dg, dS = decay_attention_backward(q, k, v, g, saved, y)
        assert dg.dtype == torch.float32 and dS.dtype == torch.float32 and dS.shape == out.shape
        x = torch.zeros(5, 4, 16, dtype=torch.bfloat16)
        y, h, stats = layer_norm_forward(x)
        assert stats.dtype == torch.float32 and stats.shape == (20, 2)
        dx, dw, db = layer_norm_backward(y, h, None, stats)
        assert dw.dtype == torch.float32 and db.dtype == torch.float32 and dw.shape == (16,)
    finally:
        torch.set_default_dtype(torch.float32)
    assert [n for n, _ in host.calls] == ["atlas_decay_fwd", "atlas_decay_bwd", "atlas_layernorm_fwd", "atlas_layernorm_bwd"]


def test_every_device_buffer_names_its_type():
    """A buffer that the library fills never takes torch's default type, in any of the package's calls."""
    bare = []
    for path in glob.glob(os.path.join(os.path.dirname(scan.__file__), "*.py")):
        for n in ast.walk(ast.parse(open(path).read())):
            if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute) and n.func.attr in ("empty", "zeros", "full") \
                    and isinstance(n.func.value, ast.Name) and n.func.value.id == "torch":
                names = {k.arg for k in n.keywords}
                if "device" in names and "dtype" not in names:
                    bare.append(f"{os.path.basename(path)}:{n.lineno}")
    assert not bare


def _second_derivative(y, x):
    """Differentiates a first derivative of y by x again."""
    g, = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    (y.float().sum() + g.float().square().sum()).backward()


def test_second_derivatives_are_refused(host):
    """The backward kernels are no graph that autograd could differentiate: a penalty on a
    gradient raises and is not dropped without a word."""
    from atlas_b200.decay_attention import decay_attention
    from atlas_b200.layer_norm import layer_norm
    q, k, v, g = _decay_inputs()
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        _second_derivative(decay_attention(q, k, v, g)[0], q)
    x, r = (torch.zeros(5, 4, 16, requires_grad=True) for _ in range(2))
    with pytest.raises(RuntimeError, match="first derivatives"):
        _second_derivative(layer_norm(x), x)
    with pytest.raises(RuntimeError, match="first derivatives"):
        _second_derivative(layer_norm(x, residual=r)[1], r)
    # first derivatives are as before, with create_graph too
    assert torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)[0].shape == x.shape
    y, h = layer_norm(x, residual=r)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == r.grad.shape == x.shape and not x.grad.requires_grad


def test_every_kernel_backward_has_first_derivatives_only():
    """The same for the package's other autograd Functions: their backward is wrapped."""
    from atlas_b200 import decay_attention, layer_io, layer_norm, swa
    functions = {f for m in (scan, decay_attention, layer_io, layer_norm, swa) for f in vars(m).values()
                 if isinstance(f, type) and issubclass(f, torch.autograd.Function) and f is not scan._FirstDerivatives}
    assert len(functions) == 6
    assert [f.__name__ for f in functions if not hasattr(f.backward, "__wrapped__")] == []


def test_the_step_tells_autograd_what_it_writes(host):
    """A state that autograd has saved for a backward is not overwritten unnoticed."""
    from atlas_b200.decay_attention import decay_attention_step
    q, k, v, g = _decay_inputs(T=1)
    w = torch.ones((), requires_grad=True)
    for other in (False, True):
        state = torch.zeros(2, 3, 16, 16)
        out = torch.zeros_like(state) if other else state
        loss = (w * out).sum()
        versions = state._version, out._version
        decay_attention_step(q, k, v, g, state, out=out if other else None)
        assert out._version > versions[1] and (not other or state._version == versions[0])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        decay_attention_step(q, k, v, g, torch.zeros(2, 3, 16, 16))


def test_the_step_refuses_to_drop_gradients(host):
    """The step has no backward: inputs that want gradients are refused where gradients are recorded, and
    taken under no_grad."""
    from atlas_b200.decay_attention import decay_attention_step
    for i in range(8):
        if i in (5, 6):  # slots, scale
            continue
        ins = [*_decay_inputs(T=1), torch.zeros(2, 3, 16, 16), None, 1.0, torch.zeros(2, 3, 16, 16)]
        ins[i].requires_grad_(True)
        with pytest.raises(ValueError, match="no_grad"):
            decay_attention_step(*ins)
        assert not host.calls
        with torch.no_grad():
            decay_attention_step(*ins)
        assert len(host.calls) == 1
        host.calls.clear()
    decay_attention_step(*_decay_inputs(T=1), torch.zeros(2, 3, 16, 16))


def test_empty_views(host):
    """An empty tensor's strides say nothing (contiguous() keeps them): empty batches and sequences in any
    layout, and broadcast, are valid calls."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward, decay_attention_step
    g = torch.zeros(4)
    transposed = torch.empty(2, 16, 4, 0, dtype=torch.bfloat16).permute(0, 3, 2, 1)
    assert transposed.shape == (2, 0, 4, 16) and transposed.stride(3) != 1
    broadcast = torch.zeros(2, 1, 1, 16, dtype=torch.bfloat16).expand(2, 1, 4, 16)[:, :0]
    nobody = torch.empty(16, 5, 4, 0).permute(3, 1, 2, 0)
    for q in (transposed, broadcast, nobody, nobody.bfloat16()):
        B = q.shape[0]
        y, out, saved = decay_attention_forward(q, q, q, g)
        assert y.shape == q.shape and out.shape == (B, 4, 16, 16) and saved.numel() == 0
        assert decay_attention_backward(q, q, q, g, saved, y)[0].shape == q.shape
        assert decay_attention_step(q, q, q, g, out)[0].shape == q.shape


def test_numbers_given_as_tensors_are_read_at_every_call(host):
    """A scale or eps held in a tensor is its value now, not what it was when a plan was made for that tensor."""
    import functools

    from atlas_b200 import decay_attention as D
    from atlas_b200 import layer_norm as N
    seen = []

    @functools.lru_cache
    def plans(*keys):
        seen.append(keys)
        return made(*keys)
    for module, call in ((D, lambda t: D.decay_attention_forward(*_decay_inputs(), scale=t)),
                         (N, lambda t: N.layer_norm_forward(torch.zeros(3, 16), eps=t))):
        made, module._plans = module._plans, plans
        seen.clear()
        t = torch.tensor(0.5)
        call(t)
        t.fill_(0.25)
        call(t)
        call(0.25)
        module._plans = made
        numbers = [[k for k in keys if isinstance(k, float)] for keys in seen]
        assert numbers == [[0.5], [0.25]], module


def test_sizes_beyond_32_bits_are_refused(host, monkeypatch):
    """The C parameters hold sizes in 32 bits: larger ones raise and are not cut down."""
    from atlas_b200 import decay_attention as D
    from atlas_b200 import layer_norm as N
    from atlas_b200 import AtlasError
    big, bf = (1 << 32) + 1, torch.bfloat16
    for shape in ((big, 1, 1, 1), (1, big, 1, 1), (1, 1, big, 1), (1, 1, 1, big), (1 << 31, 1, 1, 1)):
        x = torch.empty(1, dtype=bf).expand(shape)
        with pytest.raises((ValueError, AtlasError)):
            D.decay_attention_forward(x, x, x, torch.zeros(1).expand(shape[2]))
    with pytest.raises(AtlasError):
        N.layer_norm_forward(torch.empty(1, dtype=bf).expand(big))
    q, k, v, g = _decay_inputs(T=1, H=1, D=1)
    pool = torch.empty(1).expand(big, 1, 1, 1)
    monkeypatch.setattr(D, "_need", lambda *a: None)  # (this one is not contiguous)
    with pytest.raises(ValueError):
        D.decay_attention_step(q, k, v, g, pool, torch.zeros(2, dtype=torch.int32))
    assert not host.calls


def test_products_of_sizes_do_not_wrap():
    """B * H * T near and beyond 2^63 is too large a problem, not a small one."""
    import ctypes

    from atlas_b200 import _lib as L
    from atlas_b200.decay_attention import AtlasDecayParams, _lib
    lib, s = _lib(), (ctypes.c_int64 * 3)(0, 0, 0)
    for B, T, H in ((1 << 29, 1, 1 << 29), ((1 << 31) - 1, 1 << 30, (1 << 31) - 1), (1 << 30, 0, 1 << 30), (1 << 30, 1 << 30, 1 << 5)):
        p = ctypes.byref(AtlasDecayParams(L.ATLAS_ABI_VERSION, B, T, H, 1, L.ATLAS_F32, 1.0, 0, s, s, s))
        assert lib.atlas_decay_saved_bytes(p) == 0 and b"too large" in lib.atlas_last_error_string(), (B, T, H)
        assert lib.atlas_decay_step(p, *[None] * 6, 0, *[None] * 3) == L.ATLAS_ERR_UNSUPPORTED


def test_saved_states_have_to_be_contiguous(host):
    """The backward reads as many bytes as were saved from the buffer's start on."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    q, k, v, g = _decay_inputs()
    y, _, saved = decay_attention_forward(q, k, v, g)
    every_other = torch.empty(2 * saved.numel())[::2]
    with pytest.raises(ValueError, match="saved"):
        decay_attention_backward(q, k, v, g, every_other, y)
    with pytest.raises(ValueError, match="saved"):
        decay_attention_backward(q, k, v, g, saved[:1].expand(saved.numel()), y)
    decay_attention_backward(q, k, v, g, saved, y)


def test_head_size_zero_is_refused_like_other_sizes(host):
    from atlas_b200 import AtlasError
    from atlas_b200.decay_attention import decay_attention_forward
    with pytest.raises(AtlasError, match="positive"):
        decay_attention_forward(*_decay_inputs(D=0))
