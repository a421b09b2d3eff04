"""Decay attention kernels (include/atlas_decay.h) against the token-by-token float64
recurrence and its autograd (tests/decay_ref.py).

Tolerances (relative Frobenius), from the arithmetic: a bf16 output is rounded once
(2^-9) after scores rounded once (2^-9): 4e-3.  float32 outputs are sums of up to some
hundred float32 terms: 3e-6 on the CUDA cores; on the tensor cores float32 operands are
split into parts of 24 bits and a state adds up in 24 truncating steps of 2^-23: 4e-6.
dlog_decay adds signed terms that partly cancel: 2e-5."""
import pytest
import torch

import decay_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TOL = {BF: 4e-3, F32: 3e-6}
TOL_STATE, TOL_DG = 4e-6, 2e-5


def _inputs(B, T, H, D, dtype, fused, state, seed=0, decay=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, 3, H, D, device="cuda", generator=g)
    x = (x / x.norm(dim=-1, keepdim=True).clamp(min=1e-3)).to(dtype)
    q, k, v = x.unbind(2) if fused else (x[:, :, i].clone() for i in range(3))
    if decay is None:
        decay = torch.log1p(-torch.exp2(-torch.linspace(1, 9, H)))
    log_decay = torch.as_tensor(decay, dtype=F32).cuda()
    S = 0.3 * torch.randn(B, H, D, D, device="cuda", generator=g) if state else None
    dy = torch.randn(B, T, H, D, device="cuda", generator=g).to(dtype)
    dS = 0.1 * torch.randn(B, H, D, D, device="cuda", generator=g)
    return q, k, v, log_decay, S, dy, dS


def _reference(q, k, v, log_decay, S, scale, dy=None, dS=None):
    ins = [x.detach().cpu().double().requires_grad_(True) for x in (q, k, v, log_decay)]
    st = None if S is None else S.detach().cpu().double().requires_grad_(True)
    y, out = R.decay_attention(*ins, st, scale)
    if dy is None:
        return y, out
    ((y * dy.cpu().double()).sum() + (out * dS.cpu().double()).sum()).backward()
    return y, out, [x.grad for x in ins], None if st is None else st.grad


def _check(B, T, H, D, dtype, fused=True, state=True, decay=None, scale=0.37):
    from atlas_b200 import device_status
    from atlas_b200.decay_attention import decay_attention
    q, k, v, g, S, dy, dS = _inputs(B, T, H, D, dtype, fused, state, T + D, decay)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, g)]
    st = None if S is None else S.clone().requires_grad_(True)
    y, out = decay_attention(*leaves, st, scale)
    ((y.float() * dy.float()).sum() + (out * dS).sum()).backward()
    torch.cuda.synchronize()
    device_status()
    ry, rout, rg, rS = _reference(q, k, v, g, S, scale, dy, dS)
    tol = TOL[dtype]
    assert y.dtype == dtype and R.rel(y, ry) < tol
    assert R.rel(out, rout) < TOL_STATE
    for n, x, r in zip("qkv", leaves, rg):
        assert R.rel(x.grad, r) < tol, n
    fin = torch.isfinite(g.cpu())  # the derivative at log_decay = -infinity is not defined
    if fin.any():
        r = rg[3][fin]
        assert float((leaves[3].grad.cpu().double()[fin] - r).norm()) < TOL_DG * float(r.norm()) + 1e-6
    if S is not None:
        assert R.rel(st.grad, rS) < TOL_STATE


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,H,D", [(2, 300, 3, 64), (1, 1, 2, 64), (2, 2, 1, 64), (1, 127, 2, 64), (1, 128, 2, 64),
                                     (1, 129, 2, 64), (1, 257, 2, 128), (2, 200, 2, 96), (1, 150, 2, 32), (3, 70, 2, 8),
                                     (1, 140, 2, 24), (2, 33, 2, 7), (1, 65, 3, 1), (1, 131, 1, 127)])
def test_forward_backward(B, T, H, D, dtype):
    _check(B, T, H, D, dtype)


@pytest.mark.parametrize("B,T,H,D", [(1, 4133, 1, 64), (1, 1100, 2, 128), (1, 600, 3, 40), (2, 321, 5, 72)])
def test_many_segments(B, T, H, D):
    """Few heads: sequences cut into many segments, the last one short."""
    _check(B, T, H, D, BF)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("fused,state", [(False, False), (False, True), (True, False)])
def test_without_state_and_unfused(dtype, fused, state):
    _check(2, 200, 2, 64, dtype, fused, state)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 32)])
@pytest.mark.parametrize("decay", [[0.0, -1e-4], [-5.0, -0.7], [float("-inf"), -30.0]])
def test_extreme_decays(dtype, D, decay):
    """No decay, decays that leave only the last tokens, and none at all; nothing overflows."""
    _check(1, 300, 2, D, dtype, decay=decay)


def test_default_scale_and_forward_only():
    from atlas_b200.decay_attention import decay_attention_forward
    q, k, v, g, S, _, _ = _inputs(1, 140, 2, 64, BF, True, True)
    y, out, saved = decay_attention_forward(q, k, v, g, S, need_saved=False)
    y2, out2, saved2 = decay_attention_forward(q, k, v, g, S, scale=0.125)
    assert saved is None and saved2 is not None
    assert torch.equal(y, y2) and torch.equal(out, out2)


def test_odd_strides_take_the_other_path():
    """Rows that are not 16-byte aligned run on the CUDA cores and agree with aligned ones."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    q, k, v, g, S, dy, dS = _inputs(1, 150, 2, 64, BF, False, True)
    wide = [torch.zeros(1, 150, 2, 65, dtype=BF, device="cuda") for _ in range(3)]
    odd = []
    for w, x in zip(wide, (q, k, v)):
        w[..., 1:] = x
        odd.append(w[..., 1:])
    assert odd[0].stride(1) % 8 and odd[0].data_ptr() % 16
    res = []
    for a in ((q, k, v), odd):
        y, out, saved = decay_attention_forward(*a, g, S)
        res.append((y, out) + decay_attention_backward(*a, g, saved, dy, dS))
    for a, b, tol in zip(*res, (2 * TOL[BF], TOL_STATE + 3e-6) + (2 * TOL[BF],) * 3 + (2 * TOL_DG, TOL_STATE + 3e-6)):
        assert R.rel(a, b) < tol


@pytest.mark.parametrize("dtype", [BF, F32])
def test_broadcast_inputs(dtype):
    """k and v shared by the heads and q by the batch (stride 0): the gradients come back per
    head and autograd sums them into the shared tensors."""
    from atlas_b200.decay_attention import decay_attention
    B, T, H, D = 2, 140, 3, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q1 = torch.randn(1, T, H, D, device="cuda", generator=g).div_(8).to(dtype).requires_grad_(True)
    k1, v1 = (torch.randn(B, T, 1, D, device="cuda", generator=g).div_(8).to(dtype).requires_grad_(True) for _ in range(2))
    decay = torch.tensor([-0.01, -0.1, -1.0], device="cuda")
    dy = torch.randn(B, T, H, D, device="cuda", generator=g).to(dtype)
    y, _ = decay_attention(q1.expand(B, T, H, D), k1.expand(B, T, H, D), v1.expand(B, T, H, D), decay)
    y.backward(dy)
    r = [x.detach().cpu().double().requires_grad_(True) for x in (q1, k1, v1)]
    ry, _ = R.decay_attention(*(x.expand(B, T, H, D) for x in r), decay.cpu().double(), None, D ** -0.5)
    ry.backward(dy.cpu().double())
    assert R.rel(y, ry) < TOL[dtype]
    for x, ref in zip((q1, k1, v1), r):  # the sum over heads is rounded again
        assert R.rel(x.grad, ref.grad) < 2 * TOL[dtype]


@pytest.mark.parametrize("D", [64, 40])
def test_gradients_against_differences(D):
    """Directional derivatives of a loss of the float64 recurrence, by central differences,
    against the kernels' float32 gradients."""
    from atlas_b200.decay_attention import decay_attention
    q, k, v, g, S, dy, dS = _inputs(1, 150, 2, D, F32, True, True, 5)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v, g, S)]
    y, out = decay_attention(*leaves, scale=0.5)
    ((y * dy).sum() + (out * dS).sum()).backward()
    gen = torch.Generator().manual_seed(9)
    base = [x.detach().cpu().double() for x in leaves]

    def loss(xs):
        ry, rout = R.decay_attention(*xs, 0.5)
        return float((ry * dy.cpu().double()).sum() + (rout * dS.cpu().double()).sum())
    for i, x in enumerate(leaves):
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        eps = 1e-5
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + eps * d, base[i] - eps * d
        want = (loss(up) - loss(dn)) / (2 * eps)
        grad = x.grad.cpu().double()
        got = float((grad * d).sum())
        assert abs(got - want) < 1e-5 * float(grad.norm() * d.norm()), i


@pytest.mark.parametrize("dtype", [BF, F32])
def test_segments_and_steps_continue_a_prompt(dtype):
    """A prompt in two parts, then tokens one by one: the same outputs and state as at once."""
    from atlas_b200.decay_attention import decay_attention_forward, decay_attention_step
    q, k, v, g, S, _, _ = _inputs(2, 205, 3, 64, dtype, True, True, 1)
    y, out, _ = decay_attention_forward(q, k, v, g, S)
    y1, s1, _ = decay_attention_forward(q[:, :130], k[:, :130], v[:, :130], g, S)
    y2, s2, _ = decay_attention_forward(q[:, 130:200], k[:, 130:200], v[:, 130:200], g, s1)
    ys = [y1, y2]
    for t in range(200, 204):
        yt, st = decay_attention_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g, s2)
        assert st is s2
        ys.append(yt)
    yt, _ = decay_attention_step(q[:, 204:], k[:, 204:], v[:, 204:], g, s2)
    ys.append(yt)
    assert R.rel(torch.cat(ys, 1), y) < (2 * TOL[dtype])
    assert R.rel(s2, out) < 2 * TOL_STATE


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,H,D", [(1, 1, 12, 64), (3, 1, 2, 128), (2, 5, 2, 32), (5, 1, 3, 40), (2, 3, 2, 33), (1, 1, 1, 1)])
def test_step(B, T, H, D, dtype):
    from atlas_b200.decay_attention import decay_attention_step
    q, k, v, g, S, _, _ = _inputs(B, T, H, D, dtype, True, True, B)
    ry, rS = _reference(q, k, v, g, S, 0.5)
    keep = S.clone()
    y, out = decay_attention_step(q, k, v, g, S, scale=0.5, out=torch.empty_like(S))
    assert torch.equal(S, keep)
    # the step rounds y once, and sums at most D products
    assert R.rel(y, ry) < (2.1e-3 if dtype == BF else 3e-6) and R.rel(out, rS) < 1e-6
    y2, out2 = decay_attention_step(q, k, v, g, S, scale=0.5)
    assert out2 is S and torch.equal(y2, y) and torch.equal(S, out)


def test_step_slots():
    """States in a pool by slot: untouched rows stay, idle sequences give zeros."""
    from atlas_b200.decay_attention import decay_attention_step
    q, k, v, g, _, _, _ = _inputs(4, 1, 2, 64, BF, True, False)
    pool = torch.randn(7, 2, 64, 64, device="cuda")
    slots = torch.tensor([5, -1, 0, 7], dtype=torch.int32, device="cuda")
    keep = pool.clone()
    y, _ = decay_attention_step(q, k, v, g, pool, slots)
    for b, s in ((0, 5), (2, 0)):
        ry, rS = _reference(q[b:b + 1], k[b:b + 1], v[b:b + 1], g, keep[s:s + 1], 0.125)
        assert R.rel(y[b:b + 1], ry) < 2.1e-3 and R.rel(pool[s:s + 1], rS) < 1e-6
    assert (y[1] == 0).all() and (y[3] == 0).all()
    for s in (1, 2, 3, 4, 6):
        assert torch.equal(pool[s], keep[s])


def test_empty():
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward, decay_attention_step
    g = torch.tensor([-0.1, -0.2], device="cuda")
    for B, T in ((0, 5), (2, 0), (0, 0)):
        q = torch.empty(B, T, 2, 64, dtype=BF, device="cuda")
        S = torch.randn(B, 2, 64, 64, device="cuda")
        y, out, saved = decay_attention_forward(q, q, q, g, S)
        assert y.shape == q.shape and torch.equal(out, S)
        dq, dk, dv, dg, dS = decay_attention_backward(q, q, q, g, saved, q, S)
        assert dq.shape == q.shape and (dg == 0).all() and torch.equal(dS, S)
        y, out = decay_attention_step(q, q, q, g, S.clone())
        assert torch.equal(out, S)
    y, out, _ = decay_attention_forward(q, q, q, g)
    assert (out == 0).all()


def test_backward_is_deterministic_and_streams_are_kept():
    """Two backward passes agree bit for bit, on another stream than the tensors' own too."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    q, k, v, g, S, dy, dS = _inputs(2, 400, 3, 64, BF, True, True)
    _, _, saved = decay_attention_forward(q, k, v, g, S)
    a = decay_attention_backward(q, k, v, g, saved, dy, dS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = decay_attention_backward(q, k, v, g, saved, dy, dS)
    side.synchronize()
    for x, z in zip(a, b):
        assert torch.equal(x, z)


@pytest.mark.parametrize("T,D,need_saved", [(700, 128, True), (700, 128, False), (1500, 64, False), (300, 24, True)])
def test_state_in_its_own_place(T, D, need_saved):
    """The state left may go to where the one entering came from, also where a sequence is split."""
    from atlas_b200.decay_attention import _plan, decay_attention_forward
    q, k, v, g, S, _, _ = _inputs(2, T, 3, D, BF, True, True, T)
    y, out, saved = decay_attention_forward(q, k, v, g, S, 0.5, need_saved)
    p, q, k, v = _plan(q, k, v, g, 0.5)
    y2, S2 = torch.empty_like(y), S.clone()
    saved2 = torch.empty_like(saved) if need_saved else None
    n = p.saved_workspace_bytes if need_saved else p.fwd_workspace_bytes
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    assert 0 == p.lib.atlas_decay_fwd(p.ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), S2.data_ptr(),
                                      y2.data_ptr(), S2.data_ptr(), saved2.data_ptr() if need_saved else None,
                                      ws.data_ptr(), n, s)
    assert torch.equal(y, y2) and torch.equal(out, S2)
    assert not need_saved or torch.equal(saved, saved2)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 48)])
def test_in_a_graph(dtype, D):
    """Captured and replayed on new inputs in the same buffers: the chained kernels keep their order."""
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    ins = _inputs(1, 900, 3, D, dtype, False, True, 1)
    q, k, v, g, S, dy, dS = ins

    def call():
        y, out, saved = decay_attention_forward(q, k, v, g, S, 0.4)
        return (y, out) + decay_attention_backward(q, k, v, g, saved, dy, dS, 0.4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call()
    for seed in (2, 3):
        for t, u in zip(ins, _inputs(1, 900, 3, D, dtype, False, True, seed)):
            t.copy_(u)
        graph.replay()
        torch.cuda.synchronize()
        for x, r in zip(got, call()):
            assert torch.equal(x, r)


def test_offsets_beyond_32_bits():
    """Sequences more than 2^31 elements apart in one buffer."""
    from atlas_b200.decay_attention import decay_attention_forward, decay_attention_step
    T, H, D = 130, 1, 64
    far = (1 << 31) + 64
    buf = torch.empty(far + T * H * D, dtype=BF, device="cuda")
    q, k, v, g, _, _, _ = _inputs(2, T, H, D, BF, False, False)
    view = buf.as_strided((2, T, H, D), (far, H * D, D, 1))
    view.copy_(q)
    y, out, _ = decay_attention_forward(view, k, v, g)
    y2, out2, _ = decay_attention_forward(q, k, v, g)
    assert torch.equal(y, y2) and torch.equal(out, out2)
    S = torch.zeros(2, H, D, D, device="cuda")
    ys, _ = decay_attention_step(view[:, :1], k[:, :1], v[:, :1], g, S)
    assert R.rel(ys, y[:, :1]) < 2 * TOL[BF]


def test_refusals():
    from atlas_b200 import AtlasError
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward, decay_attention_step
    q, k, v, g, S, dy, _ = _inputs(2, 20, 2, 64, BF, False, True)
    for bad in ((q.half(), k, v, g), (q, k.float(), v, g), (q, k[:, :10], v, g), (q, k, v, g.double()),
                (q, k, v, g[:1]), (q[0], k, v, g), (q.cpu(), k, v, g)):
        with pytest.raises(ValueError):
            decay_attention_forward(*bad)
    with pytest.raises(ValueError):
        decay_attention_forward(q, k, v, g, S.double())
    with pytest.raises(ValueError):
        decay_attention_forward(q, k, v, g, S[:1])
    with pytest.raises(AtlasError):
        decay_attention_forward(q, k, v, g, scale=float("nan"))
    big = torch.zeros(1, 3, 1, 136, dtype=BF, device="cuda")
    with pytest.raises(AtlasError):
        decay_attention_forward(big, big, big, g[:1])
    _, _, saved = decay_attention_forward(q, k, v, g, S)
    with pytest.raises(ValueError):
        decay_attention_backward(q, k, v, g, saved[:-1], dy)
    with pytest.raises(ValueError):
        decay_attention_backward(q, k, v, g, saved, dy.float())
    with pytest.raises(ValueError):
        decay_attention_step(q, k, v, g, S, slots=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        decay_attention_step(q, k, v, g, S[:1])
    with pytest.raises(ValueError):
        decay_attention_step(q, k, v, g, S, out=S[:, :1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_mixer_trains_and_generates(dtype):
    """The mixer block: gradients reach every parameter, and generating token by token from
    a prompt's state gives what the whole sequence gives."""
    from atlas_b200.mixer import DecayMixer
    torch.manual_seed(0)
    B, T, C, H = 2, 150, 128, 2
    m = DecayMixer(C, H).cuda()
    x, delta = (torch.randn(B, T, C, device="cuda").to(dtype).requires_grad_(True) for _ in range(2))
    out, h, state = m(x, delta)
    (out.float().square().sum() + h.float().sum()).backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, n
    assert torch.isfinite(x.grad).all() and torch.equal(x.grad, delta.grad)
    with torch.no_grad():
        pre, _, st = m(x[:, :140], delta[:, :140])
        pool = torch.zeros(5, H, C // H, C // H, device="cuda")
        slots = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
        pool[slots.long()] = st
        outs = [pre]
        for t in range(140, T):
            o, hs = m.step(x[:, t:t + 1], pool, slots, delta[:, t:t + 1])
            assert torch.equal(hs, h[:, t:t + 1])
            outs.append(o)
    # bf16: the per-head norm follows outputs rounded differently, and two GEMMs round again
    assert R.rel(torch.cat(outs, 1), out) < (1.5e-2 if dtype == BF else 2e-5)
    assert R.rel(pool[slots.long()], state) < (1e-2 if dtype == BF else 1e-5)
