"""Decay attention and layer norm as programs call them: captured in graphs, under other default
types, far from the tests' usual sizes.  Against float64 (tests/decay_ref.py) or against the same
call made eagerly."""
import pytest
import torch

import decay_ref as R
from test_gpu_decay_attention import _inputs

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _train(ins):
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward
    q, k, v, g, S, dy, dS = ins
    y, out, saved = decay_attention_forward(q, k, v, g, S, 0.4)
    return (y, out) + decay_attention_backward(q, k, v, g, saved, dy, dS, 0.4)


def _norm(x, w, dy):
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    y, h, stats = layer_norm_forward(x, w, w)
    return (y,) + layer_norm_backward(dy, h, w, stats)


def _captured(call, stream):
    with torch.cuda.stream(stream):
        call()  # (eager scratch of this stream, smaller than the calls that come after the capture)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    return graph, out


def test_graphs_outlive_the_scratch_of_their_stream():
    """After a capture a larger eager call on the capturing stream, then tensors that may take over any
    memory that was freed: a replay writes none of them, and two graphs replayed on two
    streams give what each gives alone."""
    ins = _inputs(1, 900, 3, 64, BF, False, True, 1)
    big = _inputs(4, 3000, 6, 64, BF, False, True, 2)
    x, dy = (torch.randn(5000, 768, device="cuda").to(BF) for _ in range(2))
    w = torch.randn(768, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g1, out1 = _captured(lambda: _train(ins), side)
    g2, out2 = _captured(lambda: _norm(x, w, dy), side)
    with torch.cuda.stream(side):
        _train(big)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        guard = [torch.full((1 << 20,), 3, dtype=torch.uint8, device="cuda") for _ in range(96)]
    torch.cuda.synchronize()
    want1, want2 = _train(ins), _norm(x, w, dy)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for g, s in zip((g1, g2), streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, want in ((out1, want1), (out2, want2)):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        assert all(bool((t == 3).all()) for t in guard)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_long_generation_keeps_the_states_accuracy(dtype):
    """4096 single tokens at decays of 1 - 2^-9 .. 1 - 2^-12.  An update rounds the state once, at
    most 2^-24 of it and at random; some 2^11 of them are remembered: sqrt(2^11) 2^-24 = 2.7e-6 at most,
    below the 4e-6 that the prompt's states are held to.  A decay rounded to float32 adds up to 2^12 2^-25."""
    from atlas_b200.decay_attention import decay_attention_step
    T, H, D = 4096, 4, 64
    e = torch.tensor([9.0, 10.0, 11.0, 12.0], dtype=torch.float64)
    q, k, v, g, S, _, _ = _inputs(1, T, H, D, dtype, True, True, 4, torch.log1p(-torch.exp2(-e)).float())
    ref, kd, vd = S.double(), k.double(), v.double()
    lam = torch.exp(g.double())[None, :, None, None]
    for t in range(T):
        decay_attention_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], g, S)
        ref = lam * ref + kd[:, t, :, :, None] * vd[:, t, :, None, :]
    for h in range(H):
        assert R.rel(S[:, h], ref[:, h]) < 4e-6, h


@pytest.mark.parametrize("shape", [(40, 768), (9, 12, 64), (21, 787), (5, 8192), (3, 5069), (3, 20000), (2, 262144), (30, 8)])
def test_a_large_mean_costs_the_output_no_digits(shape):
    """Float32 vectors with a mean a thousand and ten thousand times the deviation: differences from a
    float32 near the mean are exact, and what that float32 misses of the mean is summed with them, so y
    is held to the bound of other float32 outputs (2e-6), long vectors' too."""
    from atlas_b200.layer_norm import layer_norm_forward
    g = torch.Generator(device="cuda").manual_seed(5)
    w, b = (torch.randn(shape[1:], device="cuda", generator=g) for _ in range(2))
    for mean in (1e3, -1e4):
        x = mean + torch.randn(shape, device="cuda", generator=g)
        y, _, st = layer_norm_forward(x, w, b)
        xd = x.cpu().double()
        assert R.rel(y, R.layer_norm(xd, w.cpu().double(), b.cpu().double(), 1e-5)) < 2e-6, mean
        if shape[-1] > 8:  # the mean is kept in float32
            assert (st[:, 0].cpu().double() - xd.mean(-1).reshape(-1)).abs().max() < 2 ** -23 * abs(mean) * 1.05


def _tokens(q, k, v, g, S, scale):
    """The recurrence in float64 on the GPU: y and the state left."""
    q, k, v, S = q.double(), k.double(), v.double(), S.double()
    lam, ys = torch.exp(g.double())[None, :, None, None], []
    for t in range(q.shape[1]):
        S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        ys.append(scale * (q[:, t, :, None, :] @ S)[..., 0, :])
    return torch.stack(ys, 1), S


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("D", [8, 32, 40, 48, 64, 96, 128])
def test_step_of_many_sequences(D, T, dtype):
    """More (sequence, head) pairs than the step cuts into narrow slices, in a pool with idle slots.
    Tolerances as for few sequences: y rounded once, sums of at most D products."""
    from atlas_b200.decay_attention import decay_attention_step
    B, H = 60, 6
    q, k, v, g, _, _, _ = _inputs(B, T, H, D, dtype, True, False, D)
    pool = torch.randn(B + 7, H, D, D, device="cuda")
    slots = torch.randperm(B + 7, device="cuda")[:B].to(torch.int32)
    slots[5], slots[41] = -1, B + 7
    on = (slots >= 0) & (slots < B + 7)
    rows = slots[on].long()
    ry, rS = _tokens(q[on], k[on], v[on], g, pool[rows], 0.3)
    new = torch.randn_like(pool)
    keep, before = new.clone(), pool.clone()
    y, out = decay_attention_step(q, k, v, g, pool, slots, scale=0.3, out=new)
    assert out is new and torch.equal(pool, before)
    assert R.rel(y[on], ry) < (2.1e-3 if dtype == BF else 3e-6) and R.rel(new[rows], rS) < 1e-6
    assert (y[~on] == 0).all()
    rest = torch.ones(B + 7, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert torch.equal(new[rest], keep[rest])
    y2, _ = decay_attention_step(q, k, v, g, pool, slots, scale=0.3)
    assert torch.equal(y2, y) and torch.equal(pool[rows], new[rows]) and torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (BF, 40), (F32, 48), (F32, 128)])
@pytest.mark.parametrize("B,T,H", [(30, 200, 6), (50, 67, 6)])
def test_more_chains_than_sms(B, T, H, dtype, D):
    """Forward and backward with a CTA for each whole sequence, more of them than run at once.
    Tolerances as in test_gpu_decay_attention.py."""
    from atlas_b200.decay_attention import decay_attention
    q, k, v, g, S, dy, dS = _inputs(B, T, H, D, dtype, True, True, B)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v, g, S)]
    y, out = decay_attention(*leaves, 0.37)
    ((y.float() * dy.float()).sum() + (out * dS).sum()).backward()
    ref = [x.detach().double().requires_grad_(True) for x in (q, k, v, g, S)]
    ry, rout = _tokens(*ref, 0.37)
    ((ry * dy.double()).sum() + (rout * dS.double()).sum()).backward()
    tol = 4e-3 if dtype == BF else 3e-6
    assert R.rel(y, ry) < tol and R.rel(out, rout) < 4e-6
    for x, r, t in zip(leaves, ref, (tol, tol, tol, 2e-5, 4e-6)):
        assert R.rel(x.grad, r.grad) < t


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(30011, 768), (9001, 2048), (3001, 12, 64), (24007, 256), (1201, 12288), (2003, 3, 1000)])
def test_norm_of_more_rows_than_the_rings_hold(shape, dtype):
    """Every team goes round its ring of vectors more than once, with a residual and dh; float64 on the
    GPU.  Tolerances as in test_gpu_layer_norm.py; thousands of rows add up in float32 (random signs:
    sqrt(30011) 2^-24 of a row's share at most)."""
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    g = torch.Generator(device="cuda").manual_seed(7)
    rn = lambda s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x, res, dy, dh = (rn(shape).to(dtype) for _ in range(4))
    w, b = 1 + 0.3 * rn(shape[1:]), 0.2 * rn(shape[1:])
    y, h, st = layer_norm_forward(x, w, b, 1e-5, res)
    dx, dw, db = layer_norm_backward(dy, h, w, st, dh)
    ref = [t.double().requires_grad_(True) for t in (h, w, b)]
    ry = R.layer_norm(*ref, 1e-5)
    ((ry * dy.double()).sum() + (ref[0] * dh.double()).sum()).backward()
    tol = 2.1e-3 if dtype == BF else 2e-6
    assert R.rel(h, (x.double() + res.double()).to(dtype)) < (1e-4 if dtype == BF else 1e-7)
    assert R.rel(y, ry) < tol and R.rel(dx, ref[0].grad) < tol
    assert R.rel(dw, ref[1].grad) < 2e-6 and R.rel(db, ref[2].grad) < 2e-6


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(700, 768), (5000, 6, 64), (3000, 787), (900, 2048), (40, 5069), (30, 20000), (5000, 7), (600, 3, 1000)])
def test_norm_outputs_in_the_place_of_inputs(shape, dtype):
    """h in the buffer of x or of residual, dx in that of dy or of dh: bit for bit as elsewhere."""
    from atlas_b200 import layer_norm as N
    g = torch.Generator(device="cuda").manual_seed(8)
    rn = lambda s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x, res, dy, dh = (rn(shape).to(dtype) for _ in range(4))
    w, b = rn(shape[1:]), rn(shape[1:])
    y, h, st = N.layer_norm_forward(x, w, b, 1e-5, res)
    dx, dw, db = N.layer_norm_backward(dy, h, w, st, dh)
    p, s = N._plan(x, w, b, 1e-5), torch.cuda.current_stream().cuda_stream
    ptr = lambda *t: [i.data_ptr() for i in t]  # noqa: E731
    for where in range(2):
        ins = [x.clone(), res.clone()]
        y2, st2 = torch.empty_like(y), torch.empty_like(st)
        assert 0 == p.lib.atlas_layernorm_fwd(p.ref, *ptr(*ins, w, b, y2, ins[where], st2), s)
        assert torch.equal(y2, y) and torch.equal(ins[where], h) and torch.equal(st2, st)
        assert torch.equal(ins[1 - where], (x, res)[1 - where])
        grads = [dy.clone(), dh.clone()]
        dw2, db2 = torch.empty_like(dw), torch.empty_like(db)
        ws = torch.empty(p.workspace_bytes, dtype=torch.uint8, device="cuda")
        assert 0 == p.lib.atlas_layernorm_bwd(p.ref, *ptr(grads[0], h, w, st, grads[1], grads[where], dw2, db2, ws),
                                              p.workspace_bytes, s)
        assert torch.equal(grads[where], dx) and torch.equal(dw2, dw) and torch.equal(db2, db)


def test_calls_under_another_default_type():
    ins = _inputs(2, 150, 2, 64, BF, True, False, 3)
    x, dy, w = torch.randn(50, 768, device="cuda").to(BF), torch.randn(50, 768, device="cuda").to(BF), torch.ones(768, device="cuda")
    want = _train(ins) + _norm(x, w, dy)
    torch.set_default_dtype(BF)
    try:
        got = _train(ins) + _norm(x, w, dy)
    finally:
        torch.set_default_dtype(F32)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_empty_views_on_the_device():
    from atlas_b200.decay_attention import decay_attention_backward, decay_attention_forward, decay_attention_step
    g, S = torch.zeros(4, device="cuda"), torch.randn(2, 4, 16, 16, device="cuda")
    q = torch.empty(2, 16, 4, 0, dtype=BF, device="cuda").permute(0, 3, 2, 1)
    y, out, saved = decay_attention_forward(q, q, q, g, S)
    dq, _, _, dg, dS = decay_attention_backward(q, q, q, g, saved, y, S)
    assert y.shape == dq.shape == q.shape and torch.equal(out, S) and torch.equal(dS, S) and (dg == 0).all()
    assert torch.equal(decay_attention_step(q, q, q, g, S.clone())[1], S)


@pytest.mark.parametrize("whole", [False, True])
def test_a_bf16_mixer_against_float64(whole):
    """The block with bf16 projections, and with every parameter in bf16 (its decays are then those of
    the rounded logits), against the formulas in float64 on the same parameters.  Up to eight roundings of
    2^-9 lie between the input and an output: n, q, k, v, the scores, a, its norm, out."""
    from atlas_b200.mixer import DecayMixer
    torch.manual_seed(1)
    B, T, C, H = 2, 150, 128, 2
    m = DecayMixer(C, H).cuda()
    if whole:
        m.bfloat16()
    else:
        m.to_qkv.bfloat16()
        m.to_out.bfloat16()
    x, delta = (torch.randn(B, T, C, device="cuda").to(BF) for _ in range(2))
    out, h, state = m(x, delta)
    P = {n: p.detach().double() for n, p in m.named_parameters()}
    hd = h.double()
    n = R.layer_norm(hd, P["norm_weight"], P["norm_bias"], m.eps)
    q, k, v = (n @ P["to_qkv.weight"].t()).view(B, T, 3, H, C // H).unbind(2)
    a, S = _tokens(q, k, v, torch.nn.functional.logsigmoid(P["decay_logit"]), torch.zeros_like(state), (C // H) ** -0.5)
    ref = R.layer_norm(a, P["head_weight"], P["head_bias"], m.eps).reshape(B, T, C) @ P["to_out.weight"].t()
    assert out.dtype == BF and R.rel(out, ref) < 8 * 2 ** -9 and R.rel(state, S) < 3 * 2 ** -9
    (out.float().square().sum() + h.float().sum()).backward()
    for name, p in m.named_parameters():
        assert torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, name
