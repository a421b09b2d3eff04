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
