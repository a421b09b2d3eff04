"""Layer norm kernels (include/atlas_norm.h) against float64 (tests/decay_ref.py).

Tolerances (relative Frobenius): a bf16 output is rounded once (at most 2^-9): 2.1e-3;
float32 sums of up to N terms in a tree, and parameter gradients of up to some thousand
rows in order: 2e-6."""
import pytest
import torch

import decay_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
TOL = {BF: 2.1e-3, F32: 2e-6}


def _make(shape, wshape, dtype, seed=0, mean=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x = (mean + 1.5 * rn(shape)).to(dtype)
    return x, rn(shape).to(dtype), 1 + 0.3 * rn(wshape), 0.2 * rn(wshape), rn(shape).to(dtype), rn(shape).to(dtype)


def _check(x, res, w, b, dy, dh, eps=1e-5, tol=None):
    """Forward and backward through autograd against the float64 formula's autograd."""
    from atlas_b200.layer_norm import layer_norm
    tol = tol or TOL[x.dtype]
    leaves = [None if t is None else t.detach().clone().requires_grad_(True) for t in (x, w, b, res)]
    got = layer_norm(leaves[0], leaves[1], leaves[2], eps, leaves[3])
    y, h = got if res is not None else (got, None)
    loss = (y.float() * dy.float()).sum()
    if h is not None:
        loss = loss + (h.float() * dh.float()).sum()
    loss.backward()
    hr = (x.double() + res.double()).to(x.dtype) if res is not None else x
    if h is not None:  # the float32 sum of two bf16 values may be rounded twice
        assert R.rel(h, hr) < (1e-4 if x.dtype == BF else 1e-7)
        hr = h.detach()
    ref = [None if t is None else t.detach().cpu().double().requires_grad_(True) for t in (hr, w, b)]
    yr = R.layer_norm(*ref, eps)
    lr = (yr * dy.cpu().double()).sum()
    if h is not None:
        lr = lr + (ref[0] * dh.cpu().double()).sum()
    lr.backward()
    assert y.dtype == x.dtype and R.rel(y, yr) < tol
    assert R.rel(leaves[0].grad, ref[0].grad) < tol
    if res is not None:
        assert torch.equal(leaves[3].grad, leaves[0].grad)
    for p, r in ((leaves[1], ref[1]), (leaves[2], ref[2])):
        if p is not None:
            assert p.grad.shape == p.shape and R.rel(p.grad, r.grad) < 2e-6


SHAPES = [((70, 768), (768,)), ((3, 5, 64), (64,)), ((9, 12, 64), (12, 64)), ((2, 33, 4, 32), (4, 32)), ((40, 8, 128), (8, 128)),
          ((33, 8, 48), (8, 48)), ((7, 3, 50), (3, 50)), ((5, 787), (787,)), ((1, 1024), (1024,)), ((6, 2048), (2048,)),
          ((4, 5069), (5069,)), ((3, 8192), (8192,)), ((3, 20000), (20000,)), ((2, 2, 9001), (2, 9001)), ((11, 7), (7,)),
          ((700, 600, 16), (600, 16)), ((5, 3, 1000), (3, 1000)), ((5000, 256), (256,)), ((13, 2), (2,)), ((6, 1, 512), (1, 512))]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,wshape", SHAPES)
def test_forward_backward(shape, wshape, dtype):
    x, res, w, b, dy, dh = _make(shape, wshape, dtype)
    _check(x, None, w, b, dy, dh)
    _check(x, res, w, b, dy, dh)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,wshape", [((20011, 33), (33,)), ((6007, 261), (261,)), ((9001, 3, 17), (3, 17)), ((2411, 1031), (1031,))])
def test_many_odd_rows(shape, wshape, dtype):
    """Rows at every alignment, more of them than the vectors that a team holds at once."""
    x, res, w, b, dy, dh = _make(shape, wshape, dtype)
    _check(x, res, w, b, dy, dh)
    _check(x, None, w, b, dy, dh)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_missing_parameters(dtype):
    x, res, w, b, dy, dh = _make((20, 4, 64), (4, 64), dtype)
    _check(x, None, None, None, dy, dh)
    _check(x, None, w, None, dy, dh)
    _check(x, None, None, b, dy, dh)
    _check(x, res, None, None, dy, dh)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [64, 768, 4096])
def test_unaligned_rows(N, dtype):
    """Buffers that start off the 16-byte grid."""
    x, res, w, b, dy, dh = _make((6, N), (N,), dtype)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731
    x = off(x)
    assert x.data_ptr() % 16
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    y, h, st = layer_norm_forward(x, off(w), off(b), 1e-5, off(res))
    y2, h2, st2 = layer_norm_forward(x.clone(), w, b, 1e-5, res)
    assert torch.equal(h, h2) and R.rel(y, y2) < (TOL[dtype] if dtype == BF else 1e-6)
    a = layer_norm_backward(off(dy), off(h), off(w), st, off(dh))
    c = layer_norm_backward(dy, h, w, st, dh)
    for i, j, t in zip(a, c, (TOL[dtype], 2e-6, 2e-6)):
        assert R.rel(i, j) < t


def test_large_mean_and_constant_rows():
    """A mean a thousand times the deviation costs the digits of the input's own rounding
    only; a constant vector gives the bias; the gradient stays finite."""
    from atlas_b200.layer_norm import layer_norm, layer_norm_forward
    g = torch.Generator(device="cuda").manual_seed(2)
    x = 1000 + torch.randn(30, 768, device="cuda", generator=g)
    w, b = torch.randn(768, device="cuda", generator=g), torch.randn(768, device="cuda", generator=g)
    y, _, st = layer_norm_forward(x, w, b)
    ref = R.layer_norm(x.cpu().double(), w.cpu().double(), b.cpu().double(), 1e-5)
    assert R.rel(y, ref) < 2e-4  # the float32 mean of values near 1000 is known to 6e-5
    c = torch.full((4, 768), 3.0, device="cuda", requires_grad=True)
    y = layer_norm(c, w, b)
    assert torch.equal(y, b.expand(4, 768))
    y.sum().backward()
    assert torch.isfinite(c.grad).all()
    n = torch.zeros(2, 1, device="cuda")
    assert (layer_norm_forward(n)[0] == 0).all()


def test_nonfinite_vectors_stay_apart():
    """An infinity or NaN spoils its own vector and no other."""
    from atlas_b200.layer_norm import layer_norm_forward
    x, _, w, b, _, _ = _make((50, 12, 64), (12, 64), BF)
    clean = layer_norm_forward(x, w, b)[0]
    x[3, 5, 7], x[20, 0, 0] = float("nan"), float("inf")
    y = layer_norm_forward(x, w, b)[0]
    bad = torch.zeros(50, 12, dtype=torch.bool, device="cuda")
    bad[3, 5] = bad[20, 0] = True
    assert torch.equal(y[~bad], clean[~bad]) and torch.isnan(y[3, 5]).all()


def test_gradients_against_differences():
    from atlas_b200.layer_norm import layer_norm
    x, res, w, b, dy, dh = _make((9, 3, 40), (3, 40), F32)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w, b)]
    y, h = layer_norm(leaves[0], leaves[2], leaves[3], 1e-3, leaves[1])
    ((y * dy).sum() + (h * dh).sum()).backward()
    base = [t.cpu().double() for t in (x, res, w, b)]

    def loss(t):
        s = t[0] + t[1]
        return float((R.layer_norm(s, t[2], t[3], 1e-3) * dy.cpu().double()).sum() + (s * dh.cpu().double()).sum())
    gen = torch.Generator().manual_seed(4)
    for i, p in enumerate(leaves):
        d = torch.randn(p.shape, generator=gen, dtype=torch.float64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        want = (loss(up) - loss(dn)) / 2e-5
        grad = p.grad.cpu().double()
        assert abs(float((grad * d).sum()) - want) < 1e-5 * float(grad.norm() * d.norm()), i


def test_empty_and_other_stream_and_determinism():
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    w = torch.ones(64, device="cuda")
    e = torch.empty(0, 64, device="cuda")
    y, h, st = layer_norm_forward(e, w, w)
    dx, dw, db = layer_norm_backward(e, h, w, st)
    assert y.shape == e.shape and dx.shape == e.shape and (dw == 0).all() and (db == 0).all()
    x, _, w, b, dy, _ = _make((3000, 768), (768,), BF)
    y, h, st = layer_norm_forward(x, w, b)
    a = layer_norm_backward(dy, h, w, st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = layer_norm_backward(dy, h, w, st)
    side.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(a, c))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are normalised as the same rows alone are."""
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    N = 1024
    rows = (1 << 21) + 3
    x = torch.zeros(rows, N, dtype=BF, device="cuda")
    tail, _, w, b, dy, _ = _make((5, N), (N,), BF)
    x[-5:] = tail
    y, h, st = layer_norm_forward(x, w, b)
    y2, _, st2 = layer_norm_forward(tail, w, b)
    assert torch.equal(y[-5:], y2) and torch.equal(st[-5:], st2)
    del y
    d = torch.zeros_like(x)
    d[-5:] = dy
    dx, dw, db = layer_norm_backward(d, h, w, st)
    dx2, dw2, db2 = layer_norm_backward(dy, tail, w, st2)
    assert torch.equal(dx[-5:], dx2) and R.rel(dw, dw2) < 2e-6 and R.rel(db, db2) < 2e-6


def test_refusals():
    from atlas_b200 import AtlasError
    from atlas_b200.layer_norm import layer_norm_backward, layer_norm_forward
    x, res, w, b, dy, _ = _make((6, 4, 64), (4, 64), BF)
    for bad in ((x.half(), w, b), (x, w.double(), b), (x, w[:2], b), (x, w, b[0]), (x.cpu(), w, b), (x, w.t(), b)):
        with pytest.raises(ValueError):
            layer_norm_forward(*bad)
    with pytest.raises(ValueError):
        layer_norm_forward(x, w, b, residual=res.float())
    with pytest.raises(AtlasError):
        layer_norm_forward(x, w, b, eps=-1.0)
    with pytest.raises(AtlasError):
        layer_norm_forward(torch.zeros(1, (1 << 20) + 1, device="cuda"))
    _, h, st = layer_norm_forward(x, w, b)
    with pytest.raises(ValueError):
        layer_norm_backward(dy[:3], h, w, st)
    with pytest.raises(ValueError):
        layer_norm_backward(dy, h, w, st[:3])
