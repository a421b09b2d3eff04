"""Cases, plain forms and exact values of the token-mixing operators next to the Atlas memory scan.

Operators (heads h, tokens t, activations (B, T, H, D), states (B, H, D, D) float32):

  decay attention   S_t = l_h S_{t-1} + k_t v_t^T,   y_t = scale q_t^T S_t,   l_h = exp(log_decay_h)
                    "prompt": a whole sequence forward, with the state that it leaves
                    "train":  forward, then the gradients of q, k, v, log_decay and the entry state
                    "step":   one or a few tokens per sequence on a pool of states
  layer norm        h = x + residual (kept in the activations' type), y = (h - mean) / sqrt(var + eps) w + b
                    "norm":   forward; with "train" also dx, dw and db

``run`` computes them in float32 with elementary torch operations where ``own`` is false and through
``atlas_b200`` where it is true.  ``exact`` is the token-by-token definition in float64.
"""

import math
import os
import sys

import torch

own = False
CHUNK = 128  # tokens that the plain form handles as one dense block
EPS = 1e-5


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the 170M model's layer on a full training-length prompt: 8 sequences of 8192, 12 heads of 64
        dict(name="prompt 8x8192x12x64", op="prompt", B=8, T=8192, H=12, D=64, dtype="bf16", state=False, fused=True),
        # one long document with head_dim 128 continued from an earlier state: the long-context sweep's smallest chain count
        dict(name="prompt 1x65536x16x128", op="prompt", B=1, T=65536, H=16, D=128, dtype="bf16", state=True, fused=False),
        # a few short prompts of odd length as a server admits them, with carried states
        dict(name="prompt 3x777x12x64", op="prompt", B=3, T=777, H=12, D=64, dtype="bf16", state=True, fused=True),
        # the CPU-sized float32 layer (4 heads of 32, 512 tokens): checks and small experiments
        dict(name="prompt 2x512x4x32 f32", op="prompt", B=2, T=512, H=4, D=32, dtype="f32", state=False, fused=True),
        # the 59M model's training step of one layer: 16 sequences of 4096, 8 heads of 64
        dict(name="train 16x4096x8x64", op="train", B=16, T=4096, H=8, D=64, dtype="bf16", state=False, fused=True),
        # head_dim 128 with a ragged last chunk and a learned entry state
        dict(name="train 4x1900x6x128", op="train", B=4, T=1900, H=6, D=128, dtype="bf16", state=True, fused=False),
        # float32 training at an unusual head size (384 channels in 8 heads of 48)
        dict(name="train 2x500x8x48 f32", op="train", B=2, T=500, H=8, D=48, dtype="f32", state=True, fused=True),
        # one sequence being generated: pure latency
        dict(name="step 1x12x64", op="step", B=1, T=1, H=12, D=64, dtype="bf16"),
        # a full decoding batch of the 170M model on a pool of state slots
        dict(name="step 256x12x64", op="step", B=256, T=1, H=12, D=64, dtype="bf16"),
        # the training step's pre-norm over the residual stream: 8 x 8192 rows of 768
        dict(name="norm 65536x768 train", op="norm", rows=65536, G=1, N=768, dtype="bf16", residual=True, train=True),
        # the per-head norm of the attention's output, a weight for each of 12 heads of 64
        dict(name="norm 16384x12x64 train", op="norm", rows=16384, G=12, N=64, dtype="bf16", residual=False, train=True),
        # the pre-norm of a small decoding batch, float32
        dict(name="norm 64x768 f32", op="norm", rows=64, G=1, N=768, dtype="f32", residual=True, train=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _odd_one_out(n):
    return n + 1 if n == 3072 else n


def _heads(rng, D):
    return rng.choice([4, 6, 8, 12] if D != 128 else [4, 6, 12])


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "step", "norm", "norm"])
    if op == "norm":
        G = rng.choice([1, 1, 1, 4, 8, 12])
        N = rng.choice([32, 48, 64, 128]) if G > 1 else _odd_one_out(_log_int(rng, 32, 6000))
        dtype = rng.choice(["bf16", "bf16", "f32"])
        rows = max(1, min(_log_int(rng, 1, 65536), (50_000_000 if dtype == "bf16" else 25_000_000) // (G * N)))
        return dict(op=op, rows=rows, G=G, N=N, dtype=dtype,
                    residual=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "step":
        D = rng.choice([32, 48, 64, 64, 128])
        H = _heads(rng, D)
        return dict(op=op, B=max(1, min(_log_int(rng, 1, 512), 50_000_000 // (H * D * D))), T=rng.choice([1, 1, 1, 2, 5]),
                    H=H, D=D, dtype=rng.choice(["bf16", "bf16", "f32"]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    D = rng.choice([64, 64, 128, 32, 96])
    H = _heads(rng, D)
    most = (30_000_000 if dtype == "bf16" else 3_000_000) // (2 if op == "train" else 1)
    T = _odd_one_out(_log_int(rng, 1, 16384))
    B = max(1, min(_log_int(rng, 1, 16), most // (T * H * D)))
    return dict(op=op, B=B, T=T, H=H, D=D, dtype=dtype, state=rng.random() < 0.5, fused=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _norm_inputs(case, gen):
    dt, G, N = _dtype(case), case["G"], case["N"]
    shape = (case["rows"], G, N) if G > 1 else (case["rows"], N)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    s = dict(case=case, x=(0.5 + 1.5 * rn(*shape)).to(dt), weight=1 + 0.2 * rn(G, N), bias=0.1 * rn(G, N))
    if G == 1:
        s["weight"], s["bias"] = s["weight"][0].clone(), s["bias"][0].clone()
    s["residual"] = rn(*shape).to(dt) if case["residual"] else None
    if case["train"]:
        s["dy"] = rn(*shape).to(dt)
        s["dh"] = rn(*shape).to(dt) if case["residual"] else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    if case["op"] == "norm":
        return _norm_inputs(case, gen)
    B, T, H, D, dt = case["B"], case["T"], case["H"], case["D"], _dtype(case)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)              # noqa: E731
    q, k, v = (unit(rn(B, T, H, D)) for _ in range(3))
    if case.get("fused", True):  # views of one projection's output, as a layer has them
        proj = torch.stack([q, k, v], 2).to(dt)
        q, k, v = proj.unbind(2)
    else:
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    # decays between about 1 - 2^-4 and 1 - 2^-10, one for each head
    e = torch.linspace(4, 10, H, device="cuda") + 0.2 * rn(H)
    s = dict(case=case, q=q, k=k, v=v, log_decay=torch.log1p(-torch.exp2(-e)), scale=D ** -0.5)
    if case["op"] == "step":
        n = B + B // 4 + 1  # more slots than running sequences
        s["pool"] = 0.3 * rn(n, H, D, D)
        s["slots"] = torch.randperm(n, device="cuda", generator=gen)[:B].to(torch.int32)
        s["out"] = s["pool"].clone()  # the states after the step, beside those before it
        return s
    s["state"] = 0.3 * rn(B, H, D, D) if case["state"] else None
    if case["op"] == "train":
        s["dy"] = rn(B, T, H, D).to(dt)
        s["dstate"] = 0.05 * rn(B, H, D, D) if case["state"] else None
    return s


# ---------------------------------------------------------------------------------------------
# plain forms: float32, elementary operations
# ---------------------------------------------------------------------------------------------
def _blocks(x, C):
    """(B, T, H, D) -> float32 (B, H, n, C, D); zero tokens fill up the FIRST block, so the last ends at T."""
    B, T, H, D = x.shape
    n = -(-T // C)
    full = x.new_zeros(B, n * C, H, D, dtype=torch.float32)
    full[:, n * C - T:] = x
    return full.reshape(B, n, C, H, D).permute(0, 3, 1, 2, 4)


def _tokens(x, T):
    """The inverse of _blocks."""
    B, H, n, C, D = x.shape
    return x.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, D)[:, n * C - T:]


def _decays(g, T, n, C):
    """Powers of the decay: within a block, into and out of it, from block to block, and from the entry state."""
    i = torch.arange(C, device=g.device, dtype=torch.float32)
    c = torch.arange(n, device=g.device, dtype=torch.float32)
    gh = g[:, None]
    lag = i[:, None] - i[None, :]
    within = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), torch.zeros(()).to(g))
    into, out = torch.exp(gh * (i + 1)), torch.exp(gh * (C - 1 - i))
    hop = c[:, None] - 1 - c[None, :]
    between = torch.where(hop >= 0, torch.exp(g[:, None, None] * C * hop.clamp(min=0)), torch.zeros(()).to(g))
    left = torch.exp(gh * C * (n - 1 - c))          # from the end of a block to the end of the sequence
    entry = torch.exp(gh * (torch.arange(T, device=g.device, dtype=torch.float32) + 1))
    return lag, i, within[None, :, None], into[None, :, None, :, None], out[None, :, None, :, None], between, left, entry


def _along_blocks(mat, x):
    """x (B, H, n, D, D) -> sum over blocks with weights mat (H, n, n)."""
    B, H, n, D, _ = x.shape
    return (mat @ x.reshape(B, H, n, D * D)).reshape(x.shape)


def _plain_attention(s):
    q, k, v, g, scale, S0 = s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"]
    T, C = q.shape[1], min(CHUNK, q.shape[1])
    Q, K, V = (_blocks(x, C) for x in (q, k, v))
    n = Q.shape[2]
    lag, i, within, into, out, between, left, entry = _decays(g, T, n, C)
    P = (Q @ K.transpose(-1, -2)) * within
    dS = (K * out).transpose(-1, -2) @ V            # what a block adds to the state at its end
    S_in = _along_blocks(between, dS)               # the state entering a block, entry state apart
    y = _tokens(P @ V + into * (Q @ S_in), T)
    S = (left[None, :, :, None, None] * dS).sum(2)
    if S0 is not None:
        y = y + entry.t()[None, :, :, None] * torch.einsum("bthd,bhde->bthe", q.float(), S0)
        S = S + torch.exp(g * T)[None, :, None, None] * S0
    y = (scale * y).to(q.dtype)
    if s["case"]["op"] == "prompt":
        return {"y": y, "state": S}
    dO = scale * _blocks(s["dy"], C)
    dP = dO @ V.transpose(-1, -2)
    A = dP * within
    QY = (Q * into).transpose(-1, -2) @ dO
    dS_out = _along_blocks(between.transpose(-1, -2), QY)  # gradient of the state leaving a block
    if s["dstate"] is not None:
        dS_out = dS_out + left[None, :, :, None, None] * s["dstate"][:, :, None]
    q_in, k_out = into * (dO @ S_in.transpose(-1, -2)), out * (V @ dS_out.transpose(-1, -2))
    dq = _tokens(A @ K + q_in, T)
    dk = _tokens(A.transpose(-1, -2) @ Q + k_out, T)
    dv = _tokens(P.transpose(-1, -2) @ dO + out * (K @ dS_out), T)
    dg = (lag * P * dP).sum((0, 2, 3, 4)) + ((i + 1)[:, None] * Q * q_in).sum((0, 2, 3, 4)) \
        + ((C - 1 - i)[:, None] * K * k_out).sum((0, 2, 3, 4)) \
        + C * torch.exp(g * C) * (dS_out * S_in).sum((0, 2, 3, 4))
    got = {"y": y, "state": S}
    if S0 is not None:
        do = scale * s["dy"].float()
        d0 = entry.t()[None, :, :, None] * torch.einsum("bthe,bhde->bthd", do, S0)
        dq = dq + d0
        steps = torch.arange(1, T + 1, device=g.device, dtype=torch.float32)
        dS0 = torch.einsum("bthd,bthe->bhde", entry.t()[None, :, :, None] * q.float(), do)
        dg = dg + (steps[None, :, None, None] * q.float() * d0).sum((0, 1, 3))
        if s["dstate"] is not None:
            far = torch.exp(g * T)
            dS0 = dS0 + far[None, :, None, None] * s["dstate"]
            dg = dg + T * far * (s["dstate"] * S0).sum((0, 2, 3))
        got["dstate"] = dS0
    return {**got, "dq": dq.to(q.dtype), "dk": dk.to(q.dtype), "dv": dv.to(q.dtype), "dlog_decay": dg}


def _plain_step(s):
    q, k, v, g = s["q"].float(), s["k"].float(), s["v"].float(), s["log_decay"]
    T = q.shape[1]
    rows = s["slots"].long()
    S0 = s["pool"][rows]
    i = torch.arange(T, device=g.device, dtype=torch.float32)
    lag = i[:, None] - i[None, :]
    within = torch.where(lag >= 0, torch.exp(g[:, None, None] * lag.clamp(min=0)), torch.zeros(()).to(g))
    P = torch.einsum("bthd,bshd->bhts", q, k) * within
    y = torch.einsum("bhts,bshe->bthe", P, v)
    y = y + torch.exp(g[None, :] * (i + 1)[:, None])[None, :, :, None] * torch.einsum("bthd,bhde->bthe", q, S0)
    kw = k * torch.exp(g[None, :] * (T - 1 - i)[:, None])[None, :, :, None]
    S = torch.exp(g * T)[None, :, None, None] * S0 + torch.einsum("bthd,bthe->bhde", kw, v)
    s["out"].index_copy_(0, rows, S)
    return {"y": (s["scale"] * y).to(s["q"].dtype), "state": s["out"]}


def _plain_norm(s):
    x, dt = s["x"], s["x"].dtype
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(dt)
    hf = h.float()
    c = hf - hf.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * rstd
    got = {"y": (n * s["weight"] + s["bias"]).to(dt)}
    if s["residual"] is not None:
        got["h"] = h
    if s["case"]["train"]:
        dy = s["dy"].float()
        dn = dy * s["weight"]
        dx = rstd * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        got.update(dx=dx.to(dt), dweight=(dy * n).sum(0), dbias=dy.sum(0))
    return got


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
def _framework():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atlas-jax_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from atlas_b200 import decay_attention, layer_norm
    return decay_attention, layer_norm


def _own(s):
    DA, LN = _framework()
    op = s["case"]["op"]
    if op == "norm":
        y, h, stats = LN.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS, s["residual"])
        got = {"y": y} if s["residual"] is None else {"y": y, "h": h}
        if s["case"]["train"]:
            got["dx"], got["dweight"], got["dbias"] = LN.layer_norm_backward(s["dy"], h, s["weight"], stats, s["dh"])
        return got
    q, k, v, g, scale = s["q"], s["k"], s["v"], s["log_decay"], s["scale"]
    if op == "step":
        y, state = DA.decay_attention_step(q, k, v, g, s["pool"], slots=s["slots"], scale=scale, out=s["out"])
        return {"y": y, "state": state}
    y, state, saved = DA.decay_attention_forward(q, k, v, g, s["state"], scale=scale, need_saved=op == "train")
    got = {"y": y, "state": state}
    if op == "train":
        dq, dk, dv, dg, dstate = DA.decay_attention_backward(q, k, v, g, saved, s["dy"], s["dstate"], scale=scale)
        got.update(dq=dq, dk=dk, dv=dv, dlog_decay=dg)
        if s["state"] is not None:
            got["dstate"] = dstate
    return got


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_norm(state) if op == "norm" else _plain_step(state) if op == "step" else _plain_attention(state)


# ---------------------------------------------------------------------------------------------
# least work
# ---------------------------------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n = case["rows"] * case["G"] * case["N"]
        moved = 2 + 2 * case["residual"]
        if case["train"]:
            moved += 2 + case["residual"]  # dy (and dh) in, dx out; h is the forward's own
        par = case["G"] * case["N"] * 4
        return {"bytes": moved * n * es + par * (4 if case["train"] else 2), "flops": n * (22 if case["train"] else 9)}
    n = case["B"] * case["T"] * case["H"]
    D = case["D"]
    state = case["B"] * case["H"] * D * D * 4
    if case["op"] == "step":
        return {"bytes": 4 * n * D * es + 2 * state, "flops": 4 * n * D * D}
    if case["op"] == "prompt":
        return {"bytes": 4 * n * D * es + (2 if case["state"] else 1) * state, "flops": 4 * n * D * D}
    return {"bytes": 8 * n * D * es + (4 if case["state"] else 1) * state, "flops": 12 * n * D * D}


# ---------------------------------------------------------------------------------------------
# exact values: the definition, token by token, in float64
# ---------------------------------------------------------------------------------------------
def _exact_attention(s, S0, dS):
    q, k, v, g, scale = s["q"].double(), s["k"].double(), s["v"].double(), s["log_decay"].double(), s["scale"]
    B, T, H, D = q.shape
    lam = torch.exp(g)[None, :, None, None]
    S = torch.zeros(B, H, D, D, dtype=torch.float64, device=q.device) if S0 is None else S0.double().clone()
    train = s["case"]["op"] == "train"
    do = scale * s["dy"].double() if train else None
    y, dq = torch.empty_like(q), torch.empty_like(q)
    dk, dv = torch.empty_like(q), torch.empty_like(q)
    G = torch.zeros_like(S)          # dS_t / dlog_decay
    dg = torch.zeros_like(S)
    for t in range(T):
        if train:
            G = lam * (G + S)
            dg += G * (q[:, t, :, :, None] * do[:, t, :, None, :])
        S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        y[:, t] = scale * (q[:, t, :, None, :] @ S)[..., 0, :]
        if train:
            dq[:, t] = (S @ do[:, t, :, :, None])[..., 0]
    got = {"y": y, "state": S}
    if not train:
        return got
    R = torch.zeros_like(S) if dS is None else dS.double().clone()  # gradient of S_t from the tokens after t
    dg += G * R
    for t in range(T - 1, -1, -1):
        R = R + q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = (R @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ R)[..., 0, :]
        R = lam * R
    got.update(dq=dq, dk=dk, dv=dv, dlog_decay=dg.sum((0, 2, 3)))
    if S0 is not None:
        got["dstate"] = R
    return got


def exact(case, seed):
    if case.get("T", 0) > 100_000:
        return None
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
        got = {}
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(s["x"].dtype).double()
            got["h"] = x
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        z = (x - mean) * (var + EPS) ** -0.5
        got["y"] = z * w + b
        if case["train"]:
            dy = s["dy"].double()
            got["dbias"], got["dweight"] = dy.sum(0), torch.einsum("r...,r...->...", dy, z)
            u = dy * w
            u = u - (u.mean(-1, keepdim=True) + z * (u * z).sum(-1, keepdim=True) / case["N"])
            got["dx"] = u * (var + EPS) ** -0.5
            if s["dh"] is not None:
                got["dx"] = got["dx"] + s["dh"].double()
        return got
    if case["op"] == "step":
        rows = s["slots"].long()
        got = _exact_attention(s, s["pool"][rows], None)
        pool = s["pool"].double()
        pool[rows] = got["state"]
        return {"y": got["y"], "state": pool}
    return _exact_attention(s, s["state"], s.get("dstate"))
