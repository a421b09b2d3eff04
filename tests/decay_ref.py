"""float64 restatements of decay attention (token by token) and layer norm, for autograd
checks of the kernels (test infrastructure)."""
import torch


def decay_attention(q, k, v, log_decay, state, scale):
    """(B, T, H, D) float64 -> (y, state)."""
    B, T, H, D = q.shape
    S = torch.zeros(B, H, D, D, dtype=torch.float64) if state is None else state
    lam = torch.exp(log_decay)[None, :, None, None]
    ys = []
    for t in range(T):
        S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        ys.append(scale * (q[:, t, :, None, :] @ S)[..., 0, :])
    y = torch.stack(ys, 1) if ys else torch.zeros_like(q)
    return y, S


def layer_norm(x, weight, bias, eps):
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    z = (x - mean) / torch.sqrt(var + eps)
    if weight is not None:
        z = z * weight
    return z if bias is None else z + bias


def rel(a, b):
    """Frobenius distance over the reference's norm."""
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    n = b.norm()
    return float((a - b).norm() / n) if n > 0 else float((a - b).norm())
