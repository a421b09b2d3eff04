"""A pre-norm token mixer over decay attention: the cheap recurrent branch that a hybrid
puts next to an Atlas memory layer or a sliding-window attention layer.

    h = x + delta;  n = layer_norm(h);  q, k, v = n W_qkv
    a = decay attention of q, k, v;  out = layer_norm per head(a) W_out

``delta`` is the output of the block before, so the residual add of the stream rides in
the norm.  Training and prompts take whole sequences (``forward``); generation advances a
pool of states by one token per running sequence (``step``).  The norms and the attention
run in libatlas_scan.so, the two projections are plain GEMMs.

For bf16 activations cast the projections (``to_qkv``, ``to_out``), not the block: the decay
logits and the norms' weights are used in float32, and a logit rounded to bf16 moves a
decay of 1 - 2^-10 by up to 2 % of its distance from 1."""

import torch
import torch.nn as nn

from .decay_attention import decay_attention, decay_attention_step
from .layer_norm import layer_norm


class DecayMixer(nn.Module):
    def __init__(self, n_embd, n_head, dim_head=None, eps=1e-5):
        super().__init__()
        D = dim_head if dim_head is not None else n_embd // n_head
        self.n_head, self.dim_head, self.eps = n_head, D, eps
        self.norm_weight, self.norm_bias = nn.Parameter(torch.ones(n_embd)), nn.Parameter(torch.zeros(n_embd))
        self.to_qkv = nn.Linear(n_embd, 3 * n_head * D, bias=False)
        # decays 1 - 2^-4 .. 1 - 2^-10 over the heads, learned as a logit
        self.decay_logit = nn.Parameter(torch.log(torch.exp2(torch.linspace(4, 10, n_head)) - 1))
        self.head_weight, self.head_bias = nn.Parameter(torch.ones(n_head, D)), nn.Parameter(torch.zeros(n_head, D))
        self.to_out = nn.Linear(n_head * D, n_embd, bias=False)

    def _qkv(self, x, delta):
        B, T, _ = x.shape
        if delta is None:
            n, h = layer_norm(x, self.norm_weight.float(), self.norm_bias.float(), self.eps), x
        else:
            n, h = layer_norm(x, self.norm_weight.float(), self.norm_bias.float(), self.eps, residual=delta)
        qkv = (n @ self.to_qkv.weight.to(n.dtype).t()).view(B, T, 3, self.n_head, self.dim_head)
        return qkv.unbind(2), h

    def _out(self, a):
        B, T, H, D = a.shape
        a = layer_norm(a, self.head_weight.float(), self.head_bias.float(), self.eps)
        return a.reshape(B, T, H * D) @ self.to_out.weight.to(a.dtype).t()

    def log_decay(self):
        return nn.functional.logsigmoid(self.decay_logit.float())

    def forward(self, x, delta=None, state=None):
        """x, delta: (B, T, n_embd); state (B, H, D, D) float32 or None.
        Returns (out, h, state): the stream goes on as h, with out as the next delta."""
        (q, k, v), h = self._qkv(x, delta)
        a, state = decay_attention(q, k, v, self.log_decay(), state)
        return self._out(a), h, state

    @torch.no_grad()
    def step(self, x, state, slots=None, delta=None):
        """One generation step: x (B, T, n_embd) with T usually 1; state is advanced in place
        (see decay_attention_step).  Returns (out, h)."""
        (q, k, v), h = self._qkv(x, delta)
        a, _ = decay_attention_step(q, k, v, self.log_decay(), state, slots)
        return self._out(a), h
