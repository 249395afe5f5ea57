"""Linear attention over state slots on the CPU in float64 (oracle; test
infrastructure only): token by token from the definition, the math of
gated_delta_rule_decode and chunk_gated_delta_rule
(muserve/model/qwen35_layer_v2.py:286-295,351-358), the conv of a prompt
(:163-201) and the gated norm behind the layer."""
from __future__ import annotations

import torch

L2_EPS = 1e-6


def gates(g, beta, a_log=None, dt_bias=None):
    """(log decay, write strength or None) in float64 of what the caller hands over."""
    g = g.double()
    beta = None if beta is None else beta.double()
    if a_log is not None:
        g = -a_log.double().exp() * torch.logaddexp(g + dt_bias.double(), torch.zeros_like(g))
        beta = None if beta is None else torch.sigmoid(beta)
    return g, beta


def normed(x, qk_norm):
    x = x.double()
    return x / (x.square().sum(-1, keepdim=True) + L2_EPS).sqrt() if qk_norm else x


def scan(q, k, v, g, beta, state, scale, qk_norm=False, a_log=None, dt_bias=None):
    """One sequence: q, k [T, Hk, D], v [T, Hv, Dv], g, beta [T, Hv], state
    [Hv, Dv, D]. Returns (o [T, Hv, Dv], state, size [Hv]): size is the largest
    |S|_F + |u| of the walk, what rounding errors of the state scale with."""
    q, k, v = normed(q, qk_norm), normed(k, qk_norm), v.double()
    g, beta = gates(g, beta, a_log, dt_bias)
    group = v.shape[1] // k.shape[1]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    s = state.double().clone()
    out = torch.zeros(v.shape, dtype=torch.float64)
    size = s.flatten(1).norm(dim=1)
    for t in range(v.shape[0]):
        s = s * g[t].exp()[:, None, None]
        u = v[t]
        if beta is not None:
            u = beta[t][:, None] * (u - (s * k[t][:, None, :]).sum(-1))
        s = s + u[:, :, None] * k[t][:, None, :]
        out[t] = scale * (s * q[t][:, None, :]).sum(-1)
        size = torch.maximum(size, s.flatten(1).norm(dim=1) + u.norm(dim=1))
    return out, s, size


def gated_norm(x, z, weight, eps):
    x, z = x.double(), z.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double() \
        * z * torch.sigmoid(z)


def conv_prompt(conv, slot, x, weight):
    """One sequence's causal conv from slot `slot` of conv [slots, C, W] (updated
    in place): x [T, C], weight [C, 4] -> (out, sum of |tap products|) float64."""
    W = conv.shape[-1]
    if x.shape[0] == 0:
        return torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    past = torch.cat([conv[slot].t(), x])            # the last W inputs, then the rows
    taps = past[W - 3:].double().unfold(0, 4, 1) * weight.double()
    conv[slot] = past[past.shape[0] - W:].t()
    y = taps.sum(-1)
    return y * torch.sigmoid(y), taps.abs().sum(-1)
