"""Plain float64 restatement of the attention operators, row by row (test infrastructure only)."""

import math

import torch


def pairs(rot, interleaved):
    """Indexes of the two members of each rotated pair."""
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def norm_rope(x, cos, sin, weight=None, eps=1e-6, interleaved=False):
    """x [..., H, D]; cos, sin [..., R/2] of each token."""
    x = x.double()
    u = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        u = u * weight.double()
    a, b = pairs(2 * cos.shape[-1], interleaved)
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    y = u.clone()
    y[..., a] = u[..., a] * c - u[..., b] * s
    y[..., b] = u[..., b] * c + u[..., a] * s
    return y


def norm_rope_backward(x, dy, cos, sin, weight=None, eps=1e-6, interleaved=False):
    """(dx, dweight) by the formula."""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    a, b = pairs(2 * cos.shape[-1], interleaved)
    c, s = cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    du = dy.clone()
    du[..., a] = dy[..., a] * c + dy[..., b] * s
    du[..., b] = dy[..., b] * c - dy[..., a] * s
    dw = (du * x * r).reshape(-1, x.shape[-1]).sum(0)
    return r * (w * du - x * r * r * (w * du * x).mean(-1, keepdim=True)), dw


def paged_attention(q, k_cache, v_cache, table, kv_lens, q_lens, window=0, scale=None):
    """(o, lse, A) in float64 with A = sum_j p_j |v_j|, the scale of what rounding the weights can change."""
    heads, dim = q.shape[1:]
    group, page = heads // k_cache.shape[2], k_cache.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    t = 0
    for n, (count, length) in enumerate(zip(q_lens, kv_lens)):
        for i in range(count):
            pos = length - count + i
            first = max(0, pos - window + 1) if window else 0
            if pos >= 0:
                key = torch.arange(first, pos + 1)
                at = table[n].long()[key // page], key % page
                k, v = (c[at].double().repeat_interleave(group, 1) for c in (k_cache, v_cache))
                logits = torch.einsum("hd,khd->hk", q[t].double(), k) * scale
                top = logits.amax(-1, keepdim=True)
                p = torch.exp(logits - top)
                total = p.sum(-1, keepdim=True)
                p = p / total
                o[t] = torch.einsum("hk,khd->hd", p, v)
                size[t] = torch.einsum("hk,khd->hd", p, v.abs())
                lse[t] = (top + total.log())[:, 0]
            t += 1
    return o, lse, size
