"""Training a model that mixes KDA layers with attention layers, and serving what was trained.

    python examples/hybrid_training.py

Whole sequences go forward and back: the KDA layers through their chunked kernels, the attention layers' queries and keys through
`qk_norm_rope`; the attention itself, which the package has for serving only, is written out in torch.  The trained model then serves
the same sequences from its caches (hybrid_serving.py), and both must say the same.
"""

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from hybrid_serving import Hybrid, serve  # noqa: E402

from experiment_swa_kda_b200 import qk_norm_rope  # noqa: E402


def attention(layer, x):
    """A `PagedAttention` layer over whole sequences x [B,T,hidden], differentiable."""
    T, heads, kv_heads = x.shape[1], layer.num_heads, layer.num_kv_heads
    q, k, v = layer.qkv_proj(x).unflatten(-1, (-1, layer.head_dim)).split((heads, kv_heads, kv_heads), 2)
    q, k = qk_norm_rope(q, k, layer.cos, layer.sin, q_weight=layer.q_norm, k_weight=layer.k_norm, eps=layer.norm_eps)
    k, v = (t.repeat_interleave(heads // kv_heads, 2) for t in (k, v))
    at = torch.arange(T, device=x.device)
    hidden = at[None, :] > at[:, None]
    if layer.window:
        hidden = hidden | (at[None, :] <= at[:, None] - layer.window)
    scores = torch.einsum("bihd,bjhd->bhij", q, k).float() * layer.head_dim ** -0.5
    p = scores.masked_fill(hidden, float("-inf")).softmax(-1).to(v.dtype)
    return layer.o_proj(torch.einsum("bhij,bjhd->bihd", p, v).flatten(2))


def forward(model, x):
    """x [B,T,hidden] through a `Hybrid`, differentiable."""
    for layer, kind in zip(model.layers, model.pattern):
        y = F.rms_norm(x, x.shape[-1:])
        x = x + (layer(y)[0] if kind == "K" else attention(layer, y))
    return x


def train(model, x, target, steps, lr=1e-3):
    """The loss of each step."""
    optimizer = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        loss = (forward(model, x).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main(tokens=200, sequences=2, steps=20, device="cuda:0"):
    torch.manual_seed(0)
    model = Hybrid().to(device)
    x = torch.randn(sequences, tokens, 512, device=device).bfloat16()
    target = x.float().roll(3, 1)      # the token three places before
    losses = train(model, x, target, steps)
    with torch.no_grad():
        whole = forward(model, x)
    served = serve(model, x, [64, 100] + [1] * (tokens - 164))
    off = ((served - whole).float().norm() / whole.float().norm()).item()
    print(f"{steps} steps: loss {losses[0]:.3f} to {losses[-1]:.3f}; served in chunks and single tokens, the trained model is {off:.1e} from its training form")
    return losses, off


if __name__ == "__main__":
    main()
