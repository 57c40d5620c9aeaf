"""Serving a model that mixes KDA layers with sliding-window and full attention: a prompt in chunks, then token by token.

    python examples/hybrid_serving.py

The KDA layers carry their fixed-size state, the attention layers their pages; both are handed in by the caller and updated as
the sequences grow.  Prints how far the pieces are from the whole prompt in one call.
"""

import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from experiment_swa_kda_b200 import KDAState, KimiDeltaAttention, PagedAttention, PagedCache  # noqa: E402


class Hybrid(nn.Module):
    """Residual blocks of mixers: "K" a KDA layer, "S" a sliding-window, "L" a full attention layer."""

    def __init__(self, pattern="KSKL", hidden_size=512, num_heads=4, num_kv_heads=2, head_dim=128, window=64, max_positions=4096):
        super().__init__()
        self.pattern = pattern
        self.shape = (num_heads, num_kv_heads, head_dim)
        self.layers = nn.ModuleList(
            KimiDeltaAttention(hidden_size, num_heads, head_dim) if kind == "K" else
            PagedAttention(hidden_size, num_heads, num_kv_heads, head_dim, window if kind == "S" else 0, max_positions) for kind in pattern)

    def states(self, sequences, max_len, device, page_size=16):
        heads, kv_heads, dim = self.shape
        return [KDAState.zeros(sequences, heads, dim, 4, device) if kind == "K" else PagedCache.zeros(sequences, max_len, page_size, kv_heads, dim, device)
                for kind in self.pattern]

    @torch.no_grad()
    def forward(self, x, states):
        """x [B,T,hidden], the next T tokens of every sequence; `states` move on by as many."""
        for i, (layer, kind) in enumerate(zip(self.layers, self.pattern)):
            y = F.rms_norm(x, x.shape[-1:])
            if kind != "K":
                states[i].kv_lens += x.shape[1]
                y = layer(y, states[i])
            elif x.shape[1] == 1:
                y = layer.decode_token(y, states[i])
            else:
                y, states[i] = layer(y, states[i], output_final_state=True)
            x = x + y
        return x


def serve(model, x, chunks):
    """x [B,T,hidden] through the model in pieces of the lengths given."""
    states = model.states(x.shape[0], x.shape[1], x.device)
    return torch.cat([model(piece, states) for piece in x.split(chunks, 1)], 1)


def main(tokens=200, sequences=2, device="cuda:0"):
    torch.manual_seed(0)
    model = Hybrid().to(device)
    x = torch.randn(sequences, tokens, 512, device=device).bfloat16()
    whole = serve(model, x, [tokens])
    pieces = serve(model, x, [64, 100] + [1] * (tokens - 164))
    off = ((pieces - whole).float().norm() / whole.float().norm()).item()
    print(f"{sequences} sequences of {tokens} tokens: chunks of 64 and 100, then {tokens - 164} single tokens, are {off:.1e} from one call")
    return off


if __name__ == "__main__":
    main()
