"""Attention operators where a caller leaves the plain path: saved-tensor hooks, padding, windows and values of any size, errors.

Bounds are those of test_attention_gpu.py."""

import contextlib

import pytest
import torch

from test_attention_gpu import BF16, DEV, F32, tables

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- norm + rotation, backward

def slices_of_a_projection(B, T, Hq, Hk, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, T, (Hq + 2 * Hk) * D, generator=gen).to(dtype).to(DEV)
    q, k = qkv[..., :Hq * D].unflatten(-1, (Hq, D)), qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
    dy = [torch.randn(B, T, h, D, generator=gen).to(dtype).to(DEV) for h in (Hq, Hk)]
    return q.detach(), k.detach(), dy


@pytest.mark.parametrize("B,T,Hq,Hk,D,R,dtype", [(2, 33, 4, 2, 64, 64, BF16), (1, 129, 3, 3, 128, 64, BF16), (2, 19, 5, 1, 34, 20, F32), (3, 1, 2, 2, 96, 96, F32)])
@pytest.mark.parametrize("hook", ["offloaded", "cloned", "stretched"])
def test_gradients_under_saved_tensor_hooks(B, T, Hq, Hk, D, R, dtype, hook):
    """What a hook hands back has the sizes of what it was given, and strides of its own."""
    import experiment_swa_kda_b200 as m
    q, k, dy = slices_of_a_projection(B, T, Hq, Hk, D, dtype, T)
    cos, sin = (t.to(DEV) for t in tables(T + 9, R))
    pos = torch.randint(0, T + 9, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    weights = [(1 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(2))).to(DEV) for _ in range(2)]

    def stretched(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 8, device=t.device, dtype=t.dtype)[..., :t.shape[-1]]
        return wide.copy_(t)

    def gradients(context):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, *weights)]
        with context:
            y = m.qk_norm_rope(leaves[0], leaves[1], cos, sin, positions=pos, q_weight=leaves[2], k_weight=leaves[3])
        return torch.autograd.grad(y, leaves, dy)

    hooks = {"offloaded": lambda: torch.autograd.graph.save_on_cpu(), "cloned": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone()),
             "stretched": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, stretched)}
    plain = gradients(contextlib.nullcontext())
    for got, want in zip(gradients(hooks[hook]()), plain):
        assert torch.equal(got, want)      # the same kernel on the same values


def test_a_hook_that_changes_a_saved_tensor_is_refused():
    import experiment_swa_kda_b200 as m
    q, k, dy = slices_of_a_projection(2, 33, 4, 2, 64, BF16, 3)
    cos, sin = (t.to(DEV) for t in tables(33, 64))
    for change in (lambda t: t[:, :-1] if t.ndim == 4 else t, lambda t: t.float() if t.ndim == 4 else t, lambda t: t[:-1] if t.ndim == 2 else t):
        x = q.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y, _ = m.qk_norm_rope(x, k, cos, sin)
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            torch.autograd.grad(y, x, dy[0])
