"""Attention operators where a caller leaves the plain path: saved-tensor hooks, padding, windows and values of any size, errors.

Bounds are those of test_attention_gpu.py."""

import contextlib
import math

import pytest
import torch

from test_attention_gpu import BF16, DEV, F32, Batch, close, tables

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


# ---------------------------------------------------------------------------------------------- padding

def check_padding(b, o, lse, want, wlse, size):
    """o = 0 and lse = -inf, bit for bit, where a token is padding; the oracle's values elsewhere."""
    pad = torch.isinf(wlse)
    assert torch.equal(o.cpu()[pad], torch.zeros_like(o.cpu()[pad])) and bool((lse.cpu()[pad] == -math.inf).all())
    close(o.cpu()[~pad], want[~pad], size[~pad], b.dtype)
    assert ((lse.double().cpu() - wlse)[~pad].abs() <= 2e-5 * (1 + wlse[~pad].abs())).all()


@pytest.mark.parametrize("tokens,real", [(130, 0), (130, 1), (130, 90), (512, 0), (512, 1), (512, 90), (64, 20)])
@pytest.mark.parametrize("Hq,Hk,D", [(4, 1, 128), (16, 4, 64), (3, 1, 128), (12, 4, 96)])
@pytest.mark.parametrize("fill", [7.0, math.nan])
def test_row_tiles_of_padding_beside_live_ones(tokens, real, Hq, Hk, D, fill):
    """Whatever the queries of padding tokens hold, whole row tiles of them too, their outputs are 0, call after call."""
    b = Batch([tokens, 5, tokens], [real, 3, 0], Hq, Hk, D, 16, BF16, seed=real)
    pos = torch.cat([torch.arange(n - a, n) for a, n in zip(b.q_lens, b.kv_lens)])
    b.dq[(pos < 0).to(DEV)] = fill
    oracle = b.oracle()
    # also with a table that leaves room for long rows, which are then cut into parts
    wide = torch.cat((b.dtable, torch.full((3, 400), -7, dtype=torch.int32, device=DEV)), 1)
    for table in (b.dtable, wide):
        b.dtable = table
        for bound in (0, tokens):
            o, lse = b.attend(return_lse=True, max_q_len=bound)
            check_padding(b, o, lse, *(oracle[i] for i in (0, 1, 2)))
            for _ in range(20):
                assert torch.equal(o, b.attend(max_q_len=bound))


# ---------------------------------------------------------------------------------------------- windows

@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 40])
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hk", [([9], [3], 1, 1), ([4, 1, 3], [1, 500, 130], 4, 1), ([130, 40], [90, 500], 4, 1), ([300], [297], 6, 2)])
def test_windows_that_hide_nothing(window, dtype, q_lens, kv_lens, Hq, Hk):
    """The largest windows there are, padding or not, are the same as none."""
    b = Batch(q_lens, kv_lens, Hq, Hk, 128, 16, dtype)
    for bound in (0, max(q_lens)):
        o, lse = b.attend(return_lse=True, max_q_len=bound)
        b.window = window
        p, plse = b.attend(return_lse=True, max_q_len=bound)
        b.window = 0
        assert torch.equal(o, p) and torch.equal(lse, plse)


# ---------------------------------------------------------------------------------------------- values of any size

@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_len,Hq,D,window", [(4, 2, 128, 0), (200, 4, 128, 0), (200, 4, 64, 120), (60, 6, 96, 30)])
def test_hidden_keys_weigh_nothing(dtype, q_len, Hq, D, window):
    """The largest finite values at keys that a row does not see change no bit of its output."""
    kv = 300
    b = Batch([q_len], [kv], Hq, 2, D, 16, dtype, window=window)
    before = b.attend()
    hidden = torch.zeros(q_len, dtype=torch.bool)
    last, early = range(kv - min(q_len - 1, 20), kv), range(kv - q_len - window + 1, kv - q_len - window + 9) if window else ()
    for pos in (*last, *early):
        at = int(b.table[0, pos // 16]), pos % 16
        b.dv[at[0], at[1]] = torch.finfo(dtype).max
        b.dv[at[0], at[1], :, ::3] = torch.finfo(dtype).min
        i = torch.arange(q_len) + kv - q_len
        hidden |= (i >= pos) & ((i < pos + window) if window else True)
    assert not hidden.all()
    after = b.attend()
    assert torch.equal(before.cpu()[~hidden], after.cpu()[~hidden])
    assert not torch.equal(before.cpu()[hidden], after.cpu()[hidden])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_len,Hq,kv", [(1, 2, 6000), (3, 4, 3000), (70, 2, 5000)])
def test_values_that_are_not_finite_reach_rows_whose_weights_vanish(dtype, q_len, Hq, kv):
    """A visible NaN is in the sum however small its weight: keys hundreds of units below the others, in parts of their own."""
    b = Batch([q_len], [kv], Hq, 1, 128, 16, dtype)
    b.dq.fill_(1.0), b.q.fill_(1.0)
    for c in (b.k, b.dk):
        c[b.table[0, :20].long()] = -100.0      # keys 0 .. 319: scores of -100 sqrt(128)
    for c in (b.v, b.dv):
        c[int(b.table[0, 3]), 5, 0, 7] = math.nan
    o, want, size = b.attend(max_q_len=q_len), *b.oracle()[::2]
    assert torch.isnan(want[..., 7]).all() and torch.isfinite(want[..., 8]).all()
    close(o, want, size, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_lens,Hq,D,window", [([1, 1, 1], 2, 128, 0), ([1, 1, 1], 16, 64, 200), ([4, 2, 1], 4, 96, 0), ([150, 70, 3], 4, 128, 0)])
def test_infinite_values_that_are_seen(dtype, q_lens, Hq, D, window):
    """A visible infinite value is the row's sum, with its sign; two of opposite signs, or a NaN, make it NaN."""
    b = Batch(q_lens, [400, 333, 270], Hq, 1, D, 16, dtype, window=window)
    for n, pos, d, x in ((0, 330, 0, math.inf), (0, 341, 1, -math.inf), (1, 240, 2, math.inf), (1, 250, 2, -math.inf), (1, 240, 3, -math.inf), (1, 250, 3, -math.inf),
                         (2, 200, 4, math.nan), (2, 200, 5, math.inf)):
        at = int(b.table[n, pos // 16]), pos % 16
        for c in (b.v, b.dv):
            c[at[0], at[1], 0, d] = x
    o, want, size = b.attend(max_q_len=max(q_lens)), *b.oracle()[::2]
    last = [sum(q_lens[:n + 1]) - 1 for n in range(3)]      # the last tokens see all of them
    assert want[last[0], 0, :2].tolist() == [math.inf, -math.inf] and torch.isnan(want[last[1], 0, 2]) and want[last[1], 0, 3] == -math.inf
    assert torch.isnan(want[last[2], 0, 4]) and want[last[2], 0, 5] == math.inf
    close(o, want, size, dtype)
    inf = torch.isinf(want)
    assert torch.equal(o.double().cpu()[inf], want[inf])


# ---------------------------------------------------------------------------------------------- errors

def test_one_call_reports_its_error_once():
    """A call that still runs when its error is raised does not raise it again from the next one."""
    import experiment_swa_kda_b200 as m
    n, length = 2048, 8192
    q = torch.zeros(n * 32, 1, 128, device=DEV)
    cache = torch.zeros(4, 16, 1, 128, device=DEV)
    table = torch.full((n, length // 16), -1, dtype=torch.int32, device=DEV)      # no page at all, in any sequence
    lens = torch.full((n,), length, dtype=torch.int32, device=DEV)
    cos = sin = torch.ones(4, 64, device=DEV)
    nothing = torch.zeros(1, 0, 1, 128, device=DEV)      # a call that looks at the status and launches nothing
    m.qk_norm_rope(nothing, nothing, cos, sin)
    torch.cuda.synchronize()
    m.paged_attention(q, cache, cache, table, lens)
    done = torch.cuda.Event()
    done.record()
    with pytest.raises(RuntimeError, match="block table"):
        while True:
            finished = done.query()
            m.qk_norm_rope(nothing, nothing, cos, sin)
            assert not finished, "the error was never reported"
    torch.cuda.synchronize()
    m.qk_norm_rope(nothing, nothing, cos, sin)


# ---------------------------------------------------------------------------------------------- the layer

@pytest.mark.parametrize("cast", [lambda l: l.bfloat16(), lambda l: l.to(torch.bfloat16), lambda l: l.half().float(), lambda l: l.double().float().bfloat16()])
def test_layer_keeps_its_tables_through_casts(cast):
    """The rotation's tables are float32 whatever the parameters' type becomes, and keep their values."""
    import experiment_swa_kda_b200 as m
    torch.manual_seed(2)
    layer = m.PagedAttention(256, 4, 2, 64, max_positions=300).to(DEV)
    cos, sin = layer.cos.clone(), layer.sin.clone()
    cast(layer)
    assert layer.cos.dtype == F32 and torch.equal(layer.cos, cos) and torch.equal(layer.sin, sin) and layer.cos.device == cos.device
    cache = m.PagedCache.zeros(2, 20, 16, 2, 64, DEV)
    cache.kv_lens += 20
    y = layer(torch.randn(2, 20, 256, device=DEV).bfloat16(), cache)
    assert torch.isfinite(y).all()


def test_layer_made_without_memory_gets_its_tables():
    import experiment_swa_kda_b200 as m
    with torch.device("meta"):
        layer = m.PagedAttention(256, 4, 2, 64, max_positions=300)
    layer = layer.to_empty(device=DEV)
    want = m.PagedAttention(256, 4, 2, 64, max_positions=300).to(DEV)
    assert torch.equal(layer.cos, want.cos) and torch.equal(layer.sin, want.sin)


def test_layer_compares_its_batch_with_the_cache():
    import experiment_swa_kda_b200 as m
    layer = m.PagedAttention(256, 4, 2, 64, max_positions=300).to(DEV)
    cache = m.PagedCache.zeros(3, 32, 16, 2, 64, DEV)
    cache.kv_lens += 2
    x = torch.zeros(2, 3, 256, device=DEV).bfloat16()
    for bad in (x, x[:1], x[0], x.expand(3, 2, 3, 256)):      # 6, 3, 3 and 18 tokens: three sequences could share them
        with pytest.raises(ValueError, match="the cache's 3 sequences"):
            layer(bad, cache)
    assert layer(x.reshape(1, 6, 256), cache, torch.tensor([0, 2, 4, 6], dtype=torch.int32, device=DEV)).shape == (1, 6, 256)
    assert layer(x.reshape(3, 2, 256), cache).shape == (3, 2, 256)
