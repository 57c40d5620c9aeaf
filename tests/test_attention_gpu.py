"""Norm + rotation, cache append and attention over a paged cache against float64 restatements (oracle/attention_oracle.py).

Bounds.  float32: the framework's 1e-5 (relative 2-norm; sums of a few thousand float32 terms stay a decade below).  bfloat16
(unit roundoff u = 2^-8): every operator rounds its float32 result once, |err| <= u |y|; attention also rounds the softmax
weights, which moves o by at most u sum_j p_j |v_j| (and the sum they are divided by, as much again); 2^-12 of that scale covers float32
and second-order terms."""

import math

import pytest
import torch

import attention_oracle as A

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


def close(got, want, size=None, dtype=None, f32=1e-5):
    got, want = got.detach().double().cpu(), want.double()
    dtype = dtype or F32
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    got, want = got[fine], want[fine]
    if dtype == F32:
        assert (got - want).norm() <= f32 * want.norm() + 1e-30
        return
    room = U * want.abs() + 1e-30
    if size is not None:
        room = room + (2 * U + 2.0 ** -12) * size[fine]
    else:
        room = room + 2.0 ** -16 * want.abs().max() if want.numel() else room
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() - room).max())


def tables(length, rot):
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    angle = torch.arange(length, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


# ---------------------------------------------------------------------------------------------- norm + rotation

ROPE = [  # B, T, Hq, Hk, D, R, interleaved, weights, dtype
    (1, 1, 1, 1, 128, 128, False, True, BF16),
    (2, 7, 3, 3, 128, 128, False, False, BF16),
    (2, 33, 16, 4, 128, 64, False, True, BF16),
    (1, 65, 4, 2, 64, 64, True, True, BF16),
    (3, 17, 6, 2, 96, 48, False, True, BF16),
    (1, 300, 8, 1, 256, 256, False, True, BF16),
    (2, 19, 5, 5, 80, 20, False, True, BF16),
    (1, 9, 2, 1, 34, 6, True, True, BF16),
    (2, 129, 3, 3, 64, 32, True, False, F32),
    (1, 70, 4, 4, 128, 128, False, True, F32),
    (1, 40, 3, 1, 50, 50, False, True, F32),
    (1, 5, 2, 2, 7, 0, False, True, F32),
    (1, 1500, 16, 2, 64, 64, False, True, F32),
]


@pytest.mark.parametrize("B,T,Hq,Hk,D,R,inter,weights,dtype", ROPE)
@pytest.mark.parametrize("layout", ["dense", "packed"])
def test_norm_rope_forward_and_backward(B, T, Hq, Hk, D, R, inter, weights, dtype, layout):
    import experiment_swa_kda_b200 as m
    gen = torch.Generator().manual_seed(B * T + D)
    if layout == "packed":
        qkv = torch.randn(B, T, (Hq + 2 * Hk) * D, generator=gen).to(dtype)
        q, k = qkv[..., :Hq * D].unflatten(-1, (Hq, D)), qkv[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
        gq, gk = (lambda t: (t[..., :Hq * D].unflatten(-1, (Hq, D)), t[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))))(qkv.to(DEV))
    else:
        q, k = (torch.randn(B, T, h, D, generator=gen).to(dtype) for h in (Hq, Hk))
        gq, gk = q.to(DEV), k.to(DEV)
    length = T + 50
    cos, sin = tables(length, R)
    pos = torch.randint(0, length, (B, T), generator=gen) if layout == "packed" else None
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=gen)) if weights else None for _ in range(2))
    at = torch.arange(T).expand(B, T) if pos is None else pos
    x = [t.detach().requires_grad_(True) for t in (gq, gk)]
    w = [None if t is None else t.to(DEV).requires_grad_(True) for t in (wq, wk)]
    yq, yk = m.qk_norm_rope(*x, cos.to(DEV), sin.to(DEV), positions=None if pos is None else pos.to(DEV), q_weight=w[0], k_weight=w[1], eps=1e-5,
                            interleaved=inter)
    dq, dk = (torch.randn(t.shape, generator=gen).to(dtype) for t in (q, k))
    leaves = x + [t for t in w if t is not None]
    grads = torch.autograd.grad((yq, yk), leaves, (dq.to(DEV), dk.to(DEV)))
    for i, (y, t, dy, weight) in enumerate(((yq, q, dq, wq), (yk, k, dk, wk))):
        close(y, A.norm_rope(t, cos[at], sin[at], weight, 1e-5, inter), dtype=dtype)
        dx, dw = A.norm_rope_backward(t, dy, cos[at], sin[at], weight, 1e-5, inter)
        close(grads[i], dx, dtype=dtype)
        if weights:      # float32 whatever the inputs' type; its terms may cancel, so it is held to the terms' size
            got = grads[2 + i].double().cpu()
            terms = (dy.double().abs().sum() / dw.numel()).item()
            assert (got - dw).abs().max() <= 1e-5 * max(terms, dw.abs().max().item())


def test_norm_rope_gradient_against_differences():
    """The formula that the kernel is held to above, against central differences in float64."""
    gen = torch.Generator().manual_seed(3)
    x, dy, w = torch.randn(2, 3, 10, generator=gen).double(), torch.randn(2, 3, 10, generator=gen).double(), torch.randn(10, generator=gen).double()
    cos, sin = tables(2, 6)
    dx, dw = A.norm_rope_backward(x, dy, cos, sin, w, 1e-3, False)
    f = lambda x, w: (A.norm_rope(x, cos, sin, w, 1e-3, False) * dy).sum()
    h = 1e-6
    for t, g, at in ((x, dx, 0), (w, dw, 1)):
        for i in range(t.numel()):
            e = torch.zeros(t.numel(), dtype=torch.float64)
            e[i] = h
            e = e.view(t.shape)
            d = (f(x + e, w) - f(x - e, w)) / (2 * h) if at == 0 else (f(x, w + e) - f(x, w - e)) / (2 * h)
            assert abs(d - g.reshape(-1)[i]) <= 1e-7 * max(1.0, abs(float(d)))


def test_norm_rope_partial_gradients_streams_and_repeats():
    import experiment_swa_kda_b200 as m
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn(2, 700, h, 128, generator=gen).to(BF16).to(DEV) for h in (4, 2))
    w = torch.ones(128, device=DEV, requires_grad=True)
    cos, sin = (t.to(DEV) for t in tables(700, 128))
    yq, yk = m.qk_norm_rope(q, k, cos, sin, q_weight=w)
    assert yq.requires_grad
    one, = torch.autograd.grad(yq.float().sum(), w, retain_graph=True)      # no cotangent for yk, no gradient for q
    two, = torch.autograd.grad(yq.float().sum(), w)
    assert torch.equal(one, two)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        zq, _ = m.qk_norm_rope(q, k, cos, sin, q_weight=w.detach())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(yq, zq)
    empty = m.qk_norm_rope(q[:, :0], k[:, :0], cos, sin, q_weight=w)
    assert empty[0].shape == (2, 0, 4, 128)
    none, = torch.autograd.grad(empty[0].float().sum(), w)
    assert torch.equal(none, torch.zeros_like(none))


def test_norm_rope_trace_and_weight_types():
    import experiment_swa_kda_b200 as m
    gen = torch.Generator().manual_seed(6)
    q, k = (torch.randn(1, 20, h, 64, generator=gen).to(BF16).to(DEV) for h in (2, 1))
    cos, sin = (t.to(DEV) for t in tables(20, 64))
    w = (1 + 0.1 * torch.randn(64, generator=gen)).to(BF16).to(DEV)
    traced = torch.jit.trace(lambda q, k, w: m.qk_norm_rope(q, k, cos, sin, k_weight=w), (q, k, w), check_trace=False)
    for a, b in zip(traced(q, k, w), m.qk_norm_rope(q, k, cos, sin, k_weight=w)):
        assert torch.equal(a, b)
    wanted = w.clone().requires_grad_(True)      # a bf16 weight gets a bf16 gradient, rounded once
    yk = m.qk_norm_rope(q, k, cos, sin, k_weight=wanted)[1]
    got, = torch.autograd.grad(yk.sum(), wanted)
    _, dw = A.norm_rope_backward(k.cpu(), torch.ones(k.shape), cos.cpu(), sin.cpu(), w.cpu(), 1e-6, False)
    assert got.dtype == BF16
    assert ((got.double().cpu() - dw).abs() <= U * dw.abs() + 1e-5 * 20).all()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            m.qk_norm_rope(torch.autograd.forward_ad.make_dual(q, q), k, cos, sin)


# ---------------------------------------------------------------------------------------------- paged batches

class Batch:
    """A packed batch over a paged cache: CPU copies for the oracle, device copies for the operators.  Whatever no new token
    reaches is NaN in the cache and nonsense in the table."""

    def __init__(self, q_lens, kv_lens, Hq, Hk, D, page, dtype, window=0, seed=0, heads_first=False, spare=3, reach=True):
        gen = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.window, self.dtype = q_lens, kv_lens, window, dtype
        n, width = len(q_lens), max(1, -(-max(kv_lens) // page)) + 1
        held = [(max(0, (b - a + 1 - window) // page) if window else 0, -(-b // page)) for a, b in zip(q_lens, kv_lens)]
        held = [(min(a, b), b) for a, b in held]
        pages = sum(b - a for a, b in held) + spare
        order = torch.randperm(pages, generator=gen).tolist()
        self.table = torch.full((n, width), -7, dtype=torch.int32)
        shape = (pages, Hk, page, D) if heads_first else (pages, page, Hk, D)
        view = (lambda t: t.transpose(1, 2)) if heads_first else (lambda t: t)
        k, v = (torch.full(shape, math.nan, dtype=dtype) for _ in range(2))
        self.k, self.v = view(k), view(v)
        for i, (a, b) in enumerate(held):
            for col in range(a, b):
                self.table[i, col] = order.pop()
            first = max(0, kv_lens[i] - q_lens[i] + 1 - window) if window else 0
            key = torch.arange(first, kv_lens[i] if reach else max(first, kv_lens[i] - q_lens[i]))
            at = self.table[i].long()[key // page], key % page
            for c in (self.k, self.v):
                c[at] = torch.randn(len(key), Hk, D, generator=gen).to(dtype)
        self.q = (1.5 * torch.randn(sum(q_lens), Hq, D, generator=gen)).to(dtype)
        self.lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
        dev = lambda t: t.to(DEV)
        self.dk, self.dv = view(dev(k)), view(dev(v))      # the same strides there
        self.dtable, self.dlens, self.dcu, self.dq = dev(self.table), dev(self.lens), dev(self.cu), dev(self.q)

    def attend(self, **more):
        import experiment_swa_kda_b200 as m
        return m.paged_attention(self.dq, self.dk, self.dv, self.dtable, self.dlens, self.dcu, window=self.window, **more)

    def oracle(self, scale=None):
        return A.paged_attention(self.q, self.k, self.v, self.table, self.kv_lens, self.q_lens, self.window, scale)


ATTEND = [  # q_lens, kv_lens, Hq, Hk, D, page, window
    ([1], [1], 1, 1, 128, 16, 0),
    ([1], [700], 3, 3, 128, 16, 0),
    ([1, 1, 1, 1], [1, 64, 65, 511], 16, 4, 128, 64, 0),
    ([1, 1, 1], [900, 130, 5], 8, 1, 128, 32, 77),
    ([1, 1, 0, 1], [33, 0, 12, 300], 4, 2, 64, 16, 0),          # an empty sequence, one without new tokens
    ([2, 5, 1], [40, 5, 129], 6, 2, 64, 8, 0),
    ([3, 4], [1, 2], 2, 1, 128, 16, 0),                           # more new tokens than cached ones: padding
    ([127, 130, 1], [127, 400, 257], 4, 2, 128, 64, 0),
    ([300], [300], 3, 1, 128, 128, 0),
    ([260, 77], [1000, 77], 16, 4, 128, 64, 100),
    ([64, 64], [64, 512], 4, 4, 128, 256, 1),
    ([200, 9], [333, 1000], 12, 4, 64, 16, 0),
    ([140], [290], 5, 1, 96, 32, 64),
    ([90, 3], [95, 200], 7, 7, 80, 64, 0),
    ([33, 1], [65, 130], 4, 2, 40, 16, 30),
    ([20, 1], [50, 150], 2, 2, 256, 16, 0),
    ([17, 2], [90, 31], 3, 1, 100, 5, 0),                         # a page size and a width of no particular kind
    ([10, 1], [37, 21], 2, 1, 33, 1, 9),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"q{max(c[0])}_kv{max(c[1])}_h{c[2]}_{c[3]}_d{c[4]}_p{c[5]}_w{c[6]}")
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("bound", [False, True], ids=["", "max_q_len"])
def test_paged_attention(case, dtype, bound):
    q_lens, kv_lens, Hq, Hk, D, page, window = case
    b = Batch(q_lens, kv_lens, Hq, Hk, D, page, dtype, window, seed=D + page, heads_first=bound)
    o, lse = b.attend(return_lse=True, max_q_len=max(q_lens) if bound else 0)
    want, wlse, size = b.oracle()
    close(o, want, size, dtype)
    got = lse.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(wlse))
    fine = torch.isfinite(wlse)
    assert ((got - wlse)[fine].abs() <= 2e-5 * (1 + wlse[fine].abs())).all()
    assert torch.equal(o, b.attend(max_q_len=max(q_lens) if bound else 0))      # the same bits again, with and without lse


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hk,D,page,window,longest", [(8, 2, 128, 16, 0, 300), (3, 3, 64, 64, 50, 200), (16, 1, 128, 128, 0, 90), (12, 1, 96, 16, 33, 400)])
def test_token_steps_of_many_sequences(dtype, Hq, Hk, D, page, window, longest):
    """More sequences than threads of a block, of every length, some empty: stretches begin and end anywhere."""
    gen = torch.Generator().manual_seed(longest)
    kv_lens = torch.randint(0, longest, (260,), generator=gen).tolist()
    b = Batch([1] * 260, kv_lens, Hq, Hk, D, page, dtype, window, seed=longest)
    o, lse = b.attend(return_lse=True, max_q_len=1)
    want, wlse, size = b.oracle()
    close(o, want, size, dtype)
    assert torch.equal(torch.isinf(lse.cpu()), torch.isinf(wlse))


@pytest.mark.parametrize("case", [
    ([70], [5000], 2, 1, 128, 64, 0),                 # one row tile and long rows: parts
    ([5, 300, 1, 33], [3000, 300, 2500, 1000], 4, 2, 64, 16, 0),
    ([200], [4000], 6, 2, 128, 32, 3000),
    ([40, 2], [1500, 2100], 40, 2, 128, 16, 0),       # groups of 20: rows that are no whole tokens
    ([300, 300], [700, 320], 16, 16, 128, 16, 130),
    ([129], [900], 32, 1, 128, 8, 0),
], ids=lambda c: f"q{max(c[0])}_kv{max(c[1])}_h{c[2]}_{c[3]}_d{c[4]}_p{c[5]}_w{c[6]}")
@pytest.mark.parametrize("bound", [False, True], ids=["", "max_q_len"])
def test_long_rows_and_wide_groups(case, bound):
    q_lens, kv_lens, Hq, Hk, D, page, window = case
    b = Batch(q_lens, kv_lens, Hq, Hk, D, page, BF16, window, seed=page, heads_first=not bound)
    o, lse = b.attend(return_lse=True, max_q_len=max(q_lens) if bound else 0)
    want, wlse, size = b.oracle()
    close(o, want, size, BF16)
    assert ((lse.double().cpu() - wlse).abs() <= 2e-5 * (1 + wlse.abs())).all()


@pytest.mark.parametrize("q_len", [1, 3, 150])
def test_equal_lengths_need_no_cu_seqlens(q_len):
    import experiment_swa_kda_b200 as m
    b = Batch([q_len] * 3, [200, 170, 513], 8, 2, 128, 16, BF16)
    plain = m.paged_attention(b.dq, b.dk, b.dv, b.dtable, b.dlens)
    close(plain, b.oracle()[0], b.oracle()[2], BF16)
    assert torch.equal(plain, b.attend(max_q_len=q_len))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_len,Hq", [(4, 2), (200, 4)])
def test_hidden_values_that_are_not_finite_stay_hidden(dtype, q_len, Hq):
    """A NaN or infinite value reaches the rows that see it and no other, whatever tile they share."""
    kv = 300
    b = Batch([q_len], [kv], Hq, 2, 128, 16, dtype, window=120)
    late, early = kv - 2, kv - q_len - 119 + 1      # seen by the last two tokens; the oldest but one of the first token's window
    for pos, x in ((late, math.nan), (early, math.inf)):
        at = int(b.table[0, pos // 16]), pos % 16
        for c in (b.v, b.dv):
            c[at[0], at[1], 1, 5] = x
    o, want, size = b.attend(), *b.oracle()[::2]
    assert torch.isnan(want).any() and torch.isfinite(want).any()
    close(o, want, size, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q_len", [1, 130])
def test_scores_of_every_size(dtype, q_len):
    """Keys of -inf and of the largest size, a row of nothing else, scores hundreds apart (up to 500 in size: float32 sums of
    128 terms leave their weights some 500 x 2^-24 x 12 = 4e-4)."""
    b = Batch([q_len, q_len], [200, 200], 4, 2, 128, 64, dtype)
    page = int(b.table[0, 1])
    for c in (b.k, b.dk):
        c[page, 3] *= 300.0                      # one key far above the rest
        c[int(b.table[1, 0]), :, 0] *= 100.0
    o, want, size = b.attend(), *b.oracle()[::2]
    close(o, want, size, dtype, f32=1e-3)
    b.q.fill_(1.0), b.dq.fill_(1.0)
    for c in (b.k, b.dk):
        c[int(b.table[0, 0]), :10] = -math.inf      # weight 0 for keys 0 .. 9
        for col in range(4):
            c[int(b.table[1, col])] = -math.inf     # -inf everywhere: 0 / 0
    o = b.attend()
    want = b.oracle()[0]
    assert torch.isnan(want[q_len:]).all() and torch.isnan(o[q_len:]).all()
    close(o[:q_len], want[:q_len], b.oracle()[2][:q_len], dtype)


def test_scale_strides_and_streams():
    import experiment_swa_kda_b200 as m
    b = Batch([70, 1], [170, 90], 4, 2, 128, 16, BF16)
    packed = torch.randn(71, 11, 128, device=DEV).to(BF16)
    packed[:, 3:7] = b.dq
    strided = m.paged_attention(packed[:, 3:7], b.dk, b.dv, b.dtable, b.dlens, b.dcu, scale=0.3)
    want, _, size = b.oracle(0.3)
    close(strided, want, size, BF16)
    odd = torch.empty(71 * 4 * 128 + 1, device=DEV, dtype=BF16)[1:].view(71, 4, 128)      # starts on 2 bytes
    odd.copy_(b.dq)
    close(m.paged_attention(odd, b.dk, b.dv, b.dtable, b.dlens, b.dcu, scale=0.3), want, size, BF16)
    wide = torch.full((b.dk.shape[0], 16, 2, 131), math.nan, device=DEV, dtype=BF16)      # rows of 131 values: no 16-byte alignment
    wk, wv = wide.clone()[..., :128], wide.clone()[..., 3:]
    wk.copy_(b.dk), wv.copy_(b.dv)
    close(m.paged_attention(b.dq, wk, wv, b.dtable, b.dlens, b.dcu, scale=0.3), want, size, BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = m.paged_attention(packed[:, 3:7], b.dk, b.dv, b.dtable, b.dlens, b.dcu, scale=0.3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, strided)


def test_offsets_beyond_32_bits():
    import experiment_swa_kda_b200 as m
    pages, page, Hk, D = 2200, 1024, 8, 128      # 2.3e9 values
    k, v = (torch.zeros(pages, page, Hk, D, device=DEV, dtype=BF16) for _ in range(2))
    for q_len, Hq in ((1, 8), (40, 16)):
        b = Batch([q_len], [1500], Hq, Hk, D, page, BF16)
        table = b.dtable.clone()
        for col in range(2):
            table[0, col] = pages - 1 - col
            k[pages - 1 - col], v[pages - 1 - col] = b.dk[int(b.table[0, col])].nan_to_num(), b.dv[int(b.table[0, col])].nan_to_num()
        o = m.paged_attention(b.dq, k, v, table, b.dlens, b.dcu)
        want, _, size = b.oracle()
        close(o, want, size, BF16)


@pytest.mark.parametrize("q_len,Hq,kv", [(1, 8, 3000), (1, 4, 60), (40, 8, 6000), (300, 3, 500)])
def test_what_follows_finds_the_output(q_len, Hq, kv):
    """Kernels that start early end behind those before them: the next one in the stream reads whole results, call after call."""
    b = Batch([q_len] * 4, [kv] * 4, Hq, 1, 128, 16, BF16)
    first = b.attend(max_q_len=q_len).clone()
    for _ in range(20):
        o = b.attend(max_q_len=q_len)
        seen = o + 0
        o.zero_()
        assert torch.equal(seen, first)


def test_graph_follows_the_arrays():
    """A captured call takes the lengths and tables of its replay."""
    import experiment_swa_kda_b200 as m
    b = Batch([1, 1, 1], [900, 40, 513], 8, 2, 128, 64, BF16)
    lens = b.dlens.clone()
    b.attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = m.paged_attention(b.dq, b.dk, b.dv, b.dtable, lens, b.dcu)
    for new in ([900, 40, 513], [17, 40, 0], [300, 1, 512]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        b.kv_lens = new
        want, _, size = b.oracle()
        close(o, want, size, BF16)


# ---------------------------------------------------------------------------------------------- append

APPEND = [  # q_lens, kv_lens, Hq, Hk, D, R, page, dtype
    ([1], [1], 3, 3, 128, 128, 16, BF16),
    ([1, 1, 1], [5, 300, 64], 16, 4, 128, 64, 64, BF16),
    ([3, 0, 40, 1], [10, 9, 40, 0], 6, 2, 64, 64, 16, BF16),      # a sequence without new tokens, and a padding token
    ([5, 2], [3, 70], 4, 1, 96, 48, 32, BF16),                      # two padding tokens first
    ([7, 1], [7, 33], 2, 2, 50, 20, 5, BF16),
    ([33, 100], [90, 129], 4, 2, 128, 128, 1, F32),
    ([9], [12], 8, 8, 64, 32, 128, F32),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"q{max(c[0])}_h{c[2]}_{c[3]}_d{c[4]}_p{c[6]}")
@pytest.mark.parametrize("inter", [False, True])
def test_append(case, inter):
    import experiment_swa_kda_b200 as m
    q_lens, kv_lens, Hq, Hk, D, R, page, dtype = case
    b = Batch(q_lens, kv_lens, Hq, Hk, D, page, dtype, seed=D, heads_first=inter, reach=False)
    gen = torch.Generator().manual_seed(9)
    T = sum(q_lens)
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=gen).to(dtype)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split((Hq * D, Hk * D, Hk * D), -1))
    dq, dk, dv = (t.unflatten(-1, (-1, D)) for t in qkv.to(DEV).split((Hq * D, Hk * D, Hk * D), -1))
    cos, sin = tables(max(kv_lens) + 1, R)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=gen) for _ in range(2))
    got = m.qk_norm_rope_append(dq, dk, dv, cos.to(DEV), sin.to(DEV), b.dk, b.dv, b.dtable, b.dlens, b.dcu, q_weight=wq.to(DEV), k_weight=wk.to(DEV),
                                interleaved=inter)
    pos = torch.cat([torch.arange(n - a, n) for a, n in zip(q_lens, kv_lens)])
    real = pos >= 0
    at = pos.clamp(min=0)
    want = A.norm_rope(q, cos[at], sin[at], wq, interleaved=inter)
    want[~real] = 0
    close(got, want, dtype=dtype)
    rotated = A.norm_rope(k, cos[at], sin[at], wk, interleaved=inter)
    kc, vc = b.k.double(), b.v.clone()
    seq = torch.repeat_interleave(torch.arange(len(q_lens)), torch.tensor(q_lens))
    where = b.table.long()[seq[real], at[real] // page], at[real] % page
    kc[where], vc[where] = rotated[real], v[real]
    close(b.dk, kc, dtype=dtype)
    assert torch.equal(b.dv.cpu().nan_to_num(7.0), vc.nan_to_num(7.0))


# ---------------------------------------------------------------------------------------------- errors

def test_refusals():
    import experiment_swa_kda_b200 as m
    b = Batch([2], [40], 4, 2, 64, 16, BF16)
    args = [b.dq, b.dk, b.dv, b.dtable, b.dlens, b.dcu]

    def refused(error, match, at=None, new=None, **more):
        a = list(args)
        if at is not None:
            a[at] = new
        with pytest.raises(error, match=match):
            m.paged_attention(*a, **more)

    refused(ValueError, "q must have shape", 0, b.dq[0])
    refused(ValueError, "share shape", 2, b.dv[:, :8])
    refused(ValueError, "divide", 0, b.dq[:, :3])
    refused(ValueError, "head_dim", 0, b.dq[..., :32])
    refused(ValueError, "block_table must be int32", 3, b.dtable.long())
    refused(ValueError, "kv_lens", 4, b.dlens[:0])
    refused(ValueError, "cu_seqlens", 5, b.dcu[:1])
    refused(ValueError, "adjacent", 0, b.dq.transpose(0, 2).contiguous().transpose(0, 2))
    refused(RuntimeError, "one dtype", 0, b.dq.float())
    refused(RuntimeError, "float32 or bfloat16", 0, b.dq.half())
    refused(RuntimeError, "CPU", 0, b.q)
    refused(RuntimeError, "CPU", 1, b.k)
    refused(RuntimeError, "inference-only", 0, b.dq.clone().requires_grad_(True))
    refused(ValueError, "scale", scale=-1.0)
    refused(ValueError, "scale", scale=math.nan)
    refused(ValueError, "window", window=-1)
    refused(ValueError, "negative", max_q_len=-1)
    cos, sin = (t.to(DEV) for t in tables(40, 64))
    k = b.dq[:, :2]
    with pytest.raises(ValueError, match="k and v must have shape"):
        m.qk_norm_rope_append(b.dq, b.dq, k, cos, sin, *args[1:])
    with pytest.raises(ValueError, match="rotate more"):
        m.qk_norm_rope_append(b.dq, k, k, torch.cat((cos, cos), 1), torch.cat((cos, cos), 1), *args[1:])
    with pytest.raises(RuntimeError, match="inference-only"):
        m.qk_norm_rope_append(b.dq, k, k, cos, sin, *args[1:], q_weight=torch.ones(64, device=DEV, requires_grad=True))
    q4, k4 = b.dq[None], k[None]
    with pytest.raises(ValueError, match="must have shapes"):
        m.qk_norm_rope(q4, k4[:, :1], cos, sin)
    with pytest.raises(ValueError, match="positions"):
        m.qk_norm_rope(q4, k4, cos, sin, positions=torch.zeros(1, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="2 tokens"):
        m.qk_norm_rope(q4, k4, cos[:1], sin[:1])
    with pytest.raises(ValueError, match="float32"):
        m.qk_norm_rope(q4, k4, cos.to(BF16), sin.to(BF16))
    with pytest.raises(ValueError, match="q_weight"):
        m.qk_norm_rope(q4, k4, cos, sin, q_weight=torch.ones(63, device=DEV))
    with pytest.raises(RuntimeError, match="CPU"):
        m.qk_norm_rope(q4.cpu(), k4.cpu(), cos.cpu(), sin.cpu())
    with pytest.raises(RuntimeError, match="same CUDA device|CPU"):
        m.qk_norm_rope(q4, k4, cos.cpu(), sin.cpu())


@pytest.mark.parametrize("q_len", [1, 150])
def test_bad_tables_are_reported(q_len):
    """What the device finds wrong is bounded there and raised by the next call."""
    import experiment_swa_kda_b200 as m

    def report(match):
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=match):
            b.attend()
        torch.cuda.synchronize()
        b.attend()      # and is gone

    b = Batch([q_len], [300], 4, 2, 128, 16, BF16)
    b.attend()
    good = b.dtable.clone()
    for bad in (-1, b.dk.shape[0]):
        b.dtable[0, 18] = bad
        b.attend()
        b.dtable.copy_(good)
        report("block table")
    b.dlens.fill_(100000)
    b.attend()
    b.dlens.copy_(b.lens)
    report("block table")
    b.dcu[1] = q_len + 5
    b.attend()
    b.dcu.copy_(b.cu)
    report("cu_seqlens")
    if q_len > 1:
        b.attend(max_q_len=q_len // 2)      # a bound that is none
        report("cu_seqlens")
    cos, sin = (t.to(DEV) for t in tables(299, 128))      # one position short
    kv = torch.zeros(q_len, 2, 128, device=DEV, dtype=BF16)
    m.qk_norm_rope_append(b.dq, kv, kv, cos, sin, b.dk.clone(), b.dv.clone(), b.dtable, b.dlens, b.dcu)
    report("position")
    m.qk_norm_rope(b.dq[None], kv[None], cos, sin, positions=torch.full((1, q_len), 299, device=DEV))
    report("position")
