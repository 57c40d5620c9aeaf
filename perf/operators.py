"""Cases of the attention operators beside the KDA layer: per-head norm + rotation of queries and keys (training, both
directions), the same with the keys and values written to a paged cache (serving), and attention of new tokens over that
cache.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form, or with `own` the package's operators; returns every output
    exact(case, seed)   the same outputs from the definition in 64 bits
    work(case)          bytes and floating-point operations a pass cannot do without
"""

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a training step's share of a 16-head attention layer with 4 key heads, 65,536 packed tokens: the large batch
        {"name": "norm_train_t65536_h16_kv4", "kind": "train", "batch": 1, "seq": 65536, "heads": 16, "kv_heads": 4, "dim": 128, "rot": 128,
         "weights": True, "interleaved": False, "dtype": "bf16"},
        # the float32 verification shape: odd length, half of each head rotated in adjacent pairs, no weights
        {"name": "norm_train_f32_t2047_d64", "kind": "train", "batch": 2, "seq": 2047, "heads": 3, "kv_heads": 3, "dim": 64, "rot": 32,
         "weights": False, "interleaved": True, "dtype": "f32"},
        # one token of one conversation of the 384-wide model goes into its cache: latency
        {"name": "append_b1_h3", "kind": "append", "seqs": 1, "q": 1, "kv": 4097, "mixed": False, "heads": 3, "kv_heads": 3, "dim": 128, "rot": 128,
         "page": 16, "window": 0, "dtype": "bf16"},
        # one token each of a large serving batch
        {"name": "append_b256_h16_kv4", "kind": "append", "seqs": 256, "q": 1, "kv": 2048, "mixed": False, "heads": 16, "kv_heads": 4, "dim": 128,
         "rot": 128, "page": 64, "window": 512, "dtype": "bf16"},
        # a long prompt's keys and values go into the cache
        {"name": "append_t8191_h16_kv4", "kind": "append", "seqs": 1, "q": 8191, "kv": 8191, "mixed": False, "heads": 16, "kv_heads": 4, "dim": 128,
         "rot": 128, "page": 64, "window": 0, "dtype": "bf16"},
        # one token of one conversation attends to 4,097 cached ones: latency
        {"name": "decode_b1_h3", "kind": "attend", "seqs": 1, "q": 1, "kv": 4097, "mixed": False, "heads": 3, "kv_heads": 3, "dim": 128,
         "page": 16, "window": 0, "dtype": "bf16"},
        # one token each of 32 conversations of unequal length: the cache's bytes count
        {"name": "decode_b32_h16_kv4", "kind": "attend", "seqs": 32, "q": 1, "kv": 16384, "mixed": False, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "window": 0, "dtype": "bf16"},
        # the same of a sliding-window layer and a large batch; pages behind the window are released
        {"name": "decode_b256_window512", "kind": "attend", "seqs": 256, "q": 1, "kv": 2048, "mixed": False, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "window": 512, "dtype": "bf16"},
        # a long prompt attends to itself: the matrix products count
        {"name": "chunk_t8191_h16_kv4", "kind": "attend", "seqs": 1, "q": 8191, "kv": 8191, "mixed": False, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 64, "window": 0, "dtype": "bf16"},
        # four chunks of long prompts in a sliding-window layer
        {"name": "chunk_window1024_t4x2048", "kind": "attend", "seqs": 4, "q": 2048, "kv": 8000, "mixed": False, "heads": 16, "kv_heads": 4,
         "dim": 128, "page": 64, "window": 1024, "dtype": "bf16"},
        # a scheduler's batch: chunks of prompts and single tokens of running conversations in one call, 64-wide heads
        {"name": "mixed_b12_d64", "kind": "attend", "seqs": 12, "q": 509, "kv": 4095, "mixed": True, "heads": 12, "kv_heads": 4, "dim": 64,
         "page": 16, "window": 0, "dtype": "bf16"},
        # the float32 verification shape
        {"name": "chunk_f32_t257_d64", "kind": "attend", "seqs": 2, "q": 257, "kv": 515, "mixed": False, "heads": 4, "kv_heads": 2, "dim": 64,
         "page": 16, "window": 0, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _score_bytes(case):
    """float32 scores the plain form holds at once."""
    q, kv = _lengths(case)
    return 4 * case["seqs"] * case["heads"] * max(q) * max(kv)


def draw(rng):
    kind = rng.choice(("train", "append", "attend", "attend", "attend"))
    heads, kv_heads = rng.choice(((1, 1), (3, 3), (4, 2), (6, 2), (8, 1), (12, 4), (16, 4), (16, 16), (16, 1)))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    dim = rng.choice((64, 128, 128, 96))
    if kind == "train":
        batch = rng.choice((1, 2, 3))
        seq = _log_int(rng, 16, (65536 if dtype == "bf16" else 8192) // batch)
        return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rng.choice((dim, dim, dim // 2)),
                "weights": rng.random() < 0.6, "interleaved": rng.random() < 0.3, "dtype": dtype}
    page, window = rng.choice((16, 32, 64, 128)), rng.choice((0, 0, 512, 1024, 77))
    if kind == "append":
        seqs = _log_int(rng, 1, 256)
        q = 1 if rng.random() < 0.5 else _log_int(rng, 2, max(2, 8192 // seqs))
        return {"kind": kind, "seqs": seqs, "q": q, "kv": max(q, _log_int(rng, 1, 4096)), "mixed": q > 1 and rng.random() < 0.5, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rot": rng.choice((dim, dim // 2)), "page": page, "window": window, "dtype": dtype}
    if dtype == "f32":
        seqs, q, kv = _log_int(rng, 1, 8), _log_int(rng, 1, 300), _log_int(rng, 1, 1024)
    elif rng.random() < 0.5:
        seqs, q, kv = _log_int(rng, 1, 256), 1, _log_int(rng, 16, 16384)
    else:
        seqs, q, kv = _log_int(rng, 1, 16), _log_int(rng, 2, 8192), _log_int(rng, 2, 16384)
    case = {"kind": kind, "seqs": seqs, "q": q, "kv": max(q, kv), "mixed": q > 1 and rng.random() < 0.5, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "window": window, "dtype": dtype}
    # no more than the largest listed case: its products, its scores in the plain form, half a GB of cache
    big = {c["name"]: c for c in listed()}["chunk_t8191_h16_kv4"]
    for _ in range(64):
        cached = 4 * dim * kv_heads * seqs * case["kv"]
        if work(case)["flops"] <= work(big)["flops"] and _score_bytes(case) <= _score_bytes(big) and cached <= 1 << 29:
            break
        if case["seqs"] > 1:
            case["seqs"] = seqs = max(1, seqs // 2)
        elif case["q"] > case["kv"] // 2 and case["q"] > 1:
            case["q"] = case["q"] * 2 // 3
        else:
            case["kv"] = max(case["q"], case["kv"] * 2 // 3)
    return case


def _lengths(case):
    """New tokens and cached tokens (the new ones among them) of each sequence: the first has the most, the others a
    spread of them.  A mixed batch has a single new token in every second sequence."""
    q, kv = [], []
    for n in range(case["seqs"]):
        part = 1.0 - 0.85 * ((n * 0.6180339887) % 1.0)
        a = 1 if case["mixed"] and n % 2 else max(1, round(case["q"] * part)) if case["mixed"] else case["q"]
        q.append(a)
        kv.append(max(a, round(case["kv"] * part)))
    return q, kv


def _pairs(q, kv, window):
    """Visible (query, key) pairs of one sequence: query i of q sees min(kv - q + i + 1, window) keys."""
    first = kv - q + 1
    if not window:
        return q * first + q * (q - 1) // 2
    short = min(q, max(0, window - first))      # queries that see fewer than `window`
    return short * first + short * (short - 1) // 2 + (q - short) * window


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "train":
        n = case["batch"] * case["seq"] * (h + hk) * d      # values of q and k together
        # q, k, dq', dk' in; q', k', dq, dk out; the tables; the weights and their gradients
        return {"bytes": 4 * n * e + 4 * case["seq"] * case["rot"] + (16 * d if case["weights"] else 0), "flops": 20 * n}
    q, kv = _lengths(case)
    tokens, win = sum(q), case["window"]
    if case["kind"] == "append":
        return {"bytes": tokens * (2 * h + 4 * hk) * d * e + 4 * tokens * case["rot"] + 12 * len(q), "flops": 10 * tokens * (h + hk) * d}
    seen = sum(min(b, win + a - 1) if win else b for a, b in zip(q, kv))
    return {"bytes": 2 * tokens * h * d * e + 2 * seen * hk * d * e + 4 * seen // case["page"] + 8 * len(q),
            "flops": 4 * d * h * sum(_pairs(a, b, win) for a, b in zip(q, kv))}


def _tables(length, rot, device):
    """cos and sin [length, rot / 2] of the usual frequencies."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, h, hk, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)

    if case["kind"] == "train":
        b, t = case["batch"], case["seq"]
        # q and k are slices of one projection's output, as a layer has them
        qkv = randn(b, t, (h + 2 * hk) * d)
        q, k = (x.unflatten(-1, (-1, d)) for x in (qkv[..., :h * d], qkv[..., h * d:(h + hk) * d]))
        s = {"case": case, "q": q.detach().requires_grad_(True), "k": k.detach().requires_grad_(True), "dq": randn(b, t, h, d), "dk": randn(b, t, hk, d)}
        s["cos"], s["sin"] = _tables(t, case["rot"], DEVICE)
        for name in ("q_weight", "k_weight"):
            w = torch.randn(d, generator=gen, device=DEVICE).mul_(0.1).add_(1.0)
            s[name] = w.requires_grad_(True) if case["weights"] else None
        return s

    q_lens, kv_lens = _lengths(case)
    page, win, n = case["page"], case["window"], case["seqs"]
    width = -(-max(kv_lens) // page)
    # pages a sequence holds: from the first one its oldest new token sees (sliding window) to the last
    held = [(max(0, b - a + 1 - win) // page if win else 0, -(-b // page)) for a, b in zip(q_lens, kv_lens)]
    pages = sum(b - a for a, b in held) + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    lo, hi = (torch.tensor(x, device=DEVICE) for x in zip(*held))
    col = torch.arange(width, device=DEVICE)
    inside = (col >= lo[:, None]) & (col < hi[:, None])
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    table[inside] = order[:int(inside.sum())]
    tokens = sum(q_lens)
    s = {"case": case, "table": table, "kv_lens": torch.tensor(kv_lens, dtype=torch.int32, device=DEVICE), "max_q": max(q_lens), "max_kv": max(kv_lens),
         "k_cache": randn(pages, page, hk, d), "v_cache": randn(pages, page, hk, d)}
    s["cu"] = torch.tensor([0] + q_lens, device=DEVICE).cumsum(0).to(torch.int32)
    if case["kind"] == "append":
        qkv = randn(tokens, (h + 2 * hk) * d)
        s["q"], s["k"], s["v"] = (x.unflatten(-1, (-1, d)) for x in qkv.split((h * d, hk * d, hk * d), -1))
        s["cos"], s["sin"] = _tables(max(kv_lens), case["rot"], DEVICE)
        s["q_weight"], s["k_weight"] = (torch.randn(d, generator=gen, device=DEVICE).mul_(0.1).add_(1.0) for _ in range(2))
    else:
        s["q"] = randn(tokens, h, d, scale=1.5)
    return s


# ---------------------------------------------------------------------------------------------- plain forms, 32 bits

def _norm_rope(x, cos, sin, weight, interleaved):
    """x [..., H, D] float32; cos, sin [..., R/2] of each token."""
    u = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        u = u * weight
    half = cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    rot, rest = u[..., :2 * half], u[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        return torch.cat((torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), rest), -1)
    a, b = rot[..., :half], rot[..., half:]
    return torch.cat((a * c - b * s, b * c + a * s, rest), -1)


def _places(s):
    """Sequence and position of each token."""
    cu = s["cu"].long()
    at = torch.arange(s["q"].shape[0], device=DEVICE)
    seq = torch.searchsorted(cu[1:], at, right=True)
    return seq, s["kv_lens"].long()[seq] - (cu[seq + 1] - at)


def _plain_train(s):
    inter = s["case"]["interleaved"]
    wanted = [s["q"], s["k"]] + [s[n] for n in ("q_weight", "k_weight") if s[n] is not None]
    q = _norm_rope(s["q"].float(), s["cos"], s["sin"], s["q_weight"], inter).to(s["q"].dtype)
    k = _norm_rope(s["k"].float(), s["cos"], s["sin"], s["k_weight"], inter).to(s["k"].dtype)
    grads = torch.autograd.grad((q, k), wanted, (s["dq"], s["dk"]))
    return [q, k, *grads]


def _plain_append(s):
    seq, pos = _places(s)
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _norm_rope(s["q"].float(), cos, sin, s["q_weight"], False).to(s["q"].dtype)
    k = _norm_rope(s["k"].float(), cos, sin, s["k_weight"], False).to(s["k"].dtype)
    page = s["case"]["page"]
    slot = s["table"].long()[seq, pos // page], pos % page
    s["k_cache"].index_put_(slot, k)
    s["v_cache"].index_put_(slot, s["v"])
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attend(s):
    case = s["case"]
    h, hk, d, win = case["heads"], case["kv_heads"], case["dim"], case["window"]
    n, mq = case["seqs"], s["max_q"]
    seq, pos = _places(s)
    row = torch.arange(len(seq), device=DEVICE) - s["cu"].long()[seq]
    q = torch.zeros(n, mq, h, d, device=DEVICE)
    q[seq, row] = s["q"].float() * d ** -0.5
    at = torch.full((n, mq), -1, device=DEVICE)
    at[seq, row] = pos
    table = s["table"].long().clamp(min=0)
    k, v = (c[table].flatten(1, 2)[:, :s["max_kv"]].permute(0, 2, 1, 3).float() for c in (s["k_cache"], s["v_cache"]))
    q = q.view(n, mq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    scores = q @ k.transpose(-1, -2)
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if win:
        seen &= key > at[..., None] - win
    seen = seen[:, None, None].expand(n, hk, h // hk, mq, -1).reshape(scores.shape)
    scores.masked_fill_(~seen, float("-inf"))
    del seen
    scores -= scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    o = o.view(n, hk, h // hk, mq, d).permute(0, 3, 1, 2, 4).reshape(n, mq, h, d)
    return o[seq, row].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if not own:
        return {"train": _plain_train, "append": _plain_append, "attend": _plain_attend}[case["kind"]](s)
    import experiment_swa_kda_b200 as m
    if case["kind"] == "train":
        q, k = m.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                              interleaved=case["interleaved"])
        wanted = [s["q"], s["k"]] + [s[n] for n in ("q_weight", "k_weight") if s[n] is not None]
        return [q, k, *torch.autograd.grad((q, k), wanted, (s["dq"], s["dk"]))]
    if case["kind"] == "append":
        q = m.qk_norm_rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu"],
                                  q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return [q, s["k_cache"], s["v_cache"]]
    return m.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu"], max_q_len=s["max_q"], window=case["window"])


# ---------------------------------------------------------------------------------------------- the definition, 64 bits

def _turn(half, width, interleaved):
    """Places of the two members of each rotated pair."""
    i = torch.arange(half, device=DEVICE)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def _exact_forward(x, cos, sin, weight, interleaved):
    x = x.detach().double()
    w = torch.ones(x.shape[-1], device=DEVICE, dtype=torch.float64) if weight is None else weight.detach().double()
    r = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) ** -0.5
    a, b = _turn(cos.shape[-1], x.shape[-1], interleaved)
    c, s = cos.double()[..., None, :], sin.double()[..., None, :]
    y = x * r * w
    ya, yb = y[..., a], y[..., b]
    y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
    return y


def _exact_backward(x, dy, cos, sin, weight, interleaved):
    x, g = x.detach().double(), dy.double().clone()
    w = torch.ones(x.shape[-1], device=DEVICE, dtype=torch.float64) if weight is None else weight.detach().double()
    r = (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) ** -0.5
    a, b = _turn(cos.shape[-1], x.shape[-1], interleaved)
    c, s = cos.double()[..., None, :], sin.double()[..., None, :]
    ga, gb = g[..., a], g[..., b]
    g[..., a], g[..., b] = ga * c + gb * s, gb * c - ga * s
    dw = (g * x * r).flatten(0, -2).sum(0)
    g = g * w
    return r * g - x * r ** 3 * (g * x).sum(-1, keepdim=True) / x.shape[-1], dw


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "train":
        out = [_exact_forward(s[n], s["cos"], s["sin"], s[n + "_weight"], case["interleaved"]) for n in "qk"]
        back = [_exact_backward(s[n], s["d" + n], s["cos"], s["sin"], s[n + "_weight"], case["interleaved"]) for n in "qk"]
        return out + [dx for dx, _ in back] + ([dw for _, dw in back] if case["weights"] else [])
    q_lens, kv_lens = _lengths(case)
    page, win, d = case["page"], case["window"], case["dim"]
    outs, start = [], 0
    k_all, v_all = s["k_cache"].double(), s["v_cache"].double()
    if case["kind"] == "append":
        rotated = []
        for n, (a, b) in enumerate(zip(q_lens, kv_lens)):
            rows = slice(start, start + a)
            cos, sin = s["cos"][b - a:b], s["sin"][b - a:b]
            rotated.append(_exact_forward(s["q"][rows], cos, sin, s["q_weight"], False))
            at = torch.arange(b - a, b, device=DEVICE)
            slot = s["table"][n].long()[at // page], at % page
            k_all[slot] = _exact_forward(s["k"][rows], cos, sin, s["k_weight"], False)
            v_all[slot] = s["v"][rows].double()
            start += a
        return [torch.cat(rotated), k_all, v_all]
    group = case["heads"] // case["kv_heads"]
    for n, (a, b) in enumerate(zip(q_lens, kv_lens)):
        q = s["q"][start:start + a].double()
        first = max(0, b - a + 1 - win) if win else 0
        key = torch.arange(first, b, device=DEVICE)
        slot = s["table"][n].long()[key // page], key % page
        k, v = k_all[slot], v_all[slot]
        pos = torch.arange(b - a, b, device=DEVICE)[:, None]
        hidden = key > pos
        if win:
            hidden |= key <= pos - win
        o = torch.empty_like(q)
        for j in range(case["heads"]):
            logits = (q[:, j] @ k[:, j // group].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            o[:, j] = torch.softmax(logits, -1) @ v[:, j // group]
        outs.append(o)
        start += a
    return torch.cat(outs)
