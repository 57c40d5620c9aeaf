"""Cases of the serving operators around a shared prefix: pages dealt out and slots mapped on the GPU from the lengths of
requests, and attention of a batch whose sequences start with the same cached text.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: the plain form, or with `own` the package's operators; returns every output
    exact(case, seed)   the same outputs from the definition, in 64 bits
    work(case)          bytes and floating-point operations a pass cannot do without
"""

import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one conversation of four draft tokens, of which the model may reject some: latency
        {"name": "plan_b1_draft", "kind": "plan", "rows": 1, "kv": 4097, "mode": "draft", "new": 4, "page": 16, "width": 512, "pages": 1024, "start": "none",
         "short": False},
        # the same of a large serving batch whose sequences share a prefix
        {"name": "plan_b256_draft", "kind": "plan", "rows": 256, "kv": 4096, "mode": "draft", "new": 4, "page": 64, "width": 128, "pages": 16384,
         "start": "prefix", "short": False},
        # every fourth request leaves and as many prompts come, in pages of 16
        {"name": "plan_b256_turnover", "kind": "plan", "rows": 256, "kv": 2048, "mode": "turnover", "new": 509, "page": 16, "width": 256, "pages": 32768,
         "start": "none", "short": False},
        # more prompts than the pool has pages for: some have to wait
        {"name": "plan_b100_short", "kind": "plan", "rows": 100, "kv": 4000, "mode": "turnover", "new": 1021, "page": 32, "width": 160, "pages": 1240,
         "start": "window", "short": True},
        # the largest pool: 4,096 requests, a quarter of them coming and going
        {"name": "plan_b4096_turnover", "kind": "plan", "rows": 4096, "kv": 1024, "mode": "turnover", "new": 61, "page": 16, "width": 128, "pages": 262144,
         "start": "none", "short": False},
        # one token each of 8 conversations of the 384-wide model behind one instruction text: latency
        {"name": "shared_b8_h3", "kind": "attend", "seqs": 8, "groups": 1, "q": 1, "prefix": 2048, "tail": 100, "mixed": False, "idle": False, "heads": 3,
         "kv_heads": 3, "dim": 128, "page": 16, "dtype": "bf16"},
        # one token each of 32 samples drawn from one long document
        {"name": "shared_b32_h16_kv4", "kind": "attend", "seqs": 32, "groups": 1, "q": 1, "prefix": 16384, "tail": 512, "mixed": False, "idle": False,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # one token each of a large batch behind one instruction text
        {"name": "shared_b256_h16_kv4", "kind": "attend", "seqs": 256, "groups": 1, "q": 1, "prefix": 8192, "tail": 1024, "mixed": False, "idle": False,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # several instruction texts, idle places in the batch, 64-wide heads
        {"name": "shared_b101_groups7_d64", "kind": "attend", "seqs": 101, "groups": 7, "q": 1, "prefix": 5003, "tail": 300, "mixed": False, "idle": True,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 16, "dtype": "bf16"},
        # five draft tokens of 64 conversations are checked at once
        {"name": "shared_b64_q5", "kind": "attend", "seqs": 64, "groups": 1, "q": 5, "prefix": 4097, "tail": 640, "mixed": False, "idle": False, "heads": 16,
         "kv_heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # four questions about one document come in: the matrix products count
        {"name": "shared_b4_q512", "kind": "attend", "seqs": 4, "groups": 1, "q": 512, "prefix": 8000, "tail": 512, "mixed": False, "idle": False, "heads": 16,
         "kv_heads": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # the float32 verification shape: chunks and single tokens in one call
        {"name": "shared_f32_b6_d64", "kind": "attend", "seqs": 6, "groups": 2, "q": 33, "prefix": 515, "tail": 70, "mixed": True, "idle": False, "heads": 4,
         "kv_heads": 2, "dim": 64, "page": 16, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    if rng.random() < 0.4:
        mode = rng.choice(("draft", "turnover"))
        page = rng.choice((16, 32, 64))
        rows = _log_int(rng, 1, 2048)
        kv = _log_int(rng, 64, 4096 if rows <= 256 else 1024)
        new = rng.randint(1, 8) if mode == "draft" else _log_int(rng, 2, max(2, min(1024, 65536 // rows)))
        width = -(-(kv + max(new, 8)) // page) + rng.choice((0, 1, 17))
        case = {"kind": "plan", "rows": rows, "kv": kv, "mode": mode, "new": new, "page": page, "width": width, "pages": 0,
                "start": rng.choice(("none", "none", "prefix", "window")), "short": mode == "turnover" and rng.random() < 0.25}
        case["pages"] = min(262144, rows * width + rng.randint(1, 1000))
        if case["short"]:      # room for the second step, and for about half of what the first would have besides
            a, b = _held(case)
            case["pages"] = max(1, b, (a + b) // 2)
        return case
    heads, kv_heads = rng.choice(((3, 3), (4, 2), (6, 2), (8, 1), (12, 4), (16, 4), (16, 16), (16, 1)))
    dtype = rng.choice(("bf16", "bf16", "bf16", "bf16", "f32"))
    f32 = dtype == "f32"
    seqs = _log_int(rng, 1, 8 if f32 else 256)
    q = rng.choice((1, 1, rng.randint(2, 8), _log_int(rng, 9, 40 if f32 else 600)))
    case = {"kind": "attend", "seqs": seqs, "groups": rng.choice((1, 1, 1, min(seqs, rng.randint(2, 8)))), "q": q, "prefix": _log_int(rng, 16, 1024 if f32 else 16384),
            "tail": max(q, _log_int(rng, 1, 200 if f32 else 1024)), "mixed": q > 1 and rng.random() < 0.4, "idle": rng.random() < 0.2, "heads": heads,
            "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128, 96)), "page": rng.choice((16, 32, 64, 128)), "dtype": dtype}
    # no more than the largest listed case: its products, its scores in the plain form, half a GB of cache
    big = {c["name"]: c for c in listed()}["shared_b4_q512"]
    for _ in range(64):
        cached = 4 * case["dim"] * kv_heads * (case["seqs"] * case["tail"] + case["groups"] * case["prefix"])
        if work(case)["flops"] <= work(big)["flops"] and _score_bytes(case) <= _score_bytes(big) and cached <= 1 << 29:
            break
        if case["seqs"] > case["groups"] and case["seqs"] > 1:
            case["seqs"] = max(case["groups"], case["seqs"] // 2)
        elif case["prefix"] > 256:
            case["prefix"] = case["prefix"] * 2 // 3
        else:
            case["q"] = max(1, case["q"] // 2)
    return case


# ---------------------------------------------------------------------------------------------- lengths

def _spread(n):
    """A spread of (0.15, 1]: the first has the most."""
    return 1.0 - 0.85 * ((n * 0.6180339887) % 1.0)


def _plan_lengths(case):
    """Two steps of a scheduler, (lengths, new tokens) of every row in each, and the rows' starts.

    draft: each running request has `new` more tokens, then gives back those that were rejected.  turnover: rows 3, 7, 11 ... leave
    while rows 1, 5, 9 ... get prompts, and the other way round; the rest go on by a token.  Where the pool is short the prompts of the
    second step are half as long, and it has room for those."""
    kv, new, page = case["kv"], case["new"], case["page"]
    room = case["width"] * page
    first, second, starts = [], [], []
    for n in range(case["rows"]):
        length = max(1, min(round(kv * _spread(n)), room - max(new, 1)))
        start = {"none": 0, "prefix": min(length, kv // 4), "window": max(0, length - 512)}[case["start"]]
        if case["mode"] == "draft":
            kept = (n * 7) % (new + 1)
            first.append((length + new, new))
            second.append((length + kept, kept))
        else:
            prompt = max(1, min(round(new * _spread(n + 1)), room))
            comes, leaves = (prompt, prompt), (0, 0)
            if n % 4 == 1:
                start = 0
                first.append(comes)
                second.append(leaves)
            elif n % 4 == 3:
                start = 0
                first.append(leaves)
                second.append((max(1, prompt // 2),) * 2 if case["short"] else comes)
            else:
                first.append((length + 1, 1))
                second.append((length, 1))
        starts.append(start)
    return first, second, starts


def _held(case):
    """Pages all rows want to hold in each step."""
    first, second, starts = _plan_lengths(case)
    page = case["page"]
    return [sum(-(-a // page) - min(s, a) // page for (a, _), s in zip(step, starts)) for step in (first, second)]


def _lengths(case):
    """Of each sequence: its group (or -1: an idle place in the batch), new tokens, and tokens behind the prefix, the new ones among
    them.  Groups have unequal numbers of sequences, prefixes unequal lengths."""
    n, g = case["seqs"], case["groups"]
    group, q, tail = [], [], []
    cuts = [round(n * (i / g) ** 1.3) for i in range(g + 1)]
    for i in range(n):
        part = _spread(i)
        group.append(next((x for x in range(g) if cuts[x] <= i < cuts[x + 1]), g - 1))
        a = 1 if case["mixed"] and i % 2 else max(1, round(case["q"] * part)) if case["mixed"] else case["q"]
        q.append(a)
        tail.append(max(a, round(case["tail"] * part)))
        if case["idle"] and i % 11 == 5:
            tail[-1] = None      # a place without a request: its tokens are padding
    prefix = [max(1, round(case["prefix"] * _spread(x))) for x in range(g)]
    return cuts, group, q, tail, prefix


def _score_bytes(case):
    """float32 scores the plain form holds at once."""
    cuts, group, q, tail, prefix = _lengths(case)
    return 4 * case["heads"] * max(max(q) * (b - a) * p for a, b, p in zip(cuts, cuts[1:], prefix)) if case["seqs"] else 0


def work(case):
    if case["kind"] == "plan":
        first, second, _ = _plan_lengths(case)
        tokens = sum(b for _, b in first) + sum(b for _, b in second)
        # both steps: the table, the pages' flags, lengths and starts in; position and slot of each token out, a product and a sum each
        return {"bytes": 2 * (4 * case["rows"] * case["width"] + case["pages"] + 16 * case["rows"]) + 12 * tokens, "flops": 2 * tokens}
    e = 2 if case["dtype"] == "bf16" else 4
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    cuts, group, q, tail, prefix = _lengths(case)
    tokens = sum(q)
    cached = sum(t for t in tail if t) + sum(prefix)
    pairs = sum(a * prefix[g] + a * (t - a) + a * (a + 1) // 2 for g, a, t in zip(group, q, tail) if t)
    return {"bytes": 2 * tokens * h * d * e + 2 * cached * hk * d * e + 4 * cached // case["page"] + 12 * len(q), "flops": 4 * d * h * pairs}


# ---------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "plan":
        first, second, starts = _plan_lengths(case)
        s = {"case": case, "max_tokens": max(sum(b for _, b in first), sum(b for _, b in second), 1)}
        rng = random.Random(seed)
        order = list(range(case["rows"]))
        rng.shuffle(order)      # other seeds deal the same requests to other rows
        ints = lambda x: torch.tensor([x[i] for i in order], dtype=torch.int32, device=DEVICE)
        for name, step in (("first", first), ("second", second)):
            s[name + "_lens"], s[name + "_new"] = ints([a for a, _ in step]), ints([b for _, b in step])
        s["starts"] = ints(starts) if case["start"] != "none" else None
        # the pool as an earlier step left it: the second step's rows hold pages from all over it
        col = torch.arange(case["width"], device=DEVICE)
        lens, start = s["second_lens"], torch.minimum(ints(starts), s["second_lens"])
        held = (col >= (start // case["page"])[:, None]) & (col < (-(-lens // case["page"]))[:, None])
        pages = torch.randperm(case["pages"], generator=gen, device=DEVICE)[:int(held.sum())]
        s["table"] = torch.full(held.shape, -1, dtype=torch.int32, device=DEVICE)
        s["table"][held] = pages.to(torch.int32)
        s["free"] = torch.ones(case["pages"], dtype=torch.bool, device=DEVICE)
        s["free"][pages] = False
        return s

    dtype, h, hk, d, page, n = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["page"], case["seqs"]
    cuts, group, q_lens, tail, prefix = _lengths(case)
    kv_lens = [prefix[g] + t if t else 0 for g, t in zip(group, tail)]
    width = max(1, -(-max(kv_lens) // page))
    # a sequence holds pages from the one its prefix ends in; the prefix has its own
    held = [(prefix[g] // page, -(-b // page)) if b else (0, 0) for g, b in zip(group, kv_lens)]
    of_prefix = [-(-p // page) for p in prefix]
    own_pages = sum(b - a for a, b in held)
    pages = own_pages + sum(of_prefix) + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)

    def fill(ranges, width, taken):
        lo, hi = (torch.tensor(x, device=DEVICE)[:, None] for x in zip(*ranges))
        col = torch.arange(width, device=DEVICE)
        inside = (col >= lo) & (col < hi)
        table = torch.full(inside.shape, -1, dtype=torch.int32, device=DEVICE)
        table[inside] = order[taken:taken + int(inside.sum())]
        return table

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)
    return {"case": case, "q": randn(sum(q_lens), h, d, scale=1.5), "k_cache": randn(pages, page, hk, d), "v_cache": randn(pages, page, hk, d),
            "table": fill(held, width, 0), "prefix_table": fill([(0, x) for x in of_prefix], max(of_prefix), own_pages),
            "kv_lens": i32(kv_lens), "prefix_lens": i32(prefix), "cu_groups": i32(cuts), "cu": i32([0] + q_lens).cumsum(0).to(torch.int32),
            # what a scheduler knows on the host as well
            "cuts": cuts, "prefix": prefix, "max_q": max(q_lens), "max_tail": max(t or 0 for t in tail)}


# ---------------------------------------------------------------------------------------------- plain forms

def _plain_plan(s, lens, new):
    """One step; writes the table, the flags and, where rows have to wait, the lengths."""
    case, table, free = s["case"], s["table"], s["free"]
    page, (rows, width), pages, most = case["page"], table.shape, free.numel(), s["max_tokens"]
    kv, add = lens.long(), new.long()
    start = torch.zeros_like(kv) if s["starts"] is None else torch.minimum(s["starts"].long(), kv)
    col = torch.arange(width, device=DEVICE)

    def release(end):      # entries outside of [start, end) go back; a spare flag takes what names no page
        out = (col < (start // page)[:, None]) | (col >= end[:, None])
        flags = torch.cat((free, free.new_zeros(1)))
        flags[torch.where(out & (table >= 0), table, pages).long()] = True
        free.copy_(flags[:pages])
        table.masked_fill_(out, -1)
        return ~out

    missing = release((kv + page - 1) // page) & (table < 0)
    need = missing.sum(1)
    want, asked = need.cumsum(0), add.cumsum(0)
    granted = ((want <= free.sum()) & (asked <= most)) | ((need == 0) & (add == 0))
    add = torch.where(granted, add, 0)
    lens.copy_(torch.where(granted, kv, kv - new.long()))
    kv = lens.long()
    # the k-th free page to the k-th missing entry
    missing &= granted[:, None]
    rank = (want - need)[:, None] + missing.cumsum(1) - 1
    total = missing.sum()
    order = free.long().cumsum(0) - 1
    dealt = torch.zeros(pages + 1, dtype=torch.int32, device=DEVICE)
    dealt[torch.where(free, order, pages)] = torch.arange(pages, device=DEVICE, dtype=torch.int32)
    free &= order >= total
    table.copy_(torch.where(missing, dealt[rank.clamp(0, pages)], table))
    release((kv + page - 1) // page)
    # where the new tokens go
    cu = torch.cat((add.new_zeros(1), add.cumsum(0)))
    t = torch.arange(most, device=DEVICE)
    seq = torch.searchsorted(cu[1:], t, right=True)
    is_token = t < cu[-1]
    row = seq.clamp(max=rows - 1)
    pos = torch.where(is_token, kv[row] - add[row] + t - cu[row], -1)
    at = table[row, (pos // page).clamp(min=0)].long()
    slots = torch.where(is_token, at * page + pos % page, -1)
    return cu.to(torch.int32), pos.to(torch.int32), slots


def _plain_attend(s):
    """The prefix of each group in one product for all of its tokens, then each sequence's own keys; one softmax over both."""
    case = s["case"]
    h, hk, d, n, mq, page = case["heads"], case["kv_heads"], case["dim"], case["seqs"], s["max_q"], case["page"]
    cu, kv = s["cu"].long(), s["kv_lens"].long()
    at = torch.arange(s["q"].shape[0], device=DEVICE)
    seq = torch.searchsorted(cu[1:], at, right=True)
    row = at - cu[seq]
    new = cu[1:] - cu[:-1]
    q = torch.zeros(n, mq, h, d, device=DEVICE)
    q[seq, row] = s["q"].float() * d ** -0.5
    q = q.view(n, mq, hk, h // hk, d).permute(0, 2, 3, 1, 4)      # [N, Hk, group, rows, D]
    sequences = torch.arange(n, device=DEVICE)
    group = torch.searchsorted(s["cu_groups"].long()[1:], sequences, right=True).clamp(max=case["groups"] - 1)
    prefix = s["prefix_lens"].long()[group]
    behind = kv - new >= prefix      # padding is behind nothing
    # own keys, from the prefix's end on
    key = torch.where(behind, prefix, 0)[:, None] + torch.arange(s["max_tail"], device=DEVICE)
    entry = torch.gather(s["table"].long(), 1, (key // page).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    k, v = (c[entry, key % page].permute(0, 2, 3, 1).float() for c in (s["k_cache"], s["v_cache"]))      # [N, Hk, D, keys]
    pos = (kv - new)[:, None] + torch.arange(mq, device=DEVICE)
    hidden = (key[:, None, :] > pos[:, :, None])[:, None, None]
    own_scores = torch.einsum("nkgid,nkdj->nkgij", q, k).masked_fill(hidden, float("-inf"))
    top = own_scores.amax(-1, keepdim=True)
    prefix_scores = []
    for g, length in enumerate(s["prefix"]):
        a, b = s["cuts"][g], s["cuts"][g + 1]
        pages = s["prefix_table"][g, :-(-length // page)].long()
        kp = s["k_cache"][pages].flatten(0, 1)[:length].permute(1, 2, 0).float()
        x = torch.einsum("nkgid,kdj->nkgij", q[a:b], kp).masked_fill(~behind[a:b].view(-1, 1, 1, 1, 1), float("-inf"))
        top[a:b] = torch.maximum(top[a:b], x.amax(-1, keepdim=True))
        prefix_scores.append(x)
    top = top.clamp(min=-3e38)
    p = (own_scores - top).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("nkgij,nkdj->nkgid", p, v)
    for g, length in enumerate(s["prefix"]):
        a, b = s["cuts"][g], s["cuts"][g + 1]
        pages = s["prefix_table"][g, :-(-length // page)].long()
        vp = s["v_cache"][pages].flatten(0, 1)[:length].transpose(0, 1).float()
        p = (prefix_scores[g] - top[a:b]).exp()
        total[a:b] += p.sum(-1, keepdim=True)
        o[a:b] += torch.einsum("nkgij,kjd->nkgid", p, vp)
    o = (o / total.clamp(min=1e-38)).permute(0, 3, 1, 2, 4).reshape(n, mq, h, d)
    return o[seq, row].to(s["q"].dtype)


def run(s):
    case = s["case"]
    if case["kind"] == "plan":
        outs = []
        for step in ("first", "second"):
            # lengths are written where rows have to wait: the scheduler's own copy stays
            lens = s[step + "_lens"].clone() if case["short"] else s[step + "_lens"]
            if own:
                import experiment_swa_kda_b200 as m
                outs += m.plan_pages(s["table"], lens, s["free"], s[step + "_new"], page_size=case["page"], max_tokens=s["max_tokens"], starts=s["starts"])
            else:
                outs += _plain_plan(s, lens, s[step + "_new"])
            outs.append(lens)
        return outs + [s["table"], s["free"]]
    if not own:
        return _plain_attend(s)
    import experiment_swa_kda_b200 as m
    return m.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["prefix_table"], s["prefix_lens"], s["cu_groups"],
                                     s["cu"], max_q_len=s["max_q"])


# ---------------------------------------------------------------------------------------------- the definition

def _exact_plan(case, s):
    page, most = case["page"], s["max_tokens"]
    table, free = s["table"].tolist(), s["free"].tolist()
    starts = [0] * case["rows"] if s["starts"] is None else s["starts"].tolist()
    outs = []
    for step in ("first", "second"):
        lens, new = s[step + "_lens"].tolist(), s[step + "_new"].tolist()
        wanted = [range(min(a, b) // page, -(-b // page)) for a, b in zip(starts, lens)]
        for row, cols in zip(table, wanted):
            for c, p in enumerate(row):
                if p >= 0 and c not in cols:
                    free[p], row[c] = True, -1
        missing = [[c for c in cols if row[c] < 0] for row, cols in zip(table, wanted)]
        pool = [p for p, is_free in enumerate(free) if is_free]
        want = asked = taken = 0
        cu, positions, slots = [0], [], []
        for n, row in enumerate(table):
            want, asked = want + len(missing[n]), asked + new[n]
            if (want <= len(pool) and asked <= most) or (not missing[n] and not new[n]):
                for c in missing[n]:
                    row[c], free[pool[taken]] = pool[taken], False
                    taken += 1
                here = range(lens[n] - new[n], lens[n])
                positions += here
                slots += [row[p // page] * page + p % page for p in here]
            else:
                lens[n] -= new[n]
            cu.append(len(positions))
        for row, a, b in zip(table, starts, lens):
            for c in range(-(-b // page), len(row)):
                if row[c] >= 0:
                    free[row[c]], row[c] = True, -1
        rest = [-1] * (most - len(positions))
        outs += [torch.tensor(x, dtype=t, device=DEVICE) for x, t in ((cu, torch.int32), (positions + rest, torch.int32), (slots + rest, torch.int64),
                                                                      (lens, torch.int32))]
    return outs + [torch.tensor(table, dtype=torch.int32, device=DEVICE), torch.tensor(free, device=DEVICE)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(case, s)
    cuts, group, q_lens, tail, prefix = _lengths(case)
    page, each = case["page"], case["heads"] // case["kv_heads"]
    outs, start = [], 0
    for i, (g, a, t) in enumerate(zip(group, q_lens, tail)):
        q = s["q"][start:start + a].double()
        start += a
        if not t:
            outs.append(torch.zeros_like(q))
            continue
        length = prefix[g] + t
        key = torch.arange(length, device=DEVICE)
        pages = torch.where(key < prefix[g], s["prefix_table"][g][(key // page).clamp(max=s["prefix_table"].shape[1] - 1)], s["table"][i][key // page]).long()
        k, v = s["k_cache"][pages, key % page].double(), s["v_cache"][pages, key % page].double()
        hidden = key > torch.arange(length - a, length, device=DEVICE)[:, None]
        o = torch.empty_like(q)
        for j in range(case["kv_heads"]):
            logits = (q[:, j * each:(j + 1) * each] @ k[:, j].T / math.sqrt(case["dim"])).masked_fill(hidden[:, None], -math.inf)
            o[:, j * each:(j + 1) * each] = torch.softmax(logits, -1) @ v[:, j]
        outs.append(o)
    return torch.cat(outs)
