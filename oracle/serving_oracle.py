"""Plain restatements of the serving operators around a shared prefix, row by row (test infrastructure only)."""

import math

import torch


def plan_pages(table, kv_lens, page_free, new_lens, page_size, max_tokens, starts=None, overtake=False):
    """Lists in, (table, kv_lens, page_free, cu_seqlens, positions, slots) out; the lists given are left as they are.  overtake: rows that wait
    do not count against those behind them."""
    table, kv_lens, page_free, new_lens = [list(r) for r in table], list(kv_lens), list(page_free), list(new_lens)
    rows, width, pages = len(table), len(table[0]), len(page_free)
    starts = [0] * rows if starts is None else list(starts)
    for n in range(rows):
        kv_lens[n] = max(kv_lens[n], 0)
        new_lens[n] = min(max(new_lens[n], 0), kv_lens[n])
        if kv_lens[n] > width * page_size:
            kv_lens[n], new_lens[n] = min(kv_lens[n] - new_lens[n], width * page_size), 0
        starts[n] = min(max(starts[n], 0), kv_lens[n])

    def release(n, end):
        for c in range(width):
            if not starts[n] // page_size <= c < end:
                if 0 <= table[n][c] < pages:
                    page_free[table[n][c]] = True
                table[n][c] = -1

    ends = [-(-x // page_size) for x in kv_lens]
    for n in range(rows):
        release(n, ends[n])
    pool = [p for p in range(pages) if page_free[p]]
    lacks = [[c for c in range(starts[n] // page_size, ends[n]) if not 0 <= table[n][c] < pages] for n in range(rows)]
    need = tokens = taken = 0
    cu, positions, slots, waits = [0], [], [], []
    for n in range(rows):
        need, tokens = need + len(lacks[n]), tokens + new_lens[n]
        if (need <= len(pool) and tokens <= max_tokens) or (not lacks[n] and not new_lens[n]):
            for c in lacks[n]:
                table[n][c] = pool[taken]
                page_free[pool[taken]] = False
                taken += 1
            for p in range(kv_lens[n] - new_lens[n], kv_lens[n]):
                positions.append(p)
                slots.append(table[n][p // page_size] * page_size + p % page_size)
        else:
            kv_lens[n] -= new_lens[n]
            waits.append(n)
            if overtake:
                need, tokens = need - len(lacks[n]), tokens - new_lens[n]
        cu.append(len(positions))
    for n in waits:      # what its new tokens would have needed, and only that
        end = -(-kv_lens[n] // page_size)
        for c in range(end, width):
            if 0 <= table[n][c] < pages:
                page_free[table[n][c]] = True
            if table[n][c] != -1:
                table[n][c] = -1
    rest = [-1] * (max_tokens - len(positions))
    return table, kv_lens, page_free, cu, positions + rest, slots + rest


def shared_prefix_attention(q, k_cache, v_cache, table, kv_lens, q_lens, prefix_table, prefix_lens, cu_groups, scale=None):
    """(o, lse, A) in float64 with A = sum_j p_j |v_j|, the scale of what rounding the weights can change."""
    heads, dim = q.shape[1:]
    group, page = heads // k_cache.shape[2], k_cache.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    o, size = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    t = 0
    for n, (count, length) in enumerate(zip(q_lens, kv_lens)):
        shared = 0
        for g, (a, b) in enumerate(zip(cu_groups, cu_groups[1:])):
            if a <= n < b and length - count >= prefix_lens[g]:
                shared, of = prefix_lens[g], prefix_table[g]
        at = torch.arange(max(length, 0))
        pages = torch.tensor([int(of[p // page]) if p < shared else int(table[n][p // page]) for p in at.tolist()], dtype=torch.long)
        k, v = (c[pages, at % page].double().repeat_interleave(group, 1) for c in (k_cache, v_cache))
        for i in range(count):
            pos = length - count + i
            if pos >= 0:
                logits = torch.einsum("hd,khd->hk", q[t].double(), k[:pos + 1]) * scale
                top = logits.amax(-1, keepdim=True)
                p = torch.exp(logits - top)
                total = p.sum(-1, keepdim=True)
                p = p / total
                seen = v[:pos + 1]
                o[t] = torch.einsum("hk,khd->hd", p, seen)
                size[t] = torch.einsum("hk,khd->hd", p, seen.abs())
                lse[t] = (top + total.log())[:, 0]
            t += 1
    return o, lse, size
