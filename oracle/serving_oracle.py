"""Plain restatements of the serving operators around a shared prefix, row by row (test infrastructure only)."""

import math

import torch


def plan_pages(table, kv_lens, page_free, new_lens, page_size, max_tokens, starts=None):
    """Lists in, (table, kv_lens, page_free, cu_seqlens, positions, slots) out; the lists given are left as they are."""
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
