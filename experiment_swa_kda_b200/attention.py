"""Softmax-attention layers beside the KDA layers: per-head norm and rotation of queries and keys, a paged cache, attention
of new tokens over it.

The reference's models mix KDA layers with full and sliding-window attention (nanochat/gpt.py:116-157: rotary embedding,
norm of q and k, flash attention or its fallback).  There these layers are composed from library calls; here they are
kernels of this package:

    qk_norm_rope         training and prefill: norm + rotation, differentiable
    qk_norm_rope_append  serving: the same, keys and values written to the pages of a cache
    paged_attention      serving: a chunk of new tokens, or one token, of every sequence of a batch over that cache
    shared_prefix_attention   the same for sequences that start with a common text, which is read once
    plan_pages           serving: block tables and slots of a step from the lengths of its requests

A batch of new tokens is packed, [tokens, heads, D], with `cu_seqlens` [N+1] as in `chunk_kda`, or without it when every
sequence has as many.  `kv_lens` [N] counts a sequence's tokens, the new ones among them; `block_table` [N, P] names their
pages.  These three are read on the device: a decode loop captures the calls in a CUDA graph and updates the arrays in place.
Tokens behind cu_seqlens[N] belong to no sequence.  A step of fixed size, as a captured one is, has such tokens wherever a request waits or
ends (`plan_pages`) and says so with `padded`: they are padding then.  Without it they are reported as an inconsistent `cu_seqlens`.
(The KDA layers beside these take packed batches that are full.)
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import _native, ops
from .kda import Linear

Tensor = torch.Tensor

_MAX_DIM = 256


def _same_device(first: Tensor, *others: Optional[Tensor]) -> None:
    for t in (first, *others):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("attention operators cannot run on CPU tensors (there is no CPU fallback)")
        if t.device != first.device:
            raise RuntimeError("all attention tensors must be on the same CUDA device")


def _same_dtype(first: Tensor, *others: Tensor) -> None:
    ops._dt(first)
    if any(t.dtype != first.dtype for t in others):
        raise RuntimeError("q, k, v and the cache must share one dtype")


def _check_rotation(q: Tensor, cos: Tensor, sin: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor]) -> None:
    dim = q.shape[-1]
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"head_dim must be between 1 and {_MAX_DIM}")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
        raise ValueError("cos and sin must share shape [positions, rotary_dim / 2]")
    if 2 * cos.shape[1] > dim:
        raise ValueError("cos and sin rotate more values than a head has")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("cos and sin have no gradient")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (dim,) or not w.is_floating_point()):
            raise ValueError(f"{name} must have shape {(dim,)}")


def qk_norm_rope(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, *, positions: Optional[Tensor] = None, q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """RMS norm of every head of q [B,T,Hq,D] and k [B,T,Hk,D], then the rotation by position; returns dense (q', k').

    `cos`, `sin` [P, R/2] float32 rotate the first R <= D values of a head in pairs (i, i + R/2), or (2i, 2i+1) when
    `interleaved`: (a, b) -> (a cos - b sin, b cos + a sin).  `positions` [B,T] int32 or int64, or None: 0 .. T-1.  `q_weight`,
    `k_weight` [D] or None.  q and k may be slices of one projection's output.  Differentiable in q, k and the weights."""
    out = None
    if q.is_cuda:
        call = lambda q, k, cos, sin, pos, qw, kw: _native.load().norm_rope(q, k, cos, sin, pos, qw, kw, eps, bool(interleaved))
        tensors = (q, k, cos, sin, positions, q_weight, k_weight)
        out = call(*tensors)
        if out is None:
            out = ops.traced(call, tensors)
    if out is not None:
        return out
    if q.ndim != 4 or k.ndim != 4 or q.shape[:2] != k.shape[:2] or q.shape[-1] != k.shape[-1] or 0 in q.shape[2:] or 0 in k.shape[2:]:
        raise ValueError("q and k must have shapes [B, T, Hq, D] and [B, T, Hk, D]")
    _check_rotation(q, cos, sin, q_weight, k_weight)
    if positions is not None:
        if positions.shape != q.shape[:2] or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64 with shape [B, T]")
    elif q.shape[1] > cos.shape[0]:
        raise ValueError(f"{q.shape[1]} tokens, but cos and sin have {cos.shape[0]} positions")
    _same_device(q, k, cos, sin, positions, q_weight, k_weight)
    _same_dtype(q, k)
    raise RuntimeError("qk_norm_rope: too many rows for one call")


def _check_paged(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens):
    if q.ndim != 3 or 0 in q.shape[1:]:
        raise ValueError("q must have shape [tokens, Hq, D]")
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] == 0:
        raise ValueError("k_cache and v_cache must share shape [pages, page_size, Hk, D]")
    heads, dim = q.shape[1:]
    if k_cache.shape[3] != dim or not dim <= _MAX_DIM:
        raise ValueError(f"q and the cache must share a head_dim of at most {_MAX_DIM}")
    if k_cache.shape[2] == 0 or heads % k_cache.shape[2] != 0:
        raise ValueError("the cache's heads must divide the query heads")
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or block_table.shape[0] == 0:
        raise ValueError("block_table must be int32 with shape [N, pages of a sequence]")
    n = block_table.shape[0]
    if tuple(kv_lens.shape) != (n,) or kv_lens.dtype != torch.int32:
        raise ValueError(f"kv_lens must be int32 with shape {(n,)}")
    if cu_seqlens is None:
        if q.shape[0] % n != 0:
            raise ValueError("without cu_seqlens every sequence has the same number of new tokens")
    elif tuple(cu_seqlens.shape) != (n + 1,) or cu_seqlens.dtype != torch.int32:
        raise ValueError(f"cu_seqlens must be int32 with shape {(n + 1,)}")
    _same_device(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    _same_dtype(q, k_cache, v_cache)
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache), ("block_table", block_table)):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must have adjacent values along its last dimension")
    if not kv_lens.is_contiguous() or (cu_seqlens is not None and not cu_seqlens.is_contiguous()):
        raise ValueError("kv_lens and cu_seqlens must be contiguous")


def _no_grad(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is inference-only")


def qk_norm_rope_append(q: Tensor, k: Tensor, v: Tensor, cos: Tensor, sin: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor,
                        kv_lens: Tensor, cu_seqlens: Optional[Tensor] = None, *, q_weight: Optional[Tensor] = None,
                        k_weight: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False, padded: bool = False) -> Tensor:
    """`qk_norm_rope` of a serving batch with its keys and values going to their pages: returns q' [tokens,Hq,D], dense, and
    writes k' and v IN PLACE into k_cache, v_cache [pages, page_size, Hk, D].

    The i-th of a sequence's n new tokens has position kv_len - n + i; a token whose position is negative is padding (q' = 0,
    nothing is written), and so is one behind the last sequence (`padded`: there may be some).  Inference only."""
    out = None
    if q.is_cuda:
        out = _native.load().append(q, k, v, cos, sin, k_cache, v_cache, block_table, kv_lens, cu_seqlens, q_weight, k_weight, eps, bool(interleaved),
                                     bool(padded))
    if out is not None:
        return out
    _check_paged(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    expected = (q.shape[0], k_cache.shape[2], q.shape[2])
    if tuple(k.shape) != expected or tuple(v.shape) != expected:
        raise ValueError(f"k and v must have shape {expected}")
    _check_rotation(q, cos, sin, q_weight, k_weight)
    _same_device(q, k, v, cos, sin, q_weight, k_weight)
    _same_dtype(q, k, v)
    for name, t in (("k", k), ("v", v)):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must have adjacent values along its last dimension")
    _no_grad("qk_norm_rope_append", q, k, v, k_cache, v_cache, q_weight, k_weight)
    raise RuntimeError("qk_norm_rope_append: the batch or the block table is too large for one call, or a trace is being recorded")


def paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, kv_lens: Tensor, cu_seqlens: Optional[Tensor] = None, *,
                    max_q_len: int = 0, window: int = 0, scale: Optional[float] = None, return_lse: bool = False, padded: bool = False):
    """Causal attention of new tokens q [tokens,Hq,D] over a paged cache that holds their own keys and values already.

    The token at position p sees positions p - window + 1 .. p (window 0: all up to p); Hq / Hk query heads share a kv head.
    `max_q_len` bounds the new tokens of any sequence (0: unknown).  A batch that says so is cut into blocks accordingly, and
    where max_q_len * Hq / Hk <= 16 a kernel for token steps takes it: one token of 32 conversations of up to 16,384 tokens took 107 us
    with the bound, 195 packed without.

    bfloat16 runs on the tensor cores if D is a multiple of 8 up to 128, the page size 8, 16, 32, 64 or a multiple of 128, and the
    cache lies on 16 bytes at strides of whole 16 bytes.  Everything else (float32, wider heads, other pages) runs on the CUDA
    cores, 14 times slower and more: take such page sizes where there is a choice.

    Returns o [tokens,Hq,D], or (o, lse [tokens,Hq]) with the natural log of each row's sum of exponentials.  A padding token
    (negative position, or behind the last sequence; `padded`: there may be some of these) gets o = 0 and lse = -inf.  Pages that no new token reaches are not touched, and their entries in
    the table may be anything.  Inference only."""
    out = None
    if q.is_cuda:
        out = _native.load().attention(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, max_q_len, window, scale, bool(return_lse), bool(padded))
    if out is not None:
        return out if return_lse else out[0]
    _check_paged(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    if window < 0 or max_q_len < 0:
        raise ValueError("window and max_q_len must not be negative")
    if scale is not None and not (0 < scale < float("inf")):
        raise ValueError("scale must be positive and finite")
    _no_grad("paged_attention", q, k_cache, v_cache)
    raise RuntimeError("paged_attention: the batch or the block table is too large for one call, or a trace is being recorded")


def shared_prefix_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, kv_lens: Tensor, prefix_table: Tensor, prefix_lens: Tensor,
                            cu_groups: Optional[Tensor] = None, cu_seqlens: Optional[Tensor] = None, *, max_q_len: int = 0,
                            scale: Optional[float] = None, return_lse: bool = False, padded: bool = False):
    """`paged_attention` of sequences that start with a common text: its keys and values are in the cache once, and read once for all of
    the sequences.

    Sequences cu_groups[g] .. cu_groups[g+1] - 1 are group g (`cu_groups` [G+1] int32, or None: N / G each); its text is `prefix_lens`[g] tokens
    in the pages `prefix_table`[g] ([G,W] int32, [G] int32).  `kv_lens` count the prefix too.  A sequence shares it if its new tokens all lie
    behind it: its own row of `block_table` then names the pages of positions from prefix_lens[g] on - by position / page_size, as in
    `paged_attention` -, and the entries before that are not looked at.  The page in which the prefix ends is the sequence's own where its own
    tokens go on in it.  A sequence whose new tokens do not all lie behind the prefix (padding, a shorter text) or that is in no group
    has all of its keys in its own pages.

    bfloat16 under the conditions of `paged_attention` runs on the tensor cores, where the new tokens of all sequences of a group share each
    key tile of the prefix.  Weights are rounded to bfloat16 there, as `paged_attention` does with chunks, but for those of own keys where
    max_q_len * Hq / Hk <= 16: an error of up to 2^-8 of the sum of weights times |v|, measured 1.35 times that of rounding the result alone.
    `paged_attention` of token steps holds all weights to 2^-16; where that is wanted, rows that name the prefix's pages in their own tables have it,
    at the price of reading them each.

    Which kernels take a call goes by the widths of the two tables, since lengths are not known on the host: they may be as wide as one another, as rows of one
    pool's table are, or end where the texts do.

    Returns o, or (o, lse), as `paged_attention` does.  There is no window: a sliding-window layer sees little of a prefix.  Inference only."""
    out = None
    if q.is_cuda:
        out = _native.load().shared_attention(q, k_cache, v_cache, block_table, kv_lens, prefix_table, prefix_lens, cu_groups, cu_seqlens, max_q_len, scale,
                                              bool(return_lse), bool(padded))
    if out is not None:
        return out if return_lse else out[0]
    _check_paged(q, k_cache, v_cache, block_table, kv_lens, cu_seqlens)
    if prefix_table.ndim != 2 or prefix_table.dtype != torch.int32 or not 1 <= prefix_table.shape[0] <= block_table.shape[0]:
        raise ValueError("prefix_table must be int32 with shape [G, pages of a prefix], with a group for one sequence at least")
    groups = prefix_table.shape[0]
    if tuple(prefix_lens.shape) != (groups,) or prefix_lens.dtype != torch.int32:
        raise ValueError(f"prefix_lens must be int32 with shape {(groups,)}")
    if cu_groups is None:
        if block_table.shape[0] % groups != 0:
            raise ValueError("without cu_groups every group has the same number of sequences")
    elif tuple(cu_groups.shape) != (groups + 1,) or cu_groups.dtype != torch.int32:
        raise ValueError(f"cu_groups must be int32 with shape {(groups + 1,)}")
    _same_device(q, prefix_table, prefix_lens, cu_groups)
    if prefix_table.shape[1] > 1 and prefix_table.stride(1) != 1:
        raise ValueError("prefix_table must have adjacent values along its last dimension")
    if not prefix_lens.is_contiguous() or (cu_groups is not None and not cu_groups.is_contiguous()):
        raise ValueError("prefix_lens and cu_groups must be contiguous")
    if max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    if scale is not None and not (0 < scale < float("inf")):
        raise ValueError("scale must be positive and finite")
    _no_grad("shared_prefix_attention", q, k_cache, v_cache)
    raise RuntimeError("shared_prefix_attention: the batch or a block table is too large for one call, or a trace is being recorded")


def plan_pages(block_table: Tensor, kv_lens: Tensor, page_free: Tensor, new_lens: Tensor, *, page_size: int, max_tokens: int,
               starts: Optional[Tensor] = None, overtake: bool = False) -> Tuple[Tensor, Tensor, Tensor]:
    """Deals out the pages of a step and maps its new tokens to them; returns (cu_seqlens [N+1], positions [max_tokens], slots [max_tokens]).

    The caller sets `kv_lens` [N] to what its requests shall have after the step, `new_lens` [N] of these being new; a row whose
    request has ended has length 0, one that takes back rejected tokens a smaller length.  IN PLACE the rows of `block_table` [N,P]
    then hold exactly the columns from starts[n] / page_size (None: 0) up to their length: what they held besides goes back to the
    pool `page_free` [pages] bool, and what they lack takes the lowest free pages, rows in order.  `starts` is where a row's own pages
    begin: behind a prefix it shares, or where a sliding window has left off; a new token before it has no page and a negative slot.

    A row is served if the pages lacking up to and with it are there and the new tokens up to and with it are at most `max_tokens`.  One
    that is not waits: IN PLACE its length is less by its new tokens, none of which cu_seqlens counts.  The sums run over the rows that wait as
    well, so rows are served in their order, and one that asks for more than there is holds up every row behind it that asks for anything, running
    requests among them: keep prompts behind these, or pass `overtake`.  Then a row that waits counts for nothing, and all are served that still
    find their pages and tokens.

    positions [max_tokens] int32 are the new tokens' places in their sequences, slots [max_tokens] int64 those in a cache of
    [pages * page_size] rows; -1 behind the last.  They are for layers of the caller's own: append and attention go by lengths and tables, and
    `qk_norm_rope` takes no position of -1.  Nothing synchronises; a captured graph follows the arrays.  What goes on from here with
    max_tokens tokens - `qk_norm_rope_append`, the attention, `PagedAttention` - takes this cu_seqlens with `padded`, since a step need not be full.
    A call without cu_seqlens counts new tokens in every row, and would write one that waits over the last of what it has.  A pool starts out with all
    pages free and a table of -1."""
    out = None
    if block_table.is_cuda:
        out = _native.load().plan(block_table, kv_lens, page_free, new_lens, starts, page_size, max_tokens, bool(overtake))
    if out is not None:
        return out
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or 0 in block_table.shape:
        raise ValueError("block_table must be int32 with shape [N, pages of a sequence]")
    rows, width = block_table.shape
    for name, t in (("kv_lens", kv_lens), ("new_lens", new_lens), ("starts", starts)):
        if t is not None and (tuple(t.shape) != (rows,) or t.dtype != torch.int32):
            raise ValueError(f"{name} must be int32 with shape {(rows,)}")
    if page_free.ndim != 1 or page_free.dtype != torch.bool:
        raise ValueError("page_free must be bool with shape [pages]")
    if page_size < 1 or max_tokens < 0:
        raise ValueError("page_size must be positive and max_tokens not negative")
    _same_device(block_table, kv_lens, page_free, new_lens, starts)
    if (width > 1 and block_table.stride(1) != 1) or (rows > 1 and block_table.stride(0) < width):
        raise ValueError("block_table must have adjacent values along its last dimension, and rows that do not overlap")
    if not all(t.is_contiguous() for t in (kv_lens, page_free, new_lens, starts) if t is not None):
        raise ValueError("kv_lens, page_free, new_lens and starts must be contiguous")
    raise RuntimeError("plan_pages: the batch, the table or the pool is too large for one call, or a trace is being recorded")


# ------------------------------------------------------------------------------------------
# the layer
# ------------------------------------------------------------------------------------------

@dataclass
class PagedCache:
    """Pages of one attention layer and where the sequences of a serving batch have theirs.  The caller's scheduler owns it: it
    hands out pages through `block_table`, and sets `kv_lens` before a step to what a sequence will have after it."""

    k: Tensor               # [pages, page_size, Hk, D]
    v: Tensor
    block_table: Tensor     # [N, pages of a sequence] int32
    kv_lens: Tensor         # [N] int32
    page_free: Optional[Tensor] = None      # [pages] bool: the pool of `plan`
    prefix_table: Optional[Tensor] = None   # texts that sequences share (`shared_prefix_attention`)
    prefix_lens: Optional[Tensor] = None
    cu_groups: Optional[Tensor] = None

    @staticmethod
    def zeros(sequences: int, max_len: int, page_size: int, num_kv_heads: int, head_dim: int, device, dtype=torch.bfloat16) -> "PagedCache":
        """Room for `max_len` tokens of every sequence, pages dealt out in order."""
        each = -(-max_len // page_size)
        pages = lambda: torch.zeros(sequences * each, page_size, num_kv_heads, head_dim, device=device, dtype=dtype)
        table = torch.arange(sequences * each, device=device, dtype=torch.int32).view(sequences, each)
        return PagedCache(pages(), pages(), table, torch.zeros(sequences, device=device, dtype=torch.int32))

    @staticmethod
    def pool(sequences: int, max_len: int, pages: int, page_size: int, num_kv_heads: int, head_dim: int, device, dtype=torch.bfloat16) -> "PagedCache":
        """`pages` pages for all sequences together, none dealt out yet: `plan` does that step by step, up to `max_len` tokens of a sequence."""
        store = lambda: torch.zeros(pages, page_size, num_kv_heads, head_dim, device=device, dtype=dtype)
        table = torch.full((sequences, -(-max_len // page_size)), -1, device=device, dtype=torch.int32)
        return PagedCache(store(), store(), table, torch.zeros(sequences, device=device, dtype=torch.int32),
                          torch.ones(pages, device=device, dtype=torch.bool))

    def plan(self, new_lens: Tensor, max_tokens: int, starts: Optional[Tensor] = None, overtake: bool = False) -> Tuple[Tensor, Tensor, Tensor]:
        """`plan_pages` of this cache, whose `kv_lens` the caller has set for the step."""
        if self.page_free is None:
            raise RuntimeError("this cache's pages are dealt out already; PagedCache.pool makes one whose pages are planned")
        return plan_pages(self.block_table, self.kv_lens, self.page_free, new_lens, page_size=self.k.shape[1], max_tokens=max_tokens, starts=starts,
                          overtake=overtake)


class PagedAttention(nn.Module):
    """A full (`window` 0) or sliding-window attention layer for serving, the neighbour of `KimiDeltaAttention` in a model that mixes
    both: projections -> norm, rotation and cache append in one launch -> attention over the pages -> output projection."""

    def __init__(self, hidden_size: int, num_heads: int, num_kv_heads: int, head_dim: int, window: int = 0, max_positions: int = 65536,
                 rope_base: float = 10000.0, norm_eps: float = 1e-6):
        super().__init__()
        if num_kv_heads <= 0 or num_heads % num_kv_heads != 0:
            raise ValueError("num_kv_heads must divide num_heads")
        self.num_heads, self.num_kv_heads, self.head_dim, self.window, self.norm_eps = num_heads, num_kv_heads, head_dim, window, norm_eps
        self.qkv_proj = Linear(hidden_size, (num_heads + 2 * num_kv_heads) * head_dim, bias=False)
        self.q_norm = nn.Parameter(torch.ones(head_dim))
        self.k_norm = nn.Parameter(torch.ones(head_dim))
        self.o_proj = Linear(num_heads * head_dim, hidden_size, bias=False)
        self.max_positions, self.rope_base = max_positions, rope_base
        for name, table in zip(("cos", "sin"), self._tables(torch.get_default_device())):
            self.register_buffer(name, table, persistent=False)

    def _tables(self, device) -> Tuple[Tensor, Tensor]:
        place = {"dtype": torch.float64, "device": "cpu"}
        freq = self.rope_base ** (-torch.arange(0, self.head_dim, 2, **place) / self.head_dim)
        angle = torch.arange(self.max_positions, **place)[:, None] * freq
        return angle.cos().float().to(device), angle.sin().float().to(device)

    def _apply(self, fn, *args, **kwargs):
        """Casts of the module are its parameters': the rotation's tables stay float32, and are made again where a cast has rounded
        them or they had no values yet."""
        had_values = not self.cos.is_meta
        super()._apply(fn, *args, **kwargs)
        if self.cos.dtype != torch.float32 or not had_values:
            self.cos, self.sin = self._tables(self.cos.device)
        return self

    @torch.no_grad()
    def forward(self, hidden_states: Tensor, cache: PagedCache, cu_seqlens: Optional[Tensor] = None, max_q_len: int = 0, padded: bool = False) -> Tensor:
        """hidden_states [B,T,hidden], T new tokens of each of the cache's B sequences, or [1,tokens,hidden], packed, with `cu_seqlens`
        (`padded`: which may end before the last token)."""
        lead = hidden_states.shape[:-1]
        if self.window and cache.prefix_table is not None:
            raise ValueError("a sliding-window layer does not share a prefix: its cache must not have one")
        if cu_seqlens is None:
            sequences = cache.block_table.shape[0]
            if hidden_states.ndim != 3 or hidden_states.shape[0] != sequences:
                raise ValueError(f"hidden_states must have shape [B, T, hidden] with the cache's {sequences} sequences, or come with cu_seqlens")
            max_q_len = hidden_states.shape[1]
        qkv = self.qkv_proj(hidden_states).reshape(-1, self.num_heads + 2 * self.num_kv_heads, self.head_dim)
        q, k, v = qkv.split((self.num_heads, self.num_kv_heads, self.num_kv_heads), 1)
        place = (cache.k, cache.v, cache.block_table, cache.kv_lens, cu_seqlens)
        q = qk_norm_rope_append(q, k, v, self.cos, self.sin, *place, q_weight=self.q_norm, k_weight=self.k_norm, eps=self.norm_eps, padded=padded)
        if cache.prefix_table is None:
            o = paged_attention(q, *place, max_q_len=max_q_len, window=self.window, padded=padded)
        else:
            o = shared_prefix_attention(q, *place[:4], cache.prefix_table, cache.prefix_lens, cache.cu_groups, cu_seqlens, max_q_len=max_q_len,
                                        padded=padded)
        return self.o_proj(o.reshape(*lead, self.num_heads * self.head_dim))


__all__ = ["PagedAttention", "PagedCache", "paged_attention", "plan_pages", "qk_norm_rope", "qk_norm_rope_append", "shared_prefix_attention"]
