"""Operators of a packed batch: many requests of the language model served in one step.

One step takes q_len[b] >= 0 new tokens of each request b (a prompt, a chunk of one, or the one token
of an answer in progress) as consecutive rows of one packed batch:

    packed_layout            page tables, cache rows and positions of the step, from the lengths alone
    qk_norm_rope             per-head norms, multi-axis rotation and the K / V write of the step's rows
    packed_attention         causal grouped-query attention of the step's tokens over their caches
    shared_prefix_attention  the same for requests that continue one shared prefix (a document, an
                             image with its instructions), whose keys are read once for all of them

All tensors are CUDA tensors; outputs are given by the caller, as in ops/kernels.py, and every call
launches on the current stream without synchronising. Cache pages hold 128 rows of [kv_heads *
head_dim] bf16. Shapes, types and devices are checked in the C++ bindings; values on the device
(lengths, pages, rows) are not read by the host: a page or row outside its pool is never written, and
as a key it reads as a row of zeros. After an error that a kernel has recorded (ops/native.check_errors)
rows of the attention may stay as they were.
"""
from __future__ import annotations

from typing import Optional

import torch

from .kernels import _count
from .native import err_word, lib

PAGE = 128  # rows per K/V cache page


def _err(q: torch.Tensor) -> torch.Tensor:
    if q.device.type != "cuda":
        raise RuntimeError(f"packed attention: q must be a CUDA tensor, got one on {q.device}")
    return err_word(q.device)


def packed_layout(q_len: torch.Tensor, past: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
                  free_start: torch.Tensor, *, q_start: torch.Tensor, kv_len: torch.Tensor, rows: torch.Tensor,
                  req: torch.Tensor, pos: torch.Tensor, free_next: torch.Tensor) -> None:
    """Layout of one step (int32 throughout): q_len [B] new tokens after past [B] cached ones.

    q_start [B + 1]: first packed row of each request (the sum of q_len stays below 2^31; a length below
    zero counts as zero). kv_len [B] = past + q_len, at most 2^31 - 1, like pos. table [>= B, W]:
    each request's pages; the entries of blocks that `past` filled are read, those of the blocks this
    step adds are written with free_pages[free_start[0]], the next one, ..., in request order.
    rows / req / pos [N]: cache row, request and position of every token (row -1 where its page is below
    zero or 2^24 and more); N may exceed the sum of q_len (a fixed-size batch), the tokens past it get -1. free_next [2]: the index of the first page
    still free, and how many blocks went without a page (free list or table too short): their
    table entries and their tokens' rows are -1; give a step the last one's free_next[:1] to carry on.
    No output may lie in the place of an input or of another output."""
    _count()
    lib().packed_layout(q_len, past, table, free_pages, free_start, q_start, kv_len, rows, req, pos, free_next)


def qk_norm_rope(qkv: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, axis: torch.Tensor, q_out: torch.Tensor,
                 k_cache: torch.Tensor, v_cache: torch.Tensor, *, heads: int, kv_heads: int, head_dim: int,
                 rows: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> None:
    """qkv [N, (heads + 2 kv_heads) head_dim] projection rows (bias included) -> q_out [N, heads *
    head_dim] and the tokens' cache rows (rows [N] int32, negative: not cached; None: row n).

    Each query / key head is RMS-normalised where its weight [head_dim] is given, then rotated
    (rotate-half pairs i, i + head_dim / 2) by pos[axis[i], n] * inv_freq[i]: pos int32 [axes, N]
    below 2^24, inv_freq fp32 and axis int32 [head_dim / 2] (a pair whose axis is no row of pos is
    not rotated). q_out may be the query columns of qkv itself."""
    _count()
    lib().qk_norm_rope(qkv, pos, inv_freq, axis, q_out, k_cache, v_cache, heads, kv_heads, head_dim, rows, q_weight,
                       k_weight, eps)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, *, q_start: torch.Tensor,
                     kv_len: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                     table: Optional[torch.Tensor] = None, k_start: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal grouped-query attention of a packed batch: q / o [N, heads * head_dim] bf16 rows,
    token t of request b sees the first kv_len[b] - q_len[b] + t + 1 of its keys.

    Keys are cache pages (table [>= B, W] into pools k / v of whole pages) or, with k_start [B], the
    kv_len[b] packed rows of k / v from k_start[b]. Rows before q_start[0] or past q_start[B] are not
    touched (a call may take some of the batch's requests: slices of q_start, kv_len and table); a token
    that sees no key gets zeros (lse -inf). Cached rows past kv_len may hold anything. lse: fp32 [N, heads]
    natural log-sum-exp of the scaled scores. scale: head_dim ** -0.5 by default; positive and finite."""
    _count(2)
    lib().packed_attention(q, k, v, o, q_start, kv_len, heads, kv_heads, head_dim,
                           head_dim ** -0.5 if scale is None else scale, table, k_start, None, 0, lse, _err(q))
    return o


def shared_prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, *, q_start: torch.Tensor,
                            kv_len: torch.Tensor, table: torch.Tensor, prefix_table: torch.Tensor, prefix_len: int,
                            heads: int, kv_heads: int, head_dim: int, scale: Optional[float] = None,
                            lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """packed_attention for a batch whose requests continue one shared prefix: its prefix_len keys
    (pages prefix_table [>= ceil(prefix_len / 128)] of the same pools) are visible to every token of the
    call's requests, in front of the request's own kv_len[b] keys, which are paged through `table` and causal as there.
    kv_len counts a request's own keys only and may be zero."""
    _count(2)
    lib().packed_attention(q, k, v, o, q_start, kv_len, heads, kv_heads, head_dim,
                           head_dim ** -0.5 if scale is None else scale, table, None, prefix_table, prefix_len, lse, _err(q))
    return o
