"""Paged KV cache and drafted trees: what a speculative (or plain batched) decode
step needs between its projections, for requests of any mix of lengths.

A step runs

1. :func:`paged_plan` -- once: block table, slot map, positions and tree masks
   from the requests' lengths, on the GPU;
2. :func:`qk_norm_rope_append` and :func:`tree_attention` -- per layer;
3. :func:`tree_commit` -- once: the drafted path that the model agrees with, and
   the move of its cache rows.

Nothing is read back to the host between them, so a step can be captured in a
CUDA graph.  The reference (arvindcr4/nibblegemm) has no counterpart: its decode
step is projections only (``bench/bench_model.py:57-86``).

A cache is a pair of [pages, page_size, kv heads, D] tensors (K and V, same
strides, D contiguous, ``page_size`` a power of two of 8 to 1024), one pair per
layer or with a leading layer dimension; :func:`paged_cache` makes one.  Requests
name their pages in an int32 [requests, blocks] block table.  The new tokens of
all requests lie behind one another, ``cu_new`` says where each request's begin.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _after, extension


class PagedPlan(NamedTuple):
    """One step's layout (all on the GPU; see :func:`paged_plan`)."""

    cu_new: torch.Tensor  # int32 [requests + 1]: where each request's new tokens begin
    slots: torch.Tensor  # int32 [tokens]: page * page_size + row, -1 = not stored
    positions: torch.Tensor  # int32 [tokens]
    kv_lens: torch.Tensor  # int32 [requests]: cached + new, 0 = not granted
    held: torch.Tensor  # int32 [requests]: pages held after the step's allocation
    taken: torch.Tensor  # int32 [1]: pages taken from the free list
    mask: Optional[torch.Tensor]  # int64 [tokens, words]: ancestors-or-self bits


class TreeCommit(NamedTuple):
    """What :func:`tree_commit` kept."""

    accepted: torch.Tensor  # int32 [requests]: kept nodes, the root among them
    path: torch.Tensor  # int32 [requests, max_path]: their places in the tree, -1 beyond
    bonus: torch.Tensor  # int64 [requests]: the model's token after the last kept node
    kv_lens: torch.Tensor  # int32 [requests]: cached tokens after the step; 0 where the plan granted nothing


def _binding():
    b = extension().binding
    if b is None:
        raise _lib.NibbleError("the compiled binding is missing: build it with `python -m nibblegemm_b200.build`")
    return b


def _done(status: int, op: str) -> None:
    if status:
        _lib.check(status, op)
    _after(op)


def paged_cache(num_pages: int, page_size: int, kv_heads: int, head_dim: int, layers: Optional[int] = None,
                dtype: torch.dtype = torch.float16, device="cuda"):
    """A zeroed (K, V) cache pair, [pages, page_size, kv_heads, head_dim] with
    ``layers`` in front if given.  In memory a head's rows of a page lie together,
    so one head's attention reads whole page_size * head_dim runs."""
    lead = () if layers is None else (layers,)
    return tuple(torch.zeros(*lead, num_pages, kv_heads, page_size, head_dim, dtype=dtype,
                             device=device).transpose(-3, -2) for _ in range(2))


def rope_turns(rotary_dim: int, theta: float = 500000.0, device="cuda") -> torch.Tensor:
    """Rotation frequencies theta^(-2i / rotary_dim) / (2 pi) in turns per
    position, as int64 multiples of 2^-64 turn, for :func:`qk_norm_rope_append`.

    position * turns modulo 2^64 is the exact phase at any position.  Scaled
    frequencies (long-context variants) are given the same way: int64 of
    frequency / (2 pi) * 2^64, below half a turn."""
    if rotary_dim < 0 or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16, not {rotary_dim}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    turns = torch.pow(torch.tensor(float(theta), dtype=torch.float64), -2.0 * i / max(1, rotary_dim)) / (2 * math.pi)
    return (turns * 2.0**64).round().to(torch.int64).to(device)


def paged_plan(cached: torch.Tensor, new: torch.Tensor, held: torch.Tensor, block_table: torch.Tensor,
               free_pages: torch.Tensor, *, page_size: int, num_tokens: int,
               parents: Optional[torch.Tensor] = None, mask_words: int = 0,
               cursor: Optional[torch.Tensor] = None) -> PagedPlan:
    """Plan one step: ``new[b]`` tokens for each request with ``cached[b]`` tokens
    in ``held[b]`` pages (int32 [requests] each).

    Pages are taken in request order from ``free_pages`` (int32), from entry
    ``cursor`` (int32 [1], default 0) on, and written into ``block_table``
    (int32 [requests, blocks], in place).  A request whose pages are not there or
    do not fit its row of the table is not granted: slots -1, ``kv_lens`` 0.  One that
    does not fit takes nothing from the others; ``taken`` counts the pages that were given out.

    ``num_tokens`` is the capacity of the per-token outputs (rows past the last
    new token get slot -1).  ``parents`` (int32 [num_tokens], within the request,
    below the token's own index, -1 for a root) makes trees: positions are
    ``cached + depth`` and, with ``mask_words``, ``mask`` holds 64 * mask_words
    bits a token for :func:`tree_attention`.  Inconsistent lengths or parents are
    reported by :func:`check_device`.  ``cached``, ``new`` and ``held`` are left as they are."""
    out, status = _binding().paged_plan(cached, new, held, block_table, free_pages, page_size, num_tokens, parents,
                                        mask_words, cursor)
    _done(status, "paged_plan")
    return PagedPlan(*out)


def qk_norm_rope_append(qkv: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                        turns: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, *, q_heads: int, eps: float = 1e-5,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-head RMSNorm of q and k, rotation, and append of k and v, in one pass.

    ``qkv`` [tokens, (q_heads + 2 kv_heads) * D] (rows may be strided) is the fused
    projection's output; ``q_weight`` / ``k_weight`` [D] are the norms' weights
    (both None: no norm).  The first ``2 * len(turns)`` values of a head are
    rotated in pairs (i, i + len(turns)) by ``positions * turns`` (see
    :func:`rope_turns`; an empty ``turns``: no rotation).  k and v go to row
    ``slots[m]`` of the caches (negative: nowhere); the queries [tokens, q_heads, D] are
    returned (in ``out`` if given).  Arithmetic in fp32, one rounding at the end."""
    q, status = _binding().qk_norm_rope_append(qkv, q_weight, k_weight, turns, positions, slots, k_cache, v_cache,
                                               q_heads, eps, out)
    _done(status, "qk_norm_rope_append")
    return q


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                   kv_lens: torch.Tensor, cu_new: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of each request's new tokens over its first ``kv_lens[b]`` cache
    rows, whose last ``cu_new[b+1] - cu_new[b]`` are the new tokens' own.

    ``q`` [tokens, q_heads, D] may be strided.  A token sees every row before the
    new ones, and of those the ones its ``mask`` row names (int64 [tokens, words],
    bit j = new token j of the request); without a mask new token i sees 0 .. i, so
    chains, prompts and single tokens need none.  A token that sees nothing, or is no
    request's, gives zeros.  ``scale`` defaults to 1 / sqrt(D).  Returns out like q, and with
    ``return_lse`` also the fp32 [tokens, q_heads] logarithm of the sum of
    exponentials (-inf where nothing is seen).  D 64 or 128.  Scores, sums and the output's
    accumulation are fp32; the probabilities are rounded to the type of ``q`` for the product with V.

    Scratch memory (79 MB) is kept for each stream; a call that is captured takes it from its
    graph's own memory, so graphs may be replayed at the same time."""
    y, lse, status = _binding().tree_attention(q, k_cache, v_cache, block_table, kv_lens, cu_new, mask,
                                               q.size(-1) ** -0.5 if scale is None else scale, return_lse, out)
    _done(status, "tree_attention")
    return (y, lse) if return_lse else y


def tree_commit(draft: torch.Tensor, parents: torch.Tensor, next_tokens: torch.Tensor, cu_new: torch.Tensor,
                kv_lens: torch.Tensor, block_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                *, max_path: int) -> TreeCommit:
    """Keep the drafted path that the model agrees with.

    From node 0 of each request on, the walk goes to the first child whose
    ``draft`` token (int64 [tokens]) is the model's ``next_tokens`` at its parent, for at most
    ``max_path`` nodes.  The kept nodes' rows of every layer (``k_cache`` / ``v_cache`` with or without a
    leading layer dimension, in place) move behind the rows that were there
    before the tree.  ``kv_lens`` and ``cu_new`` are the step's (:class:`PagedPlan`).  A request
    that was not granted has ``kv_lens`` 0 there and in the result: its cached tokens are what
    they were (``cached += accepted`` is right for every request)."""
    *out, status = _binding().tree_commit(draft, parents, next_tokens, cu_new, kv_lens, block_table, k_cache,
                                          v_cache, max_path)
    _done(status, "tree_commit")
    return TreeCommit(*out)
