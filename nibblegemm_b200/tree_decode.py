"""Ragged prompts and drafted trees on a ``Llama3Decoder``'s weights, over a paged
KV cache: the operators of ``paged.py`` put together as a server uses them.

``TreeDecoder.step`` takes the new tokens of all requests, of any mix of lengths:
either prompts and single tokens (chains), or drafted trees whose node 0 is the last
known token; a step is all of the one or all of the other.  It plans the step on the GPU,
runs the layers (the projections are the W4A16 GEMV / GEMM), takes the model's token at
every node, and keeps the drafted path that the model agrees with.  Nothing is read back
to the host: contexts, page tables and the free list live on the GPU.

The reference (arvindcr4/nibblegemm) has no counterpart; its decode step is
projections only (``bench/bench_model.py:57-86``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .decode_model import _DT, Llama3Decoder
from .paged import paged_cache, paged_plan, qk_norm_rope_append, rope_turns, tree_attention, tree_commit

HEAD_MAX_M = 64  # tokens one call of the head takes


class TreeStep(NamedTuple):
    """One step's result (all on the GPU)."""

    tokens: torch.Tensor  # int64 [requests]: each request's next token (-1: no new tokens, or not granted)
    accepted: torch.Tensor  # int32 [requests]: new tokens kept in the cache
    path: torch.Tensor  # int32 [requests, max_path]: kept nodes of a tree (chains: all are kept, -1 throughout)
    next_tokens: torch.Tensor  # int64 [tokens]: the model's token after every new token
    granted: torch.Tensor  # bool [requests]: the pool had pages for the request


class TreeDecoder:
    """Serves up to ``requests`` sequences at a time from a pool of ``num_pages`` pages;
    ``step`` runs their new tokens, ``release`` ends some of them.

    ``model`` supplies weights and configuration (its own contiguous caches are not
    used: build it with a small ``max_ctx``).  ``q_norm`` / ``k_norm`` ([layers] lists of
    [head_dim] weights) normalise queries and keys per head in models that do."""

    def __init__(self, model: Llama3Decoder, requests: int, num_pages: int, page_size: int = 16,
                 max_blocks: Optional[int] = None, q_norm=None, k_norm=None):
        cfg, dev = model.cfg, model.device
        self.model, self.page_size, self.requests = model, page_size, requests
        self.q_norm = q_norm or [None] * model.layers
        self.k_norm = k_norm or [None] * model.layers
        self.k_cache, self.v_cache = paged_cache(num_pages, page_size, model.hkv, cfg["head_dim"], model.layers,
                                                 model.dtype, dev)
        self.turns = rope_turns(cfg["head_dim"], cfg["rope_theta"], dev)
        ints = dict(dtype=torch.int32, device=dev)
        self.cached = torch.zeros(requests, **ints)  # tokens in the cache
        self.held = torch.zeros(requests, **ints)  # pages held
        self.table = torch.full((requests, max_blocks or num_pages), -1, **ints)
        self.free_pages = torch.arange(num_pages, **ints)  # pages from `cursor` on are free
        self.cursor = torch.zeros(1, **ints)

    def step(self, tokens: torch.Tensor, counts: torch.Tensor, parents: Optional[torch.Tensor] = None,
             max_tree: int = 64, max_path: int = 16) -> TreeStep:
        """Run ``counts[b]`` (int32 [requests]) new tokens of each request.

        ``tokens`` (int64 [total]) lie request behind request.  Without ``parents`` they are
        prompts or single tokens and all are kept.  With ``parents`` (int32 [total], see
        :func:`paged_plan`) they are trees of at most ``max_tree`` nodes, of which the
        agreed path of at most ``max_path`` is kept (so a prompt does not go with them: it would be
        kept as far as the model happens to agree with it).  The head runs on every new token."""
        m, cfg = self.model, self.model.cfg
        if tokens.dim() != 1 or tokens.dtype != torch.int64 or not tokens.is_cuda:
            raise ValueError("tokens must be a 1-D int64 CUDA tensor")
        lib, dt, st = m.ext.lib, _DT[m.dtype], m._stream()
        T, H, D, eps = tokens.size(0), cfg["hidden"], cfg["head_dim"], float(cfg["eps"])
        plan = paged_plan(self.cached, counts, self.held, self.table, self.free_pages, page_size=self.page_size,
                          num_tokens=T, parents=parents, cursor=self.cursor,
                          mask_words=0 if parents is None else -(-max_tree // 64))
        e = lambda n: torch.empty(T, n, device=m.device, dtype=m.dtype)  # noqa: E731
        res, xn, qkv, o, gu, act = e(H), e(H), e((m.hq + 2 * m.hkv) * D), e(H), e(2 * m.inter), e(m.inter)
        delta = e(H)
        _lib.check(lib.ng_embed_tokens(tokens.data_ptr(), None, None, m.embed.data_ptr(), dt, T, H, cfg["vocab"],
                                       delta.data_ptr(), res.data_ptr(), st), "embed_tokens")

        def norm(x, w):
            _lib.check(lib.ng_rmsnorm(x.data_ptr(), res.data_ptr(), w.data_ptr(), xn.data_ptr(), dt, T, H, eps, st),
                       "rmsnorm")

        for li, w in enumerate(m.w):
            norm(delta, w["attn_norm"])
            m._proj(xn, w["qkv"], qkv)
            k, v = self.k_cache[li], self.v_cache[li]
            q = qk_norm_rope_append(qkv, self.q_norm[li], self.k_norm[li], self.turns, plan.positions, plan.slots,
                                    k, v, q_heads=m.hq, eps=eps)
            attn = tree_attention(q, k, v, self.table, plan.kv_lens, plan.cu_new, mask=plan.mask)
            m._proj(attn.view(T, m.hq * D), w["o"], o)
            if m.world > 1:
                torch.distributed.all_reduce(o)
            norm(o, w["mlp_norm"])
            m._proj(xn, w["gu"], gu)
            _lib.check(lib.ng_silu_mul(gu.data_ptr(), act.data_ptr(), dt, T, m.inter, st), "silu_mul")
            m._proj(act, w["down"], delta)
            if m.world > 1:
                torch.distributed.all_reduce(delta)
        norm(delta, m.final_norm)
        next_tokens = self._head(xn)

        granted = (plan.kv_lens > 0) | (counts == 0)
        if parents is None:
            last = (plan.cu_new[1:] - 1).clamp(min=0).long()
            accepted = torch.where(granted, counts, 0)
            out = torch.where((plan.kv_lens > 0) & (counts > 0), next_tokens[last], -1)
            path = torch.full((self.requests, max_path), -1, dtype=torch.int32, device=m.device)
        else:
            c = tree_commit(tokens, parents, next_tokens, plan.cu_new, plan.kv_lens, self.table, self.k_cache,
                            self.v_cache, max_path=max_path)
            accepted, out, path = c.accepted, c.bonus, c.path
        self.cached += accepted
        self.held.copy_(plan.held)
        self.cursor += plan.taken
        return TreeStep(out, accepted, path, next_tokens, granted)

    def release(self, done: torch.Tensor) -> None:
        """End the requests where ``done`` (bool [requests], on the GPU) is set: their pages go
        back to the pool and their places can take new requests.  Nothing is read back."""
        if done.shape != self.cached.shape or done.dtype != torch.bool or done.device != self.cached.device:
            raise ValueError("done must be a bool [requests] tensor on the decoder's device")
        n = self.free_pages.numel()
        mine = (done[:, None] & (torch.arange(self.table.size(1), device=done.device) < self.held[:, None])).flatten()
        back = mine.sum()
        # The entries in front of the cursor stand for pages in use, so that is where the
        # pages go; entry n is for the rest of the table.
        at = torch.where(mine, self.cursor - back + mine.cumsum(0) - 1, n)
        pages = torch.cat([self.free_pages, self.free_pages[:1]]).scatter_(0, at, self.table.flatten())
        self.free_pages.copy_(pages[:n])
        self.cursor -= back
        for x in (self.cached, self.held):
            x.masked_fill_(done, 0)
        self.table.masked_fill_(done[:, None], -1)

    def _head(self, xn: torch.Tensor) -> torch.Tensor:
        """The model's token after every row of the normed hidden state."""
        m, cfg = self.model, self.model.cfg
        lib, dt, st, H, T = m.ext.lib, _DT[m.dtype], m._stream(), cfg["hidden"], xn.size(0)
        keys = torch.full((T,), -(2 ** 63), dtype=torch.int64, device=m.device)
        self.logits = torch.empty(T, m.v1 - m.v0, dtype=m.dtype, device=m.device) if m.keep_logits else None
        for r in range(0, T, HEAD_MAX_M):
            n = min(HEAD_MAX_M, T - r)
            _lib.check(lib.ng_lm_head_argmax(xn[r].data_ptr(), m.lm_head.data_ptr(), dt, n, m.v1 - m.v0, H, m.v0,
                                             self.logits[r].data_ptr() if m.keep_logits else None,
                                             keys[r:].data_ptr(), st), "lm_head_argmax")
        if m.world > 1:
            torch.distributed.all_reduce(keys, op=torch.distributed.ReduceOp.MAX)
        tokens = torch.empty(T, dtype=torch.int64, device=m.device)
        _lib.check(lib.ng_embed_tokens(None, keys.data_ptr(), tokens.data_ptr(), m.embed.data_ptr(), dt, T, H,
                                       cfg["vocab"], None, None, st), "embed_tokens")
        return tokens
