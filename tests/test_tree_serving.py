"""``TreeDecoder`` over a longer service: requests that end and give their pages back.  Logits are compared with the fp32 model on
the whole text; gates as in ``test_tree_decode.py``."""
from __future__ import annotations

import math

import pytest
import torch

import nibblegemm_b200 as ng
from nibblegemm_b200.decode_model import Llama3Decoder
from tests.test_decode_model import TINY, _deq, _rel, _rms, _rope

pytestmark = pytest.mark.gpu

TOL = {torch.float16: 2e-2, torch.bfloat16: 4e-2}


def reference(model, tokens, q_norm=None, k_norm=None):
    """The fp32 model's logits after the last of `tokens`, all positions at once."""
    c, n = model.cfg, len(tokens)
    hq, hk, D, eps = c["heads"], c["kv_heads"], c["head_dim"], c["eps"]
    pos = torch.arange(n, device="cuda")
    x = model.embed[torch.tensor(tokens, device="cuda")].float()
    for li, w in enumerate(model.w):
        qkv = _rms(x, w["attn_norm"], eps) @ _deq(w["qkv"])
        q, k, v = (t.view(n, -1, D) for t in qkv.split([hq * D, hk * D, hk * D], 1))
        if q_norm is not None:
            q, k = _rms(q, q_norm[li], eps), _rms(k, k_norm[li], eps)
        q, k = _rope(q, pos, c["rope_theta"]), _rope(k, pos, c["rope_theta"])
        k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(D)
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), -math.inf)
        x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, hq * D) @ _deq(w["o"])
        gate, up = (_rms(x, w["mlp_norm"], eps) @ _deq(w["gu"])).chunk(2, 1)
        x = x + (torch.nn.functional.silu(gate) * up) @ _deq(w["down"])
    return (_rms(x, model.final_norm, eps) @ model.lm_head.float().t())[-1]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tokens_of(lists):
    return torch.tensor([t for x in lists for t in x], dtype=torch.int64, device="cuda")


def draw(n, seed):
    return torch.randint(0, TINY["vocab"], (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def test_requests_end_and_their_pages_serve_others():
    model = Llama3Decoder(TINY, batch=1, max_ctx=64)
    dec = ng.TreeDecoder(model, 3, 7, page_size=8, max_blocks=6)
    text = [draw(20, 1), draw(9, 2), draw(11, 3)]  # 3, 2 and 2 pages: the whole pool
    out = dec.step(tokens_of(text), ints([20, 9, 11]))
    assert out.granted.all() and dec.cursor.item() == 7
    for turn in range(4):  # each of these needs pages of one that has ended
        end = turn % 3
        dec.release(torch.arange(3, device="cuda") == end)
        assert dec.cached[end].item() == 0 and dec.held[end].item() == 0 and (dec.table[end] == -1).all()
        held = dec.held.sum().item()
        assert dec.cursor.item() == held
        pages = dec.free_pages[held:].tolist() + [p for r in dec.table.tolist() for p in r if p >= 0]
        assert sorted(pages) == list(range(7))  # every page is free or somebody's, once
        known = out.tokens.tolist()
        text = [draw(10, 20 + turn) if b == end else text[b] + [known[b]] for b in range(3)]
        counts = [10 if b == end else 1 for b in range(3)]
        out = dec.step(tokens_of([t[-n:] for t, n in zip(text, counts)]), ints(counts))
        assert out.granted.all()
        rows = torch.tensor(counts).cumsum(0) - 1
        for b in range(3):
            assert _rel(dec.logits[rows[b]], reference(model, text[b])) <= TOL[torch.float16], (turn, b)
    dec.release(torch.ones(3, dtype=torch.bool, device="cuda"))
    assert dec.cursor.item() == 0 and sorted(dec.free_pages.tolist()) == list(range(7))
    dec.release(torch.ones(3, dtype=torch.bool, device="cuda"))  # nothing is held: nothing changes
    assert dec.cursor.item() == 0 and sorted(dec.free_pages.tolist()) == list(range(7))
    for bad in (torch.ones(2, dtype=torch.bool, device="cuda"), torch.ones(3, device="cuda"), torch.ones(3, dtype=torch.bool)):
        with pytest.raises(ValueError):
            dec.release(bad)
    assert ng.extension().device_status() == 0
