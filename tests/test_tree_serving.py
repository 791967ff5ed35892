"""``TreeDecoder`` over a longer service: requests that end and give their pages back, requests
at the end of their row of the table, kept rows as later steps see them, norm weights other
than ones, and steps replayed from a CUDA graph.  Logits are compared with the fp32 model on
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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norm_weights_and_kept_rows(dtype):
    """Per-head norms that are not ones; a plain token on top of kept rows sees the whole text."""
    model = Llama3Decoder(TINY, batch=1, max_ctx=64, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    norms = [[(1 + 0.3 * torch.randn(128, generator=g, device="cuda")).to(dtype) for _ in model.w] for _ in range(2)]
    dec = ng.TreeDecoder(model, 2, 20, page_size=8, q_norm=norms[0], k_norm=norms[1])
    text = [draw(13, 1), draw(6, 2)]
    out = dec.step(tokens_of(text), ints([13, 6]))
    for b, row in enumerate((12, 18)):
        assert _rel(dec.logits[row], reference(model, text[b], *norms)) <= TOL[dtype]
    moved = 0
    for turn in range(3):
        parents = [[-1, 0, 0, 2, 2, 4], [-1, 0, 0, 0, 3]]
        state = [x.clone() for x in (dec.cached, dec.held, dec.table, dec.cursor)]
        known = out.tokens.tolist()
        trees = [[known[b]] + draw(len(parents[b]) - 1, 10 * turn + b) for b in range(2)]
        flat, n = ints(parents[0] + parents[1]), ints([6, 5])
        for depth in range(3):  # the model's own tokens, down the last child each time: nodes with gaps between
            for x, y in zip((dec.cached, dec.held, dec.table, dec.cursor), state):
                x.copy_(y)
            out = dec.step(tokens_of(trees), n, flat, max_tree=6, max_path=4)
            if depth == 2:
                break
            for b, start in enumerate((0, 6)):
                at = out.path[b, out.accepted[b] - 1].item()
                kids = [c for c in range(len(parents[b])) if parents[b][c] == at]
                if kids:
                    trees[b][kids[-1]] = out.next_tokens[start + at].item()
        for b in range(2):
            path = [c for c in out.path[b].tolist() if c >= 0]
            moved += sum(c != i for i, c in enumerate(path))
            text[b] += [trees[b][c] for c in path]
        # one plain token on top
        known = out.tokens.tolist()
        out = dec.step(out.tokens.clone(), ints([1, 1]))
        for b in range(2):
            text[b].append(known[b])
            assert _rel(dec.logits[b], reference(model, text[b], *norms)) <= TOL[dtype], (turn, b)
        assert dec.cached.tolist() == [len(x) for x in text]
    assert moved >= 6
    assert ng.extension().device_status() == 0


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


def test_a_request_at_the_end_of_its_row_drains_nothing():
    model = Llama3Decoder(TINY, batch=1, max_ctx=64)
    dec = ng.TreeDecoder(model, 2, 12, page_size=8, max_blocks=2)
    text = [draw(16, 1), draw(5, 2)]
    out = dec.step(tokens_of(text), ints([16, 5]))
    assert dec.cursor.item() == 3
    for i in range(11):  # the second request goes on to its own end
        known = out.tokens.tolist()
        text[1].append(known[1])
        out = dec.step(torch.tensor([7, known[1]], device="cuda"), ints([1, 1]))
        assert out.granted.tolist() == [False, True] and out.accepted.tolist() == [0, 1]
        assert dec.cursor.item() == dec.held.sum().item() == 2 + (1 if 6 + i <= 8 else 2)
    assert _rel(dec.logits[1], reference(model, text[1])) <= TOL[torch.float16]
    out = dec.step(torch.tensor([7, 7], device="cuda"), ints([1, 1]))
    assert out.granted.tolist() == [False, False] and dec.cursor.item() == 4
    assert ng.extension().device_status() == 0


@pytest.mark.parametrize("trees", [False, True])
def test_steps_of_a_graph(trees):
    """A captured step follows the state on the GPU: contexts grow, pages are taken."""
    model = Llama3Decoder(TINY, batch=1, max_ctx=64)
    eager, replayed = (ng.TreeDecoder(model, 2, 16, page_size=8) for _ in range(2))
    text = [draw(6, 1), draw(13, 2)]
    for dec in (eager, replayed):
        first = dec.step(tokens_of(text), ints([6, 13]))
    parents = [[-1, 0, 0, 1], [-1, 0, 1, 1, 0]] if trees else None
    n = ints([4, 5] if trees else [1, 1])
    flat = None if parents is None else ints(parents[0] + parents[1])

    def run(dec, tokens):
        return dec.step(tokens, n, flat, max_tree=5, max_path=3)

    def feed(tokens, step):  # node 0 of each request is its next token; all drafts say the same
        if not trees:
            return tokens.clone()
        return torch.cat([torch.cat([tokens[b:b + 1], torch.full((m - 1,), 3 + step, dtype=torch.int64, device="cuda")])
                          for b, m in enumerate((4, 5))])

    run(ng.TreeDecoder(model, 2, 16, page_size=8), feed(first.tokens, 0))
    torch.cuda.synchronize()
    tokens = torch.zeros(9 if trees else 2, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(replayed, tokens)
        logits = replayed.logits
    want = first
    known = first.tokens.clone()
    for step in range(7):
        want = run(eager, feed(known, step))
        tokens.copy_(feed(known, step))
        graph.replay()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(logits, eager.logits)
        for x, y in ((replayed.cached, eager.cached), (replayed.cursor, eager.cursor), (replayed.table, eager.table)):
            assert torch.equal(x, y)
        known = want.tokens.clone()
    assert eager.cursor.item() > 3  # pages were taken on the way
    assert ng.extension().device_status() == 0
