"""``TreeDecoder`` (ragged prompts, drafted trees, paged cache) against the plain
fp32 restatement of the model fed one token at a time along each path.  Gate as
for the decode step: max|err| / max|ref| <= 2e-2 (fp16) / 4e-2 (bf16) on the logits.
What is accepted follows from the model's own tokens, so it is checked exactly."""
from __future__ import annotations

import pytest
import torch

import nibblegemm_b200 as ng
from nibblegemm_b200.decode_model import Llama3Decoder
from tests.test_decode_model import TINY, RefModel, _rel

pytestmark = pytest.mark.gpu


class Sequence:
    """The fp32 model on one token list."""

    def __init__(self, model):
        self.model = model

    def logits(self, tokens):
        ref = RefModel(self.model)
        for p, t in enumerate(tokens):
            _, out = ref.step(torch.tensor([t], device="cuda"), torch.tensor([p], device="cuda"))
        return out[0]


def make(dtype, requests, pages, **kw):
    model = Llama3Decoder(TINY, batch=1, max_ctx=64, dtype=dtype)
    return ng.TreeDecoder(model, requests, pages, **kw), Sequence(model)


def walk(tree_tokens, parents, next_tokens, limit):
    path = [0]
    while len(path) < limit:
        kids = [c for c in range(len(parents)) if parents[c] == path[-1] and tree_tokens[c] == next_tokens[path[-1]]]
        if not kids:
            break
        path.append(kids[0])
    return path


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_then_trees_follow_the_model(dtype):
    tol = 2e-2 if dtype == torch.float16 else 4e-2
    dec, seq = make(dtype, 3, 24, page_size=8)
    g = torch.Generator().manual_seed(0)
    draw = lambda n: torch.randint(0, TINY["vocab"], (n,), generator=g).tolist()  # noqa: E731
    text = [draw(21), draw(3), draw(9)]  # what each request's cache holds
    counts = torch.tensor([len(x) for x in text], dtype=torch.int32, device="cuda")
    out = dec.step(torch.tensor(sum(text, []), device="cuda"), counts)
    last = (counts.cumsum(0) - 1).long()
    for b in range(3):
        assert _rel(dec.logits[last[b]], seq.logits(text[b])) <= tol
    assert out.accepted.tolist() == counts.tolist() and out.granted.all()
    assert torch.equal(out.tokens, out.next_tokens[last])

    for _ in range(3):
        known = out.tokens.tolist()  # node 0 of each tree
        # trees of 7, 1 and 4 nodes; a first pass (undone below) tells what the model wants where
        parents = [[-1, 0, 0, 1, 1, 2, 3], [-1], [-1, 0, 1, 2]]
        n = torch.tensor([len(p) for p in parents], dtype=torch.int32, device="cuda")
        state = [x.clone() for x in (dec.cached, dec.held, dec.table, dec.cursor)]
        trees = [[known[b]] + draw(len(parents[b]) - 1) for b in range(3)]
        flat = torch.tensor(sum(parents, []), dtype=torch.int32, device="cuda")
        for attempt in range(3):  # each pass can put one more of the model's own tokens into the trees
            out = dec.step(torch.tensor(sum(trees, []), device="cuda"), n, flat, max_tree=7, max_path=4)
            start = [0, 7, 8, 12]
            wants = [out.next_tokens[start[b]:start[b + 1]].tolist() for b in range(3)]
            logits = dec.logits
            paths = [walk(trees[b], parents[b], wants[b], 4) for b in range(3)]
            assert out.accepted.tolist() == [len(p) for p in paths]
            assert [[c for c in r if c >= 0] for r in out.path.tolist()] == paths
            assert out.tokens.tolist() == [wants[b][paths[b][-1]] for b in range(3)]
            for b in range(3):  # every node's logits are those of the path that leads to it
                for node in range(len(parents[b])):
                    chain, up = [], node
                    while up >= 0:
                        chain.append(trees[b][up])
                        up = parents[b][up]
                    got = logits[start[b] + node]
                    assert _rel(got, seq.logits(text[b] + chain[::-1])) <= tol, (b, node)
            if attempt == 2:
                break
            for x, y in zip((dec.cached, dec.held, dec.table, dec.cursor), state):
                x.copy_(y)
            for b, p in enumerate(paths):  # one more node of each path agrees
                kids = [c for c in range(len(parents[b])) if parents[b][c] == p[-1]]
                if kids:
                    trees[b][kids[-1]] = wants[b][p[-1]]
        for b, p in enumerate(paths):
            text[b] += [trees[b][c] for c in p]
        assert dec.cached.tolist() == [len(x) for x in text]
        assert max(len(p) for p in paths) >= 3  # nodes did move in the cache
    # the kept rows are right: a plain token on top of them sees the whole text
    out = dec.step(out.tokens.clone(), torch.ones(3, dtype=torch.int32, device="cuda"))
    assert ng.extension().device_status() == 0


def test_per_head_norms_and_a_pool_that_runs_out():
    dec, _ = make(torch.float16, 2, 3, page_size=8)
    ones = [torch.ones(128, device="cuda", dtype=torch.float16) for _ in range(2)]
    dec.q_norm = dec.k_norm = ones
    n = torch.tensor([17, 10], dtype=torch.int32, device="cuda")  # 3 pages and 2: the pool has 3
    out = dec.step(torch.arange(27, device="cuda"), n)
    assert out.granted.tolist() == [True, False]
    assert out.accepted.tolist() == [17, 0] and dec.cached.tolist() == [17, 0]
    assert out.tokens[1].item() == -1 and 0 <= out.tokens[0].item() < TINY["vocab"]
    assert dec.held.tolist() == [3, 0] and dec.cursor.item() == 3
    with pytest.raises(ValueError):
        dec.step(torch.zeros(3, device="cuda"), n)
    assert ng.extension().device_status() == 0
