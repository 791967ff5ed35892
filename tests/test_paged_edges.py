"""Edges of the paged operators: requests that outgrow their row of the table, the
largest lengths, tokens of no request, and small fp16 probabilities."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import nibblegemm_b200 as ng
from tests import test_paged as tp
from tests.test_paged import ints

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- plan
def planned(cached, new, held, width, free, page):
    """What each request gets: a request that does not fit its row of the table, or whose
    pages are not there, gets nothing; only the others' pages count."""
    off, kv, held_out, fresh = 0, [], [], []
    for c, n, h in zip(cached, new, held):
        blocks = -(-(c + n) // page)
        need = max(0, blocks - h) if blocks <= width else 0
        granted = blocks <= width and (need == 0 or off + need <= len(free))
        fresh.append(free[off:off + need] if granted else [])
        kv.append(c + n if granted else 0)
        held_out.append(max(h, blocks) if granted else h)
        off += need
    return kv, held_out, fresh


@pytest.mark.parametrize("B,width,short", [(3, 2, 0), (40, 5, 0), (40, 5, 6), (700, 9, 0), (700, 9, 200)])
def test_plan_of_requests_that_outgrow_the_table(B, width, short):
    rng = np.random.default_rng(B + short)
    page = 16
    cached = rng.integers(0, width * page + 1, B)
    new = rng.integers(0, 2 * page, B)  # some end beyond their row
    cached[0], new[0] = width * page, 1  # the first one among them
    new[1:] = np.where(rng.random(B - 1) < 0.5, np.minimum(new[1:], width * page - cached[1:]), new[1:])
    held = -(-cached // page)
    blocks = -(-(cached + new) // page)
    assert (blocks > width).any() and (blocks[1:] > held[1:]).any()
    need = int(np.where(blocks <= width, np.maximum(blocks - held, 0), 0).sum())
    pool = rng.permutation(int(held.sum()) + need + 20).tolist()
    table = np.full((B, width), -1, np.int64)
    for b in range(B):
        table[b, :held[b]] = [pool.pop() for _ in range(held[b])]
    free = pool[:need - short]  # exactly the pages that are needed, or too few
    kv, held_out, fresh = planned(cached, new, held, width, free, page)
    tab = ints(table)
    p = ng.paged_plan(ints(cached), ints(new), ints(held), tab, ints(free), page_size=page, num_tokens=int(new.sum()))
    for b in range(B):
        table[b, held[b]:held[b] + len(fresh[b])] = fresh[b]
    assert tab.tolist() == table.tolist()
    assert p.kv_lens.tolist() == kv and p.held.tolist() == list(map(int, held_out))
    assert p.taken.item() == sum(map(len, fresh))  # no page is counted that nobody has
    slots, cu = p.slots.cpu().numpy(), p.cu_new.tolist()
    for b in range(B):
        at = cached[b] + np.arange(new[b])
        want = table[b, np.minimum(at // page, width - 1)] * page + at % page if kv[b] else np.full(new[b], -1)
        assert slots[cu[b]:cu[b + 1]].tolist() == want.tolist()
    tp.assert_clean()


@pytest.mark.parametrize("cached,new", [(2**30, 2**30), (2**30 - 1, 2**30 - 1), (2**30 - 1, 4), (5, 2**30), (2**31 - 1, 8)])
@pytest.mark.parametrize("page", [8, 1024])
def test_plan_of_the_largest_lengths(cached, new, page):
    """Lengths that no table holds are refused, not wrapped around to small ones."""
    tab = ints([[0, -1, -1], [1, -1, -1]])
    before = tab.clone()
    p = ng.paged_plan(ints([3, cached]), ints([2, new]), ints([1, 1]), tab, ints([4, 5, 6]), page_size=page, num_tokens=10)
    assert p.kv_lens.tolist() == [5, 0] and p.held.tolist() == [1, 1] and p.taken.item() == 0
    assert p.slots.tolist() == [3, 4] + [-1] * 8
    assert torch.equal(tab, before)
    over = cached >= 2**30 or new >= 2**30 or new > 8  # the last: more tokens than there is room for
    assert ng.extension().device_status() == (10 if over else 0)


@pytest.mark.parametrize("words", [0, 2])
def test_plan_without_tokens(words):
    """A step of trees in which no request has a token."""
    tab = ints([[3, -1], [5, 6]])
    p = ng.paged_plan(ints([7, 20]), ints([0, 0]), ints([1, 2]), tab, ints([8]), page_size=16, num_tokens=0,
                      parents=ints([]), mask_words=words)
    assert p.cu_new.tolist() == [0, 0, 0] and p.kv_lens.tolist() == [7, 20] and p.held.tolist() == [1, 2]
    assert p.taken.item() == 0 and p.slots.shape == (0,) and p.positions.shape == (0,)
    assert (p.mask is None) if words == 0 else (p.mask.shape == (0, words))
    assert tab.tolist() == [[3, -1], [5, 6]]
    tp.assert_clean()


@pytest.mark.parametrize("tokens", [0, 4])
@pytest.mark.parametrize("words", [0, 1])
def test_plan_without_requests(tokens, words):
    p = ng.paged_plan(ints([]), ints([]), ints([]), torch.zeros(0, 3, dtype=torch.int32, device="cuda"), ints([1, 2]),
                      page_size=16, num_tokens=tokens, parents=ints([-1] * tokens) if words else None, mask_words=words)
    assert p.cu_new.tolist() == [0] and p.kv_lens.shape == (0,) and p.held.shape == (0,) and p.taken.tolist() == [0]
    assert p.slots.tolist() == [-1] * tokens and p.positions.tolist() == [0] * tokens
    assert (p.mask is None) if words == 0 else p.mask.tolist() == [[0]] * tokens
    tp.assert_clean()


# --------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_without_requests(dim):
    """Tokens of no request give zeros, also when there are no requests at all."""
    k, v = ng.paged_cache(2, 16, 2, dim)
    q = torch.randn(5, 4, dim, device="cuda").half()
    out = torch.full_like(q, 7.0)
    got, lse = ng.tree_attention(q, k, v, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), ints([]), ints([0]),
                                 return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (got == 0).all() and (lse == -float("inf")).all()
    tp.assert_clean()


@pytest.mark.parametrize("first", [1, 40, 500])
@pytest.mark.parametrize("end", [0, 3])
def test_attention_rows_in_front_of_the_first_request(first, end):
    rng = np.random.default_rng(0)
    k, v, table = tp.build_pages(rng, [50, 20], 16, 2, 128, torch.float16, False)
    T = first + 9 + end
    q = torch.randn(T, 4, 128, device="cuda").half()
    out = torch.full_like(q, 7.0)
    cu = [first, first + 4, first + 9]
    got, lse = ng.tree_attention(q, k, v, table, ints([50, 20]), ints(cu), return_lse=True, out=out)
    assert (got[:first] == 0).all() and (lse[:first] == -float("inf")).all()
    assert (got[cu[2]:] == 0).all() and (lse[cu[2]:] == -float("inf")).all()
    want = ng.tree_attention(q[first:cu[2]], k, v, table, ints([50, 20]), ints([0, 4, 9]))
    assert torch.equal(got[first:cu[2]], want)
    tp.assert_clean()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tall_at", [0, 40, 63])
@pytest.mark.parametrize("new", [1, 5])
def test_attention_small_fp16_probabilities(dim, tall_at, new):
    """Keys whose probability is 2^-25.5 of the largest still count in the output.

    fp16 has no value below 2^-24 of its own unit, but the kernel's probabilities reach up to
    2^15, so none above 2^-33 of the row's largest is lost: each is off by at most 2^-32."""
    page, kv, big = 16, 64 + new - 1, 1024.0
    k, v = ng.paged_cache(8, page, 1, dim)
    table = ints([range(8)])
    q = torch.zeros(new, 2, dim, device="cuda", dtype=torch.float16)
    q[..., 0] = 1
    rows = torch.arange(kv, device="cuda")
    height = torch.full((kv,), -25.5, device="cuda")
    height[tall_at] = 0
    k[rows // page, rows % page, 0, 0] = height.half()  # exact; scores in base 2
    value = torch.full((kv,), big, device="cuda")
    value[tall_at] = 0
    v[rows // page, rows % page, 0] = value.half()[:, None]
    scale = float(np.log(2.0))
    got, lse = ng.tree_attention(q, k, v, table, ints([kv]), ints([0, new]), scale=scale, return_lse=True)
    for i in range(new):
        seen = kv - new + i + 1
        p = torch.exp2(height[:seen].double())
        want = (p * value[:seen].double()).sum() / p.sum()
        # rounding of the result and of P, fp32 scores (25.5 * 2^-24 of a unit), and 2^-32 for each key
        tol = want * (2 * 2.0**-11 + 1e-5) + seen * 2.0**-32 * big + 2.0**-25
        assert want > 4 * tol  # all of it would be missed otherwise
        assert ((got[i].double() - want).abs() <= tol).all()
        assert ((lse[i].double() - p.sum().log()).abs() <= 1e-6).all()
    tp.assert_clean()


@pytest.mark.parametrize("dtype", tp.DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_lse_of_equal_scores(dtype, dim):
    """With queries of zeros every visible key weighs the same: lse is the logarithm of their number."""
    rng = np.random.default_rng(dim)
    new, kv = [3, 1, 70, 2], [700, 9001, 300, 2]
    k, v, table = tp.build_pages(rng, kv, 16, 2, dim, dtype, False)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.zeros(int(cu[-1]), 4, dim, device="cuda", dtype=dtype)
    got, lse = ng.tree_attention(q, k, v, table, ints(kv), ints(cu), return_lse=True)
    tp.check_attn(got, lse, tp.attn_reference(q, k, v, table, kv, cu, None, dim**-0.5), dtype)
    seen = np.concatenate([np.arange(L - n + 1, L + 1) for n, L in zip(new, kv)])
    want = torch.as_tensor(np.log(seen), device="cuda")[:, None]
    assert ((lse.double() - want).abs() <= 2e-7 * want + 5e-7).all()  # sums of ones are exact; log2 and one product
    tp.assert_clean()
