"""The paged operators on caches whose strides are not the usual ones, on rows that
belong to no request, and on trees too large for the commit's shared memory.  References
and tolerances are those of ``test_paged.py``."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import nibblegemm_b200 as ng
from tests import test_paged as tp

pytestmark = pytest.mark.gpu


def relaid(cache, how):
    """The same [pages, page, heads, dim] values under other strides; what lies between is NaN."""
    pages, page, heads, dim = cache.shape
    new = lambda *s: torch.full(s, float("nan"), dtype=cache.dtype, device="cuda")  # noqa: E731
    if how == "layers in a page":  # [pages, layers, heads, page, dim]
        view = new(pages, 3, heads, page, dim)[:, 1].transpose(1, 2)
    elif how == "k and v in a row":  # [pages, page, heads, 2, dim]
        view = new(pages, page, heads, 2, dim)[..., 0, :]
    elif how == "some of the heads":  # [pages, page, heads + 2, dim]
        view = new(pages, page, heads + 2, dim)[:, :, 1:1 + heads]
    else:  # heads outermost: [heads, pages, page, dim]
        view = new(heads, pages, page, dim).permute(1, 2, 0, 3)
    view.copy_(cache)
    return view


@pytest.mark.parametrize("how", ["layers in a page", "k and v in a row", "some of the heads", "heads outermost"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("hk", [1, 3])
def test_attention_strides(how, dim, page, hk):
    rng = np.random.default_rng(page + dim)
    torch.manual_seed(page + dim)
    dtype = torch.bfloat16
    new, kv = [5, 1, 40], [300, 64, 171]
    k, v, table = tp.build_pages(rng, kv, page, hk, dim, dtype, False)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(46, 4 * hk, dim, device="cuda").to(dtype)
    mask = tp.random_mask(rng, new, 1)
    for m in (None, mask):
        got, lse = ng.tree_attention(q, relaid(k, how), relaid(v, how), table, tp.ints(kv), tp.ints(cu), return_lse=True,
                                     mask=None if m is None else torch.as_tensor(m.view(np.int64), device="cuda"))
        tp.check_attn(got, lse, tp.attn_reference(q, k, v, table, kv, cu, m, dim**-0.5), dtype)
    tp.assert_clean()


@pytest.mark.parametrize("rows_first", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_split_over_every_cta(rows_first, dim):
    """A few long items in many parts, beside short ones, with 1, 3 and 128 rows to a tile."""
    rng = np.random.default_rng(dim)
    torch.manual_seed(dim)
    for hq, hk, new, kv in ((1, 1, [1], [9001]), (6, 2, [1, 1], [7000, 40]), (16, 1, [20, 3], [5000, 90]),
                            (8, 2, [70, 64, 33], [2600, 2048, 700])):
        k, v, table = tp.build_pages(rng, kv, 16, hk, dim, torch.float16, rows_first)
        cu = np.concatenate([[0], np.cumsum(new)])
        q = (torch.randn(int(cu[-1]), hq, dim, device="cuda") * 2).half()
        mask = tp.random_mask(rng, new, 2)
        for m in (None, mask):
            got, lse = ng.tree_attention(q, k, v, table, tp.ints(kv), tp.ints(cu), return_lse=True,
                                         mask=None if m is None else torch.as_tensor(m.view(np.int64), device="cuda"))
            tp.check_attn(got, lse, tp.attn_reference(q, k, v, table, kv, cu, m, dim**-0.5), torch.float16)
    tp.assert_clean()


def test_attention_rows_of_no_request():
    rng = np.random.default_rng(0)
    k, v, table = tp.build_pages(rng, [50], 16, 2, 128, torch.float16, False)
    q = torch.randn(9, 4, 128, device="cuda").half()
    out = torch.full_like(q, 7.0)
    got, lse = ng.tree_attention(q, k, v, table, tp.ints([50]), tp.ints([0, 4]), return_lse=True, out=out)
    assert (got[4:] == 0).all() and (lse[4:] == -float("inf")).all()
    assert torch.equal(got[:4], ng.tree_attention(q[:4], k, v, table, tp.ints([50]), tp.ints([0, 4])))
    tp.assert_clean()


@pytest.mark.parametrize("new,limit", [(2048, 16), (2049, 300), (4500, 7)])
def test_commit_of_large_trees(new, limit):
    tp.test_commit(torch.float16, [3], [new], 1, 1, 64, 64, limit, False)
