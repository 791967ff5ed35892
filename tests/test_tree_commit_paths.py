"""``tree_commit`` on trees whose kept path is long and leaves nodes out, so that many rows
move, over one another's places; also where the path ends at its limit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import nibblegemm_b200 as ng
from tests import test_paged as tp
from tests.test_paged import ints

pytestmark = pytest.mark.gpu


def drafted(rng, n, length):
    """A tree of n nodes and the model's tokens, of which a path of `length` nodes agrees."""
    path = [0] + sorted(rng.choice(np.arange(1, n), length - 1, replace=False).tolist())
    before = dict(zip(path[1:], path))
    parents = [-1] + [before.get(i, int(rng.integers(0, i))) for i in range(1, n)]
    nxt = rng.integers(0, 1 << 40, n)
    draft = rng.integers(1 << 41, 1 << 42, n)  # agrees with nothing
    for c, p in before.items():
        draft[c] = nxt[p]
    for c in range(1, n):  # younger brothers that agree as well must not be taken
        p = parents[c]
        if c not in before and p in path[:-1] and c > path[path.index(p) + 1] and rng.random() < 0.5:
            draft[c] = nxt[p]
    return parents, draft, nxt, path


CASES = [
    # new tokens of each request, agreeing nodes, limit, cached, layers, kv heads, D, page
    ([12], [7], 16, [13], 2, 2, 128, 8),
    ([64], [40], 64, [100], 3, 8, 128, 16),
    ([64, 1, 33, 64], [30, 1, 20, 17], 16, [5, 0, 31, 64], 2, 1, 64, 16),  # cut off at the limit
    ([200, 90], [180, 60], 512, [0, 300], 1, 5, 128, 64),
    ([40] * 30, [25] * 30, 32, [9] * 30, 4, 2, 64, 32),
    ([2048], [320], 512, [3], 1, 1, 64, 64),
    ([2049], [320], 512, [3], 1, 1, 64, 1024),
    ([4500, 2048, 7], [700, 600, 5], 512, [3, 70, 2], 1, 1, 64, 64),
    ([4500], [19], 17, [3], None, 2, 64, 16),
]


@pytest.mark.parametrize("dtype", tp.DTYPES)
@pytest.mark.parametrize("rows_first", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_long_paths(dtype, rows_first, case):
    new, agree, limit, ctx, layers, hk, dim, page = CASES[case]
    rng = np.random.default_rng(case)
    torch.manual_seed(case)
    trees = [drafted(rng, n, a) for n, a in zip(new, agree)]
    kv = np.array(ctx) + np.array(new)
    blocks = -(-kv // page)
    order = rng.permutation(int(blocks.sum()) + 1).tolist()
    table = np.full((len(new), int(blocks.max())), -1, np.int64)
    for b, m in enumerate(blocks):
        table[b, :m] = [order.pop() for _ in range(m)]
    k, v = (tp.make_cache(int(blocks.sum()) + 1, page, hk, dim, dtype, rows_first, layers) for _ in range(2))
    wk, wv = k.clone(), v.clone()
    paths = []
    for b, (parents, draft, nxt, path) in enumerate(trees):
        path = path[:limit]
        paths.append(path)
        row = lambda c: (int(table[b, (ctx[b] + c) // page]), (ctx[b] + c) % page)  # noqa: E731
        for w, old in ((wk, k), (wv, v)):  # from the caches as they were
            for i, c in enumerate(path):
                w[..., row(i)[0], row(i)[1], :, :] = old[..., row(c)[0], row(c)[1], :, :]
    longest = max(paths, key=len)
    assert len(longest) > 4 and sum(c != i for i, c in enumerate(longest)) > 4
    assert (max(agree) > limit) == (len(longest) == limit)
    to = lambda a, t: torch.as_tensor(np.concatenate(a), dtype=t, device="cuda")  # noqa: E731
    c = ng.tree_commit(to([t[1] for t in trees], torch.int64), to([t[0] for t in trees], torch.int32),
                       to([t[2] for t in trees], torch.int64), ints(np.concatenate([[0], np.cumsum(new)])), ints(kv),
                       ints(table), k, v, max_path=limit)
    assert c.path.tolist() == [p + [-1] * (limit - len(p)) for p in paths]
    assert c.accepted.tolist() == list(map(len, paths))
    assert c.bonus.tolist() == [int(t[2][p[-1]]) for t, p in zip(trees, paths)]
    assert c.kv_lens.tolist() == [x + len(p) for x, p in zip(ctx, paths)]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    tp.assert_clean()
