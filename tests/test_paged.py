"""The paged-cache operators (``nibblegemm_b200/paged.py``) against plain
implementations in 64 bits, at the sizes, masks, layouts and contents where such
kernels go wrong.

Tolerances, with u the unit roundoff of the activation type (8 bits of significand in bf16: 2^-8; 11 in fp16: 2^-11):

* norm + rotation: one rounding of the result, u |y|, and fp32 arithmetic before
  it: ten operations or so on values of the rotated pair's length, 2e-6 of that
  length (and half the smallest fp16 subnormal, 2^-25).
* attention: u |y| for the rounding of the result; the probabilities are rounded
  to the activation type before the product with V, u A with A = sum_j p_j |v_j|;
  the scores carry fp32 rounding errors (below 5e-5 for the values used here), so
  1e-4 A; and fp16 probabilities below 2^-14 of the row's largest are subnormal:
  2^-25 max|v| for each key.
* lse: the scores' error, 5e-5, and fp32 rounding of the result, 2e-7 |lse|.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import nibblegemm_b200 as ng
from nibblegemm_b200 import _lib

gpu = pytest.mark.gpu

UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
DTYPES = [torch.float16, torch.bfloat16]
THETA = 500000.0


def ints(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def assert_clean():
    assert ng.extension().device_status() == 0


# --------------------------------------------------------------------------- plan
def plan_reference(cached, new, held, table, free, page, capacity, parents, words, cursor=0):
    table = table.copy()
    B, width = table.shape
    cu = [0]
    slots, positions = np.full(capacity, -1, np.int64), np.zeros(capacity, np.int64)
    mask = np.zeros((capacity, words), np.uint64)
    kv, held_out, taken, off = [], [], 0, 0
    for b in range(B):
        blocks = -(-(cached[b] + new[b]) // page)
        need = max(0, blocks - held[b])
        granted = (need == 0 or off + need <= len(free) - cursor) and blocks <= width
        if granted:
            for i in range(need):
                table[b, held[b] + i] = free[cursor + off + i]
            if need:
                taken = off + need
        for i in range(new[b]):
            t = cu[b] + i
            at = cached[b] + i
            if granted:
                slots[t] = table[b, at // page] * page + at % page
            node, depth = i, 0
            if parents is None:
                depth = i
            else:
                while True:
                    if words:
                        mask[t, node // 64] |= np.uint64(1) << np.uint64(node % 64)
                    if parents[cu[b] + node] < 0:
                        break
                    node = parents[cu[b] + node]
                    depth += 1
            positions[t] = cached[b] + depth
        off += need
        cu.append(cu[b] + new[b])
        kv.append(cached[b] + new[b] if granted else 0)
        held_out.append(max(held[b], blocks) if granted else held[b])
    return dict(cu_new=cu, slots=slots, positions=positions, kv_lens=kv, held=held_out, taken=[taken], table=table,
                mask=mask.view(np.int64))


def random_parents(rng, new):
    out = []
    for n in new:
        out += [-1 if i == 0 or rng.random() < 0.03 else int(rng.integers(0, i)) for i in range(n)]
    return np.array(out, np.int64)


@gpu
@pytest.mark.parametrize("B,page,most_cached,most_new,tree,short", [
    (1, 16, 0, 1, False, 0), (1, 8, 100, 1, True, 0), (2, 64, 1000, 3, True, 0), (33, 16, 300, 64, True, 0),
    (300, 32, 4000, 5, False, 0), (40, 16, 100, 130, True, 0), (257, 1024, 5000, 2000, False, 0),
    (64, 8, 200, 40, False, 70), (64, 16, 500, 30, True, 25), (1000, 16, 50, 3, False, 0)])
def test_plan(B, page, most_cached, most_new, tree, short):
    rng = np.random.default_rng(B * 1000 + page)
    cached = rng.integers(0, most_cached + 1, B)
    new = rng.integers(0, most_new + 1, B)
    if B == 1:
        new[0] = most_new
    held = -(-cached // page) + (rng.random(B) < 0.2)  # some hold a page more than they fill
    blocks = np.maximum(-(-(cached + new) // page), held)
    width = int(blocks.max()) + 2
    pool = rng.permutation(int(blocks.sum()) + 50)
    table = np.full((B, width), -1, np.int64)
    used = 0
    for b in range(B):
        table[b, :held[b]] = pool[used:used + held[b]]
        used += held[b]
    needed = int((np.maximum(blocks - held, 0)).sum())
    cursor = 3
    free = pool[used:used + max(0, needed + cursor - short)]
    extra = 5 if B % 2 else 0
    capacity = int(new.sum()) + extra
    parents = random_parents(rng, new) if tree else None
    words = -(-most_new // 64) if tree else 0
    want = plan_reference(cached, new, held, table, free, page, capacity, parents, words, cursor)
    padded = None if parents is None else ints(np.concatenate([parents, np.full(extra, -1)]))
    wide = torch.full((B, width + 3), -7, dtype=torch.int32, device="cuda")  # rows lie apart
    wide[:, :width] = ints(table)
    inputs = ints(cached), ints(new), ints(held)
    before = [x.clone() for x in inputs]
    plan = ng.paged_plan(*inputs, wide[:, :width], ints(free), page_size=page, num_tokens=capacity, parents=padded,
                         mask_words=words, cursor=ints([cursor]))
    for name in ("cu_new", "slots", "positions", "kv_lens", "held", "taken"):
        assert getattr(plan, name).cpu().tolist() == list(map(int, want[name])), name
    assert wide[:, :width].cpu().tolist() == want["table"].tolist()
    assert (wide[:, width:] == -7).all()
    if words:
        assert plan.mask.cpu().numpy().tolist() == want["mask"].tolist()
    else:
        assert plan.mask is None
    for x, y in zip(inputs, before):
        assert torch.equal(x, y)
    assert_clean()


@gpu
@pytest.mark.parametrize("what", ["negative", "capacity", "parent", "cycle", "mask", "unmapped"])
def test_plan_reports_bad_inputs(what):
    cached, new, held = [5, 17], [4, 3], [1, 2]
    parents, words, capacity = [-1, 0, 1, 1, -1, 0, 1], 1, 7
    table = [[3, -1], [1, 2]]
    if what == "negative":
        cached = [-5, 17]
    if what == "capacity":
        capacity = 6
    if what == "parent":
        parents[2] = 3
    if what == "cycle":
        parents[6] = 2
    if what == "mask":
        cached, new, held, capacity = [0, 0], [70, 1], [0, 0], 71
        parents = [-1] + list(range(69)) + [-1]
        table = [[-1] * 8, [-1] * 8]
    if what == "unmapped":
        table = [[-1, -1], [1, 2]]
    assert_clean()
    ng.paged_plan(ints(cached), ints(new), ints(held), ints(table), ints(range(4, 14)), page_size=16,
                  num_tokens=capacity, parents=ints(parents[:capacity]), mask_words=words)
    assert ng.extension().device_status() == 10
    assert_clean()


# --------------------------------------------------------------------------- norm + rotation
def make_cache(pages, page, heads, dim, dtype, rows_first, layers=None, fill=None):
    lead = () if layers is None else (layers,)
    shape = (pages, page, heads, dim) if rows_first else (pages, heads, page, dim)
    c = torch.randn(*lead, *shape, device="cuda").to(dtype) if fill is None else \
        torch.full((*lead, *shape), fill, device="cuda", dtype=dtype)
    return c if rows_first else c.transpose(-3, -2)


def norm_reference(x, w, angle, half, eps):
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    a, b = y[..., :half], y[..., half:2 * half]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1), \
        torch.cat([(a * a + b * b).sqrt()] * 2 + [y[..., 2 * half:].abs()], -1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,hq,hk,dim,rot,page,normed,rows_first", [
    (1, 32, 8, 128, 128, 16, True, False), (1, 1, 1, 64, 64, 8, True, True), (3, 5, 1, 64, 32, 16, True, False),
    (7, 28, 4, 128, 64, 64, False, True), (33, 8, 8, 256, 256, 32, True, False), (130, 6, 2, 128, 96, 128, True, True),
    (257, 64, 8, 128, 128, 16, True, False), (5, 3, 3, 128, 0, 16, True, False), (4, 2, 1, 256, 16, 1024, False, False),
    (6000, 16, 2, 64, 64, 16, True, True)])
def test_norm_rope_append(dtype, M, hq, hk, dim, rot, page, normed, rows_first):
    torch.manual_seed(M + hq + dim)
    rng = np.random.default_rng(M)
    heads, eps = hq + 2 * hk, 1e-5
    wide = (torch.randn(M, heads * dim + 8, device="cuda") * 3).to(dtype)
    wide[0, :dim] = 0  # a head of zeros stays zeros
    qkv = wide[:, :heads * dim]  # rows lie apart
    pages = -(-M // page) + 2
    k, v = (make_cache(pages, page, hk, dim, dtype, rows_first) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    slots = rng.permutation(pages * page)[:M]
    slots[rng.random(M) < 0.1] = -1
    positions = rng.integers(0, 1 << 20, M)
    positions[0] = 2**31 - 1 if M > 1 else 0
    wq, wk = ((1 + 0.2 * torch.randn(dim, device="cuda")).to(dtype) if normed else None for _ in range(2))
    q = ng.qk_norm_rope_append(qkv, wq, wk, ng.rope_turns(rot, THETA), ints(positions), ints(slots), k, v, q_heads=hq,
                               eps=eps)
    half = rot // 2
    freq = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / max(1, half))
    angle = torch.as_tensor(positions, device="cuda").double()[:, None] * freq
    x = qkv.reshape(M, heads, dim)
    rq, lq = norm_reference(x[:, :hq], wq, angle, half, eps)
    rk, lk = norm_reference(x[:, hq:hq + hk], wk, angle, half, eps)
    u = UNIT[dtype]
    assert q.shape == (M, hq, dim) and q.dtype == dtype
    assert ((q.double() - rq).abs() <= u * rq.abs() + 2e-6 * lq + 2.0**-25).all()
    sl = torch.as_tensor(slots, device="cuda")
    keep = sl >= 0
    at = (sl[keep] // page, sl[keep] % page)
    err = (k[at].double() - rk[keep]).abs()
    assert (err <= u * rk[keep].abs() + 2e-6 * lk[keep] + 2.0**-25).all()
    assert torch.equal(v[at], x[keep][:, hq + hk:])
    k0[at], v0[at] = k[at], v[at]
    assert torch.equal(k, k0) and torch.equal(v, v0)  # nothing else was written
    assert_clean()


@gpu
def test_norm_rope_append_reports_a_slot_past_the_pool():
    k, v = (make_cache(2, 16, 1, 64, torch.float16, False, fill=2.0) for _ in range(2))
    qkv = torch.ones(3, 3 * 64, device="cuda", dtype=torch.float16)
    q = ng.qk_norm_rope_append(qkv, None, None, ng.rope_turns(0), ints([0, 1, 2]), ints([32, -5, 3]), k, v, q_heads=1)
    assert ng.extension().device_status() == 10
    assert (q == 1).all() and (k == 1).sum() == 64 and (v == 1).sum() == 64
    empty = ng.qk_norm_rope_append(qkv[:0], None, None, ng.rope_turns(0), ints([]), ints([]), k, v, q_heads=1)
    assert empty.shape == (0, 1, 64)


# --------------------------------------------------------------------------- attention
def build_pages(rng, kv, page, hk, dim, dtype, rows_first, spare=2, stale=float("nan")):
    """Caches whose unused rows and pages hold `stale`, and the block table."""
    kv = np.asarray(kv)
    blocks = -(-kv // page)
    pool = int(blocks.sum()) + spare
    order = rng.permutation(pool)
    table = np.full((len(kv), int(blocks.max(initial=1)) + 1), -1, np.int64)
    k, v = (make_cache(pool, page, hk, dim, dtype, rows_first, fill=stale) for _ in range(2))
    used = 0
    for b, n in enumerate(blocks):
        ids = order[used:used + n]
        used += n
        table[b, :n] = ids
        rows = torch.arange(int(kv[b]), device="cuda")
        pg = torch.as_tensor(ids, device="cuda")[rows // page] if len(rows) else rows
        for c in (k, v):
            c[pg, rows % page] = torch.randn(len(rows), hk, dim, device="cuda").to(dtype)
    return k, v, ints(table)


def sees_of(mask, first, n, kv):
    """[n, kv] truth values: what each new token of a request sees."""
    ctx = int(max(0, kv - n))
    sees = np.ones((n, kv), bool)
    for i in range(n):
        for key in range(ctx, kv):
            j = key - ctx
            if mask is None:
                sees[i, key] = j <= i
            else:
                word = int(mask[first + i, j // 64]) if j // 64 < mask.shape[1] else 0
                sees[i, key] = (word >> (j % 64)) & 1
    return torch.as_tensor(sees, device="cuda")


def attn_reference(q, k, v, table, kv, cu, mask, scale):
    """fp64 outputs, lse and A = sum_j p_j |v_j|, with sums over visible keys only."""
    T, hq, dim = q.shape
    page, hk = k.shape[1], k.shape[2]
    out, lse, A = (torch.zeros(T, hq, d, dtype=torch.float64, device="cuda") for d in (dim, 1, dim))
    lse -= math.inf
    vmax = torch.zeros(T, 1, 1, dtype=torch.float64, device="cuda")
    for b in range(len(kv)):
        n, L = cu[b + 1] - cu[b], int(kv[b])
        if n == 0 or L == 0:
            continue
        pages = table[b, :-(-L // page)].long()
        K = k[pages].reshape(-1, hk, dim)[:L].double()
        V = v[pages].reshape(-1, hk, dim)[:L].double()
        sees = sees_of(mask, cu[b], n, L)
        rows = slice(cu[b], cu[b + 1])
        Q = q[rows].double().view(n, hk, hq // hk, dim)
        s = torch.einsum("nhgd,khd->nhgk", Q, K) * scale
        s = torch.where(sees[:, None, None], s, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        hidden = ~sees.any(0)  # a key that no row sees must not matter, whatever it holds
        Vc = torch.where(hidden[:, None, None], 0.0, V)
        some = total > 0
        p = torch.where(some, p / total, 0.0)
        out[rows] = torch.einsum("nhgk,khd->nhgd", p, Vc).reshape(n, hq, dim)
        A[rows] = torch.einsum("nhgk,khd->nhgd", p, Vc.abs()).reshape(n, hq, dim)
        lse[rows] = torch.where(some, m + total.log(), -math.inf).reshape(n, hq, 1)
        vmax[rows] = Vc.abs().max() * L
    return out, lse[..., 0], A, vmax


def check_attn(got, lse, want, dtype):
    out, ref_lse, A, vmax = want
    u = UNIT[dtype]
    tol = u * out.abs() + (u + 1e-4) * A + (2.0**-25 * vmax if dtype == torch.float16 else 0) + 2.0**-25
    assert torch.isfinite(got).all()
    worst = ((got.double() - out).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1, worst
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse.double() - ref_lse).abs()[~empty] <= 5e-5 + 2e-7 * ref_lse.abs()[~empty]).all()
    assert (got[empty] == 0).all()


def random_mask(rng, new, words, empty=0.05):
    """Ancestor bits of random trees; some rows see nothing of the tree, and
    bits beyond the request's tokens are set, which must not matter."""
    rows = []
    for n in new:
        anc = []
        for i in range(n):
            bits = 1 << i
            if i:
                bits |= anc[int(rng.integers(0, i))]
            anc.append(bits)
        for bits in anc:
            bits = 0 if rng.random() < empty else bits
            bits |= (1 << (64 * words)) - (1 << n) if n < 64 * words and rng.random() < 0.5 else 0
            rows.append([(bits >> (64 * w)) & (2**64 - 1) for w in range(words)])
    m = np.array(rows, np.uint64).reshape(len(rows), words)
    return m


CASES = [
    # contexts, new tokens, q heads, kv heads, D, page, tree, rows first
    ([0], [1], 1, 1, 128, 16, False, False),
    ([1], [1], 4, 1, 64, 8, False, True),
    ([776], [1], 32, 8, 128, 16, False, False),
    ([127, 128, 129, 0, 5], [1, 1, 1, 1, 1], 8, 2, 128, 32, False, False),
    ([0, 3, 250], [0, 2, 5], 6, 2, 64, 16, False, True),
    ([100, 31, 0, 600], [16, 5, 40, 1], 32, 8, 128, 64, True, False),
    ([130, 0, 17], [64, 64, 33], 16, 2, 64, 128, True, False),
    ([60, 300], [70, 130], 8, 2, 128, 16, True, True),
    ([1000, 5], [61, 3], 28, 4, 128, 1024, True, False),
    ([0], [257], 4, 4, 128, 16, False, False),
    ([500, 64, 0], [200, 300, 64], 8, 1, 64, 64, False, True),
    ([9000], [4], 16, 1, 128, 64, True, False),
    ([20000, 1], [1, 1], 64, 8, 128, 16, False, False),
    ([40], [9], 96, 1, 128, 8, True, False),
    ([33, 70], [3, 2], 128, 1, 64, 16, True, False),
    (list(range(0, 600, 3)), [1] * 200, 8, 2, 128, 16, False, False),
    ([7, 0, 0, 300, 0, 2], [0, 0, 3, 0, 1, 0], 4, 2, 128, 16, True, False),
    ([3000] * 5, [33] * 5, 20, 4, 64, 256, True, False),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(dtype, case):
    ctx, new, hq, hk, dim, page, tree, rows_first = CASES[case]
    rng = np.random.default_rng(case)
    torch.manual_seed(case)
    kv = np.array(ctx) + np.array(new)
    k, v, table = build_pages(rng, kv, page, hk, dim, dtype, rows_first)
    cu = np.concatenate([[0], np.cumsum(new)])
    T = int(cu[-1])
    wide = (torch.randn(T, hq + 1, dim + 8, device="cuda") * 2).to(dtype)
    q = wide[:, :hq, :dim]  # rows and heads lie apart
    mask = random_mask(rng, new, max(1, -(-max(new) // 64))) if tree else None
    scale = dim**-0.5 * 1.3
    got, lse = ng.tree_attention(q, k, v, table, ints(kv), ints(cu),
                                 mask=None if mask is None else torch.as_tensor(mask.view(np.int64), device="cuda"),
                                 scale=scale, return_lse=True)
    check_attn(got, lse, attn_reference(q, k, v, table, kv, cu, mask, scale), dtype)
    again = ng.tree_attention(q, k, v, table, ints(kv), ints(cu),
                              mask=None if mask is None else torch.as_tensor(mask.view(np.int64), device="cuda"),
                              scale=scale)
    assert torch.equal(got, again)  # the same bits every time
    assert_clean()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,kvs", [(5, [0, 5, 3]), (1, [0, 1, 300])])
def test_attention_without_rows_to_see(dtype, n, kvs):
    """Requests that were not granted (kv 0), have no context, or fewer rows than tokens."""
    rng = np.random.default_rng(n)
    k, v, table = build_pages(rng, kvs, 16, 2, 64, dtype, False)
    q = torch.randn(3 * n, 4, 64, device="cuda").to(dtype)
    cu = [0, n, 2 * n, 3 * n]
    mask = np.zeros((3 * n, 1), np.uint64)
    for m in (None, mask):
        got, lse = ng.tree_attention(q, k, v, table, ints(kvs), ints(cu), return_lse=True,
                                     mask=None if m is None else torch.as_tensor(m.view(np.int64), device="cuda"))
        check_attn(got, lse, attn_reference(q, k, v, table, kvs, cu, m, 64**-0.5), dtype)
    assert_clean()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim,hq,n,ctx", [(128, 8, 6, 200), (64, 4, 70, 130), (128, 32, 40, 90)])
def test_attention_masked_places_may_hold_anything(dtype, bad, dim, hq, n, ctx):
    """A node whose keys and values are not finite reaches the rows that see it, and no others."""
    rng = np.random.default_rng(n)
    torch.manual_seed(n)
    page, hk, kv = 16, 2, ctx + n
    k, v, table = build_pages(rng, [kv], page, hk, dim, dtype, False)
    q = torch.randn(n, hq, dim, device="cuda").to(dtype)
    mask = random_mask(rng, [n], -(-n // 64), empty=0.0)
    words = torch.as_tensor(mask.view(np.int64), device="cuda")
    want = attn_reference(q, k, v, table, [kv], [0, n], mask, dim**-0.5)
    node = n // 2
    at = (table[0, (ctx + node) // page].long(), (ctx + node) % page)
    sees = sees_of(mask, 0, n, kv)[:, ctx + node]
    assert sees.any() and not sees.all()
    v[at[0], at[1], 0, 3] = bad
    got, lse = ng.tree_attention(q, k, v, table, ints([kv]), ints([0, n]), mask=words, return_lse=True)
    touched = torch.zeros_like(got, dtype=torch.bool)
    touched[sees, :hq // hk, 3] = True  # the heads that share that KV head
    hit = got[touched].float()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    check_attn(torch.where(touched, want[0].to(dtype), got), lse, want, dtype)
    v[at[0], at[1], 0, 3] = 0.5
    k[at[0], at[1]] = bad
    want = attn_reference(q, k, v, table, [kv], [0, n], mask, dim**-0.5)
    got, lse = ng.tree_attention(q, k, v, table, ints([kv]), ints([0, n]), mask=words, return_lse=True)
    check_attn(got[~sees], lse[~sees], [x[~sees] for x in want], dtype)
    if math.isnan(bad):
        assert torch.isnan(got[sees]).all() and torch.isnan(lse[sees]).all()
    assert_clean()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_and_equal_scores(dtype):
    """Scores of +-1000 that keep growing along the keys; and all equal."""
    torch.manual_seed(1)
    kv, dim, n = 700, 128, 3
    k, v, table = build_pages(np.random.default_rng(0), [kv], 16, 1, dim, dtype, False)
    rows = torch.arange(kv, device="cuda")
    pg = table[0].long()[rows // 16]
    q = torch.zeros(n, 2, dim, device="cuda", dtype=dtype)
    q[..., 0] = torch.tensor([16.0, -16.0], dtype=dtype, device="cuda")
    k[pg, rows % 16] = 0
    k[pg, rows % 16, 0, 0] = ((rows.float() - 350) * 2).to(dtype)
    got, lse = ng.tree_attention(q, k, v, table, ints([kv]), ints([0, n]), return_lse=True)
    out, ref, A, vmax = attn_reference(q, k, v, table, [kv], [0, n], None, dim**-0.5)
    # scores near 1000: fp32 rounding of score * log2(e) is up to 2^-14 of a unit
    tol = UNIT[dtype] * out.abs() + (UNIT[dtype] + 5e-4) * A + 2.0**-25 * (1 + vmax)
    assert ((got.double() - out).abs() <= tol).all()
    assert ((lse.double() - ref).abs() <= 5e-4).all()
    q.zero_()
    got = ng.tree_attention(q, k, v, table, ints([kv]), ints([0, n]))
    check_attn(got, *[attn_reference(q, k, v, table, [kv], [0, n], None, 1.0)[1].float()],
               attn_reference(q, k, v, table, [kv], [0, n], None, 1.0), dtype)


@gpu
def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 bytes per cache (and 2^31 values): pages at its far end."""
    page, hk, dim, dtype = 64, 8, 128, torch.float16
    pages = (1 << 32) // (page * hk * dim * 2) + 40
    k, v = (torch.zeros(pages, hk, page, dim, device="cuda", dtype=dtype).transpose(1, 2) for _ in range(2))
    ids = [pages - 1, 0, pages - 30, 7]
    torch.manual_seed(0)
    for i in ids:
        k[i], v[i] = (torch.randn(page, hk, dim, device="cuda").to(dtype) for _ in range(2))
    kv, n = 4 * page - 5, 3
    q = torch.randn(n, 32, dim, device="cuda").to(dtype)
    got, lse = ng.tree_attention(q, k, v, ints([ids]), ints([kv]), ints([0, n]), return_lse=True)
    check_attn(got, lse, attn_reference(q, k, v, ints([ids]), [kv], [0, n], None, dim**-0.5), dtype)
    qkv = torch.randn(1, (32 + 16) * dim, device="cuda").to(dtype)
    ng.qk_norm_rope_append(qkv, None, None, ng.rope_turns(0), ints([0]), ints([pages * page - 1]), k, v, q_heads=32)
    assert torch.equal(v[pages - 1, page - 1], qkv.view(48, dim)[40:])
    assert_clean()


@gpu
def test_attention_page_outside_the_pool_is_reported():
    k, v, table = build_pages(np.random.default_rng(0), [100, 40], 16, 1, 64, torch.float16, False, stale=0.0)
    q = torch.randn(2, 2, 64, device="cuda").half()
    want = ng.tree_attention(q, k, v, table, ints([100, 40]), ints([0, 1, 2]))
    assert_clean()
    for page in (-1, 1 << 20):
        bad = table.clone()
        bad[0, 2] = page
        got = ng.tree_attention(q, k, v, bad, ints([100, 40]), ints([0, 1, 2]))
        assert ng.extension().device_status() == 10
        assert torch.isfinite(got).all() and torch.equal(got[1], want[1])
    # a request that is longer than its row of the table
    ng.tree_attention(q, k, v, table[:, :3].contiguous(), ints([100, 40]), ints([0, 1, 2]))
    assert ng.extension().device_status() == 10


@gpu
def test_attention_on_another_stream_and_in_a_graph():
    rng = np.random.default_rng(3)
    k, v, table = build_pages(rng, [3000, 20], 16, 2, 128, torch.bfloat16, False)
    q = torch.randn(9, 8, 128, device="cuda").bfloat16()
    kv, cu = ints([3000, 20]), ints([0, 4, 9])
    want = ng.tree_attention(q, k, v, table, kv, cu)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ng.tree_attention(q, k, v, table, kv, cu)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    with torch.cuda.stream(side):
        ng.tree_attention(q, k, v, table, kv, cu, out=out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ng.tree_attention(q, k, v, table, kv, cu, out=out)
    q.mul_(0.5)
    kv.copy_(ints([1500, 9]))  # lengths are read on the GPU, so a replay follows them
    for _ in range(3):
        out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ng.tree_attention(q, k, v, table, kv, cu))
    assert_clean()


# --------------------------------------------------------------------------- commit
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,new,layers,hk,dim,page,limit,rows_first", [
    ([0], [1], None, 1, 64, 8, 4, False), ([13], [9], 2, 2, 128, 8, 16, True),
    ([100, 0, 31, 64], [32, 70, 0, 5], 3, 8, 128, 16, 16, False), ([5] * 40, [20] * 40, 2, 1, 64, 16, 3, False),
    ([300], [200], 1, 5, 128, 64, 512, True)])
def test_commit(dtype, ctx, new, layers, hk, dim, page, limit, rows_first):
    rng = np.random.default_rng(len(ctx) + page)
    ctx, new = np.array(ctx), np.array(new)
    kv, B = ctx + new, len(ctx)
    cu = np.concatenate([[0], np.cumsum(new)])
    T = int(cu[-1])
    parents = np.concatenate([[-1 if i == 0 else int(rng.integers(max(0, i - 3), i)) for i in range(n)] for n in new])
    parents = parents.astype(np.int64)
    draft = rng.integers(0, 3, T) + 2**40  # few values: siblings often agree
    nxt = rng.integers(0, 3, T) + 2**40
    blocks = -(-kv // page)
    pool = int(blocks.sum()) + 1
    order, used = rng.permutation(pool), 0
    table = np.full((B, int(blocks.max())), -1, np.int64)
    for b in range(B):
        table[b, :blocks[b]] = order[used:used + blocks[b]]
        used += blocks[b]
    k, v = (make_cache(pool, page, hk, dim, dtype, rows_first, layers) for _ in range(2))
    wk, wv = k.clone(), v.clone()
    accepted, paths, bonus, lens = [], [], [], []
    for b in range(B):
        path = [0] if new[b] else []
        while path and len(path) < limit:
            here = path[-1]
            kids = [c for c in range(new[b]) if parents[cu[b] + c] == here and draft[cu[b] + c] == nxt[cu[b] + here]]
            if not kids:
                break
            path.append(kids[0])
        for i, c in enumerate(path):
            src, dst = ctx[b] + c, ctx[b] + i
            for w in (wk, wv):
                w[..., int(table[b, dst // page]), int(dst % page), :, :] = \
                    w[..., int(table[b, src // page]), int(src % page), :, :].clone()
        accepted.append(len(path))
        paths.append(path + [-1] * (limit - len(path)))
        bonus.append(int(nxt[cu[b] + path[-1]]) if path else -1)
        lens.append(int(ctx[b] + len(path)))
    to = lambda a, t: torch.as_tensor(np.asarray(a), dtype=t, device="cuda")  # noqa: E731
    c = ng.tree_commit(to(draft, torch.int64), ints(parents), to(nxt, torch.int64), ints(cu), ints(kv), ints(table),
                       k, v, max_path=limit)
    assert c.accepted.tolist() == accepted and c.path.tolist() == paths
    assert c.bonus.tolist() == bonus and c.kv_lens.tolist() == lens
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert_clean()


# --------------------------------------------------------------------------- refusals
@gpu
def test_refusals():
    h = torch.float16
    k, v = ng.paged_cache(4, 16, 2, 64)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=h)
    qkv = torch.zeros(3, 8 * 64, device="cuda", dtype=h)
    table, kv, cu, row = ints([[0, 1]]), ints([10]), ints([0, 3]), ints([0, 1, 2])
    turns = ng.rope_turns(64)
    words = torch.zeros(3, 1, dtype=torch.int64, device="cuda")

    def attn(**kw):
        a = dict(q=q, k=k, v=v, table=table, kv=kv, cu=cu, mask=None, scale=1.0)
        a.update(kw)
        return ng.tree_attention(a["q"], a["k"], a["v"], a["table"], a["kv"], a["cu"], mask=a["mask"], scale=a["scale"])

    def norm(**kw):
        a = dict(qkv=qkv, wq=None, wk=None, turns=turns, pos=row, slots=row, k=k, v=v, hq=4)
        a.update(kw)
        return ng.qk_norm_rope_append(a["qkv"], a["wq"], a["wk"], a["turns"], a["pos"], a["slots"], a["k"], a["v"],
                                      q_heads=a["hq"])

    def plan(**kw):
        a = dict(cached=kv, new=ints([3]), held=ints([1]), table=table, free=row, page_size=16, num_tokens=3,
                 parents=None, mask_words=0)
        a.update(kw)
        return ng.paged_plan(*[a.pop(n) for n in ("cached", "new", "held", "table", "free")], **a)

    def commit(**kw):
        tok = torch.zeros(3, dtype=torch.int64, device="cuda")
        a = dict(draft=tok, parents=row, nxt=tok, cu=cu, kv=kv, table=table, k=k, v=v, limit=4)
        a.update(kw)
        return ng.tree_commit(a["draft"], a["parents"], a["nxt"], a["cu"], a["kv"], a["table"], a["k"], a["v"],
                              max_path=a["limit"])

    big = torch.zeros(4, 2, 16, 96, device="cuda", dtype=h).transpose(1, 2)
    odd_page = torch.zeros(4, 2, 24, 64, device="cuda", dtype=h).transpose(1, 2)
    bad = [
        lambda: attn(q=q.cpu()), lambda: attn(q=q.float()), lambda: attn(q=q.bfloat16()), lambda: attn(q=q[0]),
        lambda: attn(q=q[:, :3]), lambda: attn(k=k.contiguous()), lambda: attn(k=k[:3]), lambda: attn(scale=0.0),
        lambda: attn(scale=-1.0), lambda: attn(scale=float("nan")), lambda: attn(scale=float("inf")),
        lambda: attn(table=table.long()), lambda: attn(table=ints([[0], [1]])), lambda: attn(kv=kv.long()),
        lambda: attn(cu=ints([0, 3, 3])), lambda: attn(mask=words[:2]), lambda: attn(mask=words.int()),
        lambda: attn(q=torch.zeros(3, 4, 96, device="cuda", dtype=h), k=big, v=big),
        lambda: attn(k=odd_page, v=odd_page), lambda: attn(kv=kv.cpu()),
        lambda: attn(q=torch.zeros(3 * 4 * 64 + 1, device="cuda", dtype=h)[1:].view(3, 4, 64)),
        lambda: attn(q=torch.zeros(3, 4, 68, device="cuda", dtype=h)[..., :64]),
        lambda: norm(qkv=qkv.float()), lambda: norm(qkv=qkv[:, :-64]), lambda: norm(hq=5), lambda: norm(slots=row[:2]),
        lambda: norm(pos=row.long()), lambda: norm(wq=torch.ones(64, device="cuda", dtype=h)),
        lambda: norm(turns=turns.int()), lambda: norm(turns=torch.zeros(40, dtype=torch.int64, device="cuda")),
        lambda: norm(turns=torch.zeros(9, dtype=torch.int64, device="cuda")), lambda: norm(k=big, v=big, hq=4),
        lambda: plan(cached=kv.long()), lambda: plan(new=row), lambda: plan(page_size=12), lambda: plan(page_size=4),
        lambda: plan(mask_words=1), lambda: plan(parents=row[:2]), lambda: plan(num_tokens=-1),
        lambda: plan(mask_words=65, parents=row), lambda: plan(table=table.t()),
        lambda: commit(limit=0), lambda: commit(limit=513), lambda: commit(nxt=row), lambda: commit(k=k[0], v=v[0]),
        lambda: commit(parents=row[:1]), lambda: commit(cu=ints([0])),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
    for call in (attn, norm, plan, commit):
        call()
    attn(table=ints([[0, 1]])[:, :1], kv=ints([3]))
    with pytest.raises(ValueError):
        ng.rope_turns(40)
    assert_clean()


def test_c_abi_refusals_before_any_launch():
    """The C entry points validate their arguments without touching the GPU."""
    lib = _lib.load()
    P = 0x1000  # aligned and never read

    def attn(q=P, dtype=0, D=128, page=16, scale=1.0, ws=1 << 30, hq=8, hk=2, T=4, mask=None, words=0, qs=1024):
        return lib.ng_tree_attn(q, qs, 128, P, P, 32768, 128, 2048, P, 4, 4, P, P, mask, words, P, None, dtype, 1, T, hq,
                                hk, D, 10, page, scale, P, ws, None)

    assert attn(q=None) == 1 and attn(dtype=2) == 2 and attn(D=96) == 3 and attn(page=20) == 3 and attn(hq=7) == 3
    assert attn(T=0) == 3 and attn(hq=258, hk=2) == 3 and attn(qs=1004) == 3 and attn(scale=0.0) == 5
    assert attn(mask=P, words=0) == 5 and attn(q=P + 2) == 4

    def norm(qkv=P, dtype=0, D=128, rot=128, page=16, wq=None, wk=None, stride=1536):
        return lib.ng_qk_norm_rope_append(qkv, stride, wq, wk, P, rot, P, P, P, P, P, 32768, 128, 2048, dtype, 4, 8, 2,
                                          D, 10, page, 1e-5, None)

    assert norm(qkv=None) == 1 and norm(wq=P) == 1 and norm(dtype=5) == 2 and norm(D=96) == 3 and norm(page=1) == 3
    assert norm(rot=136) == 5 and norm(rot=8) == 5 and norm(qkv=P + 8) == 4 and norm(stride=1535) == 3

    def plan(cached=P, B=1, page=16, words=0, parents=None, width=4):
        return lib.ng_paged_plan(cached, P, P, P, 4, width, P, 5, None, parents, B, 8, page, words, P, P, P, P, P, P, P,
                                 None)

    assert plan(cached=None) == 1 and plan(B=0) == 3 and plan(B=16385) == 3 and plan(page=48) == 3
    assert plan(words=1) == 1 and plan(words=65, parents=P) == 5 and plan(width=5) == 3

    def commit(draft=P, dtype=0, layers=1, limit=4, D=128, page=16):
        return lib.ng_tree_commit(draft, P, P, P, P, P, 4, 4, P, P, 0, 32768, 128, 2048, dtype, 1, 4, layers, 2, D, 10,
                                  page, limit, P, P, P, P, None)

    assert commit(draft=None) == 1 and commit(dtype=9) == 2 and commit(layers=0) == 3 and commit(limit=513) == 5
    assert commit(D=12) == 3 and commit(page=7) == 3
    assert lib.ng_tree_attn_workspace_bytes(96) == 0
