"""Cases for the operators of a drafted-token (speculative) step over a paged KV cache.

Four operators, in the order in which a step uses them:

* ``plan``    block table, slot map, positions and ancestor masks from request lengths;
* ``norm``    per-head RMSNorm of queries and keys, rotation and append to the pages;
* ``attn``    attention of trees, chains or single tokens over the pages;
* ``commit``  greedy acceptance of a drafted path and the move of its cache rows.

``run`` computes them in a plain form (``own`` false) or through the package's
public calls (``own`` true); ``exact`` gives their values in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
THETA = 500000.0
EPS = 1e-5


# --------------------------------------------------------------------------- cases
def listed():
    """The cases that are measured."""
    return [
        # One step of a small server: 16 requests, trees of about 32 drafted nodes.
        dict(name="plan_trees", op="plan", batch=16, ctx=4096, new=32, page=16, tree=True),
        # Continuous batching: 1000 requests, most with a token or two, some with prompts of thousands.
        dict(name="plan_ragged", op="plan", batch=1000, ctx=8192, new=2048, page=16, tree=False),
        # Four sequences, one token each: the smallest decode step.
        dict(name="norm_decode", op="norm", tokens=4, q_heads=32, kv_heads=8, dim=128, rot=128, page=16, dtype="fp16",
             normed=True),
        # Sixteen trees of 61 nodes with the wide head layout.
        dict(name="norm_trees", op="norm", tokens=976, q_heads=64, kv_heads=8, dim=128, rot=128, page=64, dtype="bf16",
             normed=True),
        # Four prompts of 2048 tokens in one pass.
        dict(name="norm_prompts", op="norm", tokens=8192, q_heads=32, kv_heads=8, dim=128, rot=128, page=16,
             dtype="bf16", normed=True),
        # One sequence, one token, a short context: latency alone.
        dict(name="attn_one", op="attn", batch=1, ctx=777, new=1, tree=False, q_heads=32, kv_heads=8, dim=128, page=16,
             dtype="fp16"),
        # Plain decoding of 64 sequences of up to 8192 tokens: bound by the cache read.
        dict(name="attn_decode", op="attn", batch=64, ctx=8192, new=1, tree=False, q_heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16"),
        # 32 trees of up to 64 nodes over 4096 tokens: verification of a large draft.
        dict(name="attn_trees", op="attn", batch=32, ctx=4096, new=64, tree=True, q_heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16"),
        # One tree over a long document, wide head layout: few rows, a long axis.
        dict(name="attn_long", op="attn", batch=1, ctx=131000, new=16, tree=True, q_heads=64, kv_heads=8, dim=128,
             page=64, dtype="fp16"),
        # Chunks of three prompts that continue earlier text: chains of up to 2048 tokens.
        dict(name="attn_prompts", op="attn", batch=3, ctx=4096, new=2048, tree=False, q_heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16"),
        # Four accepted paths in the cache of a 32-layer model.
        dict(name="commit_few", op="commit", batch=4, ctx=500, new=32, layers=32, kv_heads=8, dim=128, page=16,
             dtype="fp16"),
        # 64 accepted paths of larger trees, 32 layers.
        dict(name="commit_many", op="commit", batch=64, ctx=300, new=64, layers=32, kv_heads=8, dim=128, page=16,
             dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["plan", "norm", "norm", "attn", "attn", "attn", "commit"])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "plan":
        tree = rng.random() < 0.5
        return dict(op=op, batch=_spread(rng, 1, 256 if tree else 1000), ctx=_spread(rng, 1, 8192),
                    new=_spread(rng, 1, 64 if tree else 2048), page=page, tree=tree)
    heads = rng.choice([(32, 8), (64, 8), (32, 32), (16, 2), (8, 8), (24, 8), (28, 4), (16, 1)])
    if op == "norm":
        dim = rng.choice([64, 128, 128, 256])
        most = min(8192, 8192 * 48 * 128 // ((heads[0] + 2 * heads[1]) * dim))
        return dict(op=op, tokens=_spread(rng, 1, most), q_heads=heads[0], kv_heads=heads[1], dim=dim,
                    rot=rng.choice([dim, dim, dim // 2]), page=page, dtype=dtype, normed=rng.random() < 0.75)
    dim = rng.choice([64, 128, 128])
    if op == "commit":
        return dict(op=op, batch=_spread(rng, 1, 64), ctx=_spread(rng, 1, 300), new=_spread(rng, 1, 64),
                    layers=rng.choice([1, 7, 16, 32]), kv_heads=rng.choice([1, 2, 4, 8]), dim=dim, page=page,
                    dtype=dtype)
    kind = rng.choice(["one", "tree", "chain"])
    new = 1 if kind == "one" else _spread(rng, 2, 64) if kind == "tree" else _spread(rng, 2, 2048)
    ctx = _spread(rng, 1, 131000)
    # no more cached values, and no more products, than the largest listed cases
    batch = _spread(rng, 1, 64)
    values = 64 * 8192 * 8 * 128
    products = 32 * 64 * 4096 * 32 * 128
    batch = max(1, min(batch, values // ((ctx + new) * heads[1] * dim)))
    while batch * new * (ctx + new) * heads[0] * dim > products and (batch > 1 or ctx > new):
        batch, ctx = (batch // 2, ctx) if batch > 1 else (batch, max(new, ctx // 2))
    while batch * (ctx + new) * heads[1] * dim > values:
        ctx = max(1, ctx // 2)
    return dict(op=op, batch=batch, ctx=ctx, new=new, tree=kind == "tree", q_heads=heads[0], kv_heads=heads[1], dim=dim,
                page=page, dtype=dtype)


# --------------------------------------------------------------------------- inputs
def _lengths(case):
    """Cached and new tokens of each request; the same numbers for every seed.

    Contexts are spread over [ctx / 4, ctx].  Trees have between half and all of
    ``new`` nodes.  Without a tree a batch of prompts (up to 8 requests) has
    chunks of half to all of ``new``; in a larger batch an eighth of the requests
    bring up to ``new`` tokens (evenly over the logarithm) and the others one.
    """
    b = np.arange(case["batch"])
    u = (b * 0.6180339887498949 + 0.75) % 1.0
    v = (b * 0.7548776662466927 + 0.999) % 1.0
    ctx = np.maximum(1, np.round(case["ctx"] * (0.25 + u) / 1.25)).astype(np.int64)
    if case["batch"] == 1:
        ctx[:] = case["ctx"]
    if case["tree"] or case["batch"] <= 8:
        new = np.maximum(1, np.round(case["new"] * (0.5 + 0.5 * v))).astype(np.int64)
    else:
        new = np.where(b % 8 == 0, np.round(np.exp(v * math.log(case["new"]))), 1).astype(np.int64)
    return ctx, np.maximum(1, new)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _parents(new, g):
    """Random trees in topological order: node i hangs under one of the nodes
    between i / 3 and i - 1 (wide near the root, chains among them)."""
    n = int(new.sum())
    start = np.repeat(np.cumsum(new) - new, new)
    i = torch.from_numpy(np.arange(n) - start).cuda()
    low = i // 3
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    p = (low + (u * (i - low)).long()).clamp(max=i - 1)
    return torch.where(i == 0, -1, p).to(torch.int32)


def _table(ctx, new, page, g, spare):
    """A block table for ``ctx + new`` tokens of each request over shuffled
    pages, and the number of pages in the pool."""
    blocks = -(-(ctx + new) // page)
    total = int(blocks.sum())
    pool = total + spare
    width = int(blocks.max()) + 1
    ids = torch.randperm(pool, generator=g, device="cuda")[:total].to(torch.int32)
    used = torch.arange(width, device="cuda")[None] < torch.from_numpy(blocks).cuda()[:, None]
    table = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
    table[used] = ids
    return table, pool


def _cache(pool, page, heads, dim, dtype, g, layers=None):
    """A random pool of pages [pages, page, heads, dim] whose heads lie apart
    (each head's rows of a page are contiguous)."""
    shape = (pool, heads, page, dim) if layers is None else (layers, pool, heads, page, dim)
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype).transpose(-3, -2)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=torch.int32)


def _turns(rot):
    """The rotation of each frequency per position in 2^-64 of a turn."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    return (THETA ** (-2.0 * i / rot) / (2 * math.pi) * 2.0**64).round().to(torch.int64).cuda()


def prepare(case, seed):
    """What a serving program holds before the call."""
    g, order = _generator(seed), np.random.RandomState(seed % 2**32)
    op = case["op"]
    if op == "norm":
        return _prepare_norm(case, g)
    ctx, new = _lengths(case if "tree" in case else dict(case, tree=True))
    shuffle = order.permutation(case["batch"])
    ctx, new = ctx[shuffle], new[shuffle]
    page = case["page"]
    s = dict(op=op, page=page, cached=_ints(ctx), new=_ints(new), tokens=int(new.sum()),
             cu=_ints(np.concatenate([[0], np.cumsum(new)])), kv=_ints(ctx + new), parents=None,
             longest=int(new.max()), nodes=case["new"])
    if op == "commit" or case["tree"]:
        s["parents"] = _parents(new, g)
    if op == "plan":
        held = -(-ctx // page)
        table, pool = _table(ctx, new, page, g, 64)
        keep = torch.arange(table.size(1), device="cuda")[None] < _ints(held)[:, None]
        s["table"] = torch.where(keep, table, -1)
        s["held"] = _ints(held)
        taken = torch.zeros(pool, dtype=torch.bool, device="cuda")
        taken[table[keep].long()] = True
        s["free"] = torch.nonzero(~taken).flatten().to(torch.int32)
        s["words"] = -(-case["new"] // 64) if case["tree"] else 0
        return s
    dtype = DTYPES[case["dtype"]]
    s["table"], pool = _table(ctx, new, page, g, 3)
    if op == "attn":
        s["k"] = _cache(pool, page, case["kv_heads"], case["dim"], dtype, g)
        s["v"] = _cache(pool, page, case["kv_heads"], case["dim"], dtype, g)
        s["q"] = torch.randn(s["tokens"], case["q_heads"], case["dim"], generator=g, device="cuda", dtype=dtype)
        s["scale"] = case["dim"] ** -0.5
        s["mask"] = _bits(_ancestors(s), -(-case["new"] // 64), s) if case["tree"] else None
        return s
    s["k"] = _cache(pool, page, case["kv_heads"], case["dim"], dtype, g, case["layers"])
    s["v"] = _cache(pool, page, case["kv_heads"], case["dim"], dtype, g, case["layers"])
    s["draft"] = torch.randint(0, 128256, (s["tokens"],), generator=g, device="cuda")
    # The model agrees with one child of four nodes in five.
    parent = s["parents"].long() + torch.repeat_interleave(s["cu"][:-1].long(), s["new"].long())
    child = torch.full((s["tokens"],), -1, dtype=torch.int64, device="cuda")
    inner = s["parents"] >= 0
    child.scatter_reduce_(0, parent[inner], torch.nonzero(inner).flatten(), "amax")
    agrees = (child >= 0) & (torch.rand(s["tokens"], generator=g, device="cuda") < 0.8)
    other = torch.randint(0, 128256, (s["tokens"],), generator=g, device="cuda")
    s["next"] = torch.where(agrees, s["draft"][child.clamp(min=0)], other)
    s["longest_path"] = min(case["new"], 16)
    return s


def _prepare_norm(case, g):
    dtype, m, page, dim = DTYPES[case["dtype"]], case["tokens"], case["page"], case["dim"]
    heads = case["q_heads"] + 2 * case["kv_heads"]
    pool = -(-m // page) + 3
    s = dict(op="norm", q_heads=case["q_heads"])
    s["qkv"] = torch.randn(m, heads * dim, generator=g, device="cuda", dtype=dtype)
    s["k"] = _cache(pool, page, case["kv_heads"], dim, dtype, g)
    s["v"] = _cache(pool, page, case["kv_heads"], dim, dtype, g)
    s["positions"] = torch.randint(0, 131072, (m,), generator=g, device="cuda", dtype=torch.int32)
    # tokens of a page lie together, pages are anywhere; one row in about 50 is padding
    pages = torch.randperm(pool, generator=g, device="cuda")
    i = torch.arange(m, device="cuda")
    slots = pages[i // page] * page + i % page
    padding = torch.rand(m, generator=g, device="cuda") < 0.02
    s["slots"] = torch.where(padding, -1, slots).to(torch.int32)
    s["q_weight"] = s["k_weight"] = None
    if case["normed"]:
        s["q_weight"] = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
        s["k_weight"] = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(dtype)
    s["turns"] = _turns(case["rot"])
    return s


# --------------------------------------------------------------------------- plain forms
def _padded(s):
    """[batch, nodes] index of each request's new tokens, and which exist."""
    i = torch.arange(s["longest"], device="cuda")[None]
    real = i < s["new"].long()[:, None]
    return (s["cu"][:-1].long()[:, None] + i).clamp(max=s["tokens"] - 1), real


def _ancestors(s):
    """[batch, nodes, nodes] truth values: column j is row i's ancestor or i
    itself.  Paths of up to 2, 4, 8 ... edges, by squaring."""
    at, real = _padded(s)
    n = s["longest"]
    p = torch.where(real, s["parents"].long()[at], -1)
    i = torch.arange(n, device="cuda")
    a = ((p[:, :, None] == i) | (i[:, None] == i)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        a = (a @ a > 0).float()
    return (a > 0) & real[:, :, None]


def _bits(anc, words, s):
    """The rows of `anc` packed into 64-bit words, one row a token."""
    at, real = _padded(s)
    n = anc.size(1)
    rows = torch.nn.functional.pad(anc, (0, words * 64 - n))[real].view(-1, words, 64)
    return (rows.long() << torch.arange(64, device="cuda")).sum(-1)


def _plan_plain(s):
    page, cached, new, held = s["page"], s["cached"].long(), s["new"].long(), s["held"].long()
    table, free = s["table"], s["free"].long()
    width = table.size(1)
    blocks = (cached + new + page - 1) // page
    need = (blocks - held).clamp(min=0)
    end = need.cumsum(0)
    granted = ((need == 0) | (end <= free.numel())) & (blocks <= width)
    col = torch.arange(width, device="cuda")[None]
    fresh = granted[:, None] & (col >= held[:, None]) & (col < blocks[:, None])
    source = ((end - need)[:, None] + col - held[:, None]).clamp(0, max(0, free.numel() - 1))
    table = torch.where(fresh, free[source].to(torch.int32), table)
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    request = torch.repeat_interleave(torch.arange(cached.numel(), device="cuda"), new, output_size=s["tokens"])
    i = torch.arange(s["tokens"], device="cuda") - cu[request]
    at = cached[request] + i
    slots = table.view(-1)[request * width + (at // page).clamp(max=width - 1)].long() * page + at % page
    slots = torch.where(granted[request], slots, -1)
    out = dict(table=table, cu=cu.to(torch.int32), slots=slots.to(torch.int32),
               kv=torch.where(granted, cached + new, 0).to(torch.int32),
               held=torch.where(granted, torch.maximum(held, blocks), held).to(torch.int32),
               taken=torch.where(granted, end, 0).amax().to(torch.int32).view(1))
    if s["parents"] is None:
        return dict(out, positions=at.to(torch.int32))
    anc = _ancestors(s)
    depth = anc.sum(-1)[_padded(s)[1]] - 1
    return dict(out, positions=(cached[request] + depth).to(torch.int32), mask=_bits(anc, s["words"], s))


def _norm_plain(s):
    m, dim = s["qkv"].size(0), s["k"].size(-1)
    hq, hk = s["q_heads"], s["k"].size(-2)
    x = s["qkv"].view(m, -1, dim).float()
    q, k = x[:, :hq], x[:, hq:hq + hk]
    if s["q_weight"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_weight"].float()
    # the phase in 2^-64 of a turn wraps as whole numbers do: exact at any position
    phase = s["positions"].long()[:, None] * s["turns"][None]
    angle = (phase >> 32).float() * (2 * math.pi / 2.0**32)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    half = s["turns"].numel()

    def turned(y):
        a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)

    dtype, page = s["qkv"].dtype, s["k"].size(1)
    keep = torch.nonzero(s["slots"] >= 0).flatten()
    slots = s["slots"].long()[keep]
    s["k"][slots // page, slots % page] = turned(k).to(dtype)[keep]
    s["v"][slots // page, slots % page] = s["qkv"].view(m, -1, dim)[keep, hq + hk:]
    return dict(q=turned(q).to(dtype), k=s["k"], v=s["v"])


def _attn_plain(s):
    dim, hq, hk = s["q"].size(2), s["q"].size(1), s["k"].size(2)
    kv, page = s["kv"].long(), s["page"]
    longest = s["table"].size(1) * page
    key = torch.arange(longest, device="cuda")
    pages = s["table"].long().clamp(min=0)
    there = key[None] < kv[:, None]
    # [batch, kv heads, keys, dim] in 32 bits; rows past a request's end hold nothing
    k = s["k"][pages].flatten(1, 2).transpose(1, 2).float()
    v = torch.where(there[:, None, :, None], s["v"][pages].flatten(1, 2).transpose(1, 2).float(), 0.0)
    at, real = _padded(s)
    n = at.size(1)
    q = s["q"][at].float().view(len(kv), n, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    score = (q.flatten(2, 3) @ k.transpose(-1, -2)).view(len(kv), hk, hq // hk, n, longest) * s["scale"]
    node = key[None] - (kv - s["new"].long())[:, None]  # which new token a key is
    if s["mask"] is None:
        sees = node[:, None, :] <= torch.arange(n, device="cuda")[None, :, None]
    else:
        words = s["mask"][at]
        j = node.clamp(0, 64 * words.size(2) - 1)[:, None, :].expand(-1, n, -1)
        sees = ((words.gather(2, j // 64) >> (j % 64)) & 1).bool() | (node < 0)[:, None, :]
    sees = (sees & there[:, None, :])[:, None, None]
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).view(len(kv), hk, hq // hk, n, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(len(kv), n, hq, dim)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(len(kv), n, hq)
    return dict(out=out[real].to(s["q"].dtype), lse=lse[real])


def _commit_plain(s):
    at, real = _padded(s)
    b, n = at.shape
    limit, page = s["longest_path"], s["page"]
    p = torch.where(real, s["parents"].long()[at], -1)
    draft, nxt = s["draft"][at], s["next"][at]
    follows = (p >= 0) & real & (draft == nxt.gather(1, p.clamp(min=0)))
    i = torch.arange(n, device="cuda")
    # of several children that agree, the first
    same = (p[:, :, None] == p[:, None, :]) & follows[:, None, :] & (i[None, :] < i[:, None])
    follows = (follows & ~same.any(-1)) | ((i == 0) & real)
    anc = _ancestors(s)
    kept = ((anc & ~follows[:, None, :]).sum(-1) == 0) & real & anc.any(-1)
    kept = kept & anc[:, :, 0] & (anc.sum(-1) <= limit)
    accepted = kept.sum(-1)
    path = torch.where(kept, i, n).sort(-1).values
    path = torch.nn.functional.pad(path, (0, limit), value=n)[:, :limit]
    path = torch.where(path < n, path, -1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])
    bonus = torch.where(accepted > 0, nxt.gather(1, last.clamp(min=0))[:, 0], -1)
    before = s["kv"].long() - s["new"].long()
    request = torch.arange(b, device="cuda")[:, None].expand(-1, limit)[path >= 0]
    source = (before[:, None] + path)[path >= 0]
    target = (before[:, None] + torch.arange(limit, device="cuda"))[path >= 0]
    table = s["table"].long()
    from_page, to_page = table[request, source // page], table[request, target // page]
    for cache in (s["k"], s["v"]):
        cache[:, to_page, target % page] = cache[:, from_page, source % page]
    return dict(accepted=accepted.to(torch.int32), path=path.to(torch.int32), bonus=bonus,
                kv=(before + accepted).to(torch.int32), k=s["k"], v=s["v"])


# --------------------------------------------------------------------------- the passes
def run(s):
    """One pass through an operator."""
    op = s["op"]
    if not own:
        return {"plan": _plan_plain, "norm": _norm_plain, "attn": _attn_plain, "commit": _commit_plain}[op](s)
    import nibblegemm_b200 as ng
    if op == "plan":
        p = ng.paged_plan(s["cached"], s["new"], s["held"], s["table"], s["free"], page_size=s["page"],
                          num_tokens=s["tokens"], parents=s["parents"], mask_words=s["words"])
        out = dict(table=s["table"], cu=p.cu_new, slots=p.slots, kv=p.kv_lens, held=p.held, taken=p.taken,
                   positions=p.positions)
        return out if p.mask is None else dict(out, mask=p.mask)
    if op == "norm":
        q = ng.qk_norm_rope_append(s["qkv"], s["q_weight"], s["k_weight"], s["turns"], s["positions"], s["slots"],
                                   s["k"], s["v"], q_heads=s["q_heads"], eps=EPS)
        return dict(q=q, k=s["k"], v=s["v"])
    if op == "attn":
        out, lse = ng.tree_attention(s["q"], s["k"], s["v"], s["table"], s["kv"], s["cu"], mask=s["mask"],
                                     scale=s["scale"], return_lse=True)
        return dict(out=out, lse=lse)
    c = ng.tree_commit(s["draft"], s["parents"], s["next"], s["cu"], s["kv"], s["table"], s["k"], s["v"],
                       max_path=s["longest_path"])
    return dict(accepted=c.accepted, path=c.path, bonus=c.bonus, kv=c.kv_lens, k=s["k"], v=s["v"])


def work(case):
    """Bytes and operations that one pass cannot do without."""
    op = case["op"]
    if op == "norm":
        values = case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        return dict(bytes=values * 4 + case["tokens"] * 8, flops=values * 8)
    ctx, new = _lengths(case if "tree" in case else dict(case, tree=True))
    tokens = int(new.sum())
    if op == "plan":
        words = -(-case["new"] // 64) if case["tree"] else 0
        table = int((-(-(ctx + new) // case["page"]) - ctx // case["page"]).sum())
        return dict(bytes=case["batch"] * 24 + table * 8 + tokens * (8 + (4 + 8 * words if case["tree"] else 0)),
                    flops=tokens * 8)
    if op == "commit":
        rows = 2 * case["batch"] * case["layers"] * case["kv_heads"] * case["dim"] * 2
        return dict(bytes=rows * 3 * 2 + tokens * 20, flops=tokens * 4)
    heads, dim = case["q_heads"], case["dim"]
    keys = int((ctx + new).sum())
    seen = int((new * ctx).sum() + (new * (new + 1) // 2).sum())
    return dict(bytes=keys * case["kv_heads"] * dim * 4 + tokens * heads * (dim * 4 + 4), flops=4 * seen * heads * dim)


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """`run`'s outputs from the definitions, in 64 bits, a request at a time."""
    s = prepare(case, seed)
    return {"plan": _exact_plan, "commit": _exact_commit, "norm": _exact_norm, "attn": _exact_attn}[case["op"]](s)


def _exact_plan(s):
    """Whole numbers only: nothing is computed that could be inexact."""
    return None


def _exact_commit(s):
    """The caches after each request's walk from its root; the other outputs are whole."""
    k, v, page = s["k"].double(), s["v"].double(), s["page"]
    parents, draft, nxt = s["parents"].tolist(), s["draft"].tolist(), s["next"].tolist()
    cu, kv, table = s["cu"].tolist(), s["kv"].tolist(), s["table"].tolist()
    for b in range(len(kv)):
        first, n = cu[b], cu[b + 1] - cu[b]
        path = [0] if n else []
        while path and len(path) < s["longest_path"]:
            here = path[-1]
            child = [c for c in range(n) if parents[first + c] == here and draft[first + c] == nxt[first + here]]
            if not child:
                break
            path.append(child[0])
        rows = [divmod(kv[b] - n + c, page) for c in path]
        to = [divmod(kv[b] - n + c, page) for c in range(len(path))]
        for cache in (k, v):
            kept = [cache[:, table[b][p], r].clone() for p, r in rows]
            for (p, r), value in zip(to, kept):
                cache[:, table[b][p], r] = value
    return dict(accepted=None, path=None, bonus=None, kv=None, k=k, v=v)


def _exact_norm(s):
    m, dim, page = s["qkv"].size(0), s["k"].size(-1), s["k"].size(1)
    hq, hk, half = s["q_heads"], s["k"].size(-2), s["turns"].numel()
    x = s["qkv"].double().view(m, hq + 2 * hk, dim)
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    angle = s["positions"].double()[:, None, None] * THETA ** (-i / half)
    rotor = torch.polar(torch.ones_like(angle), angle)

    def head(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * rotor
        return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)

    k, v = s["k"].double(), s["v"].double()
    slots = s["slots"].long()
    rows = slots >= 0
    k[slots[rows] // page, slots[rows] % page] = head(x[:, hq:hq + hk], s["k_weight"])[rows]
    v[slots[rows] // page, slots[rows] % page] = x[rows][:, hq + hk:]
    return dict(q=head(x[:, :hq], s["q_weight"]), k=k, v=v)


def _exact_attn(s):
    hq, hk, page = s["q"].size(1), s["k"].size(2), s["page"]
    outs, lses = [], []
    for b, (kv, first, end) in enumerate(zip(s["kv"].tolist(), s["cu"][:-1].tolist(), s["cu"][1:].tolist())):
        pages = s["table"][b, :-(-kv // page)].long()
        k = s["k"][pages].reshape(-1, hk, s["k"].size(3))[:kv].double()
        v = s["v"][pages].reshape(-1, hk, s["k"].size(3))[:kv].double()
        n = end - first
        sees = torch.ones(n, kv, dtype=torch.bool, device="cuda")
        for node in range(n) if s["mask"] is not None else ():
            sees[:, kv - n + node] = (s["mask"][first:end, node // 64] >> (node % 64)) & 1 == 1
        if s["mask"] is None:
            sees = sees.tril(kv - n)
        heads = []
        for h in range(hk):
            q = s["q"][first:end, h * (hq // hk):(h + 1) * (hq // hk)].double()
            x = torch.einsum("ngd,kd->ngk", q, k[:, h]) * s["scale"]
            x = x.masked_fill(~sees[:, None], -math.inf)
            lse = torch.logsumexp(x, -1)
            heads.append((torch.einsum("ngk,kd->ngd", torch.exp(x - lse[..., None]), v[:, h]), lse))
        outs.append(torch.cat([o for o, _ in heads], 1))
        lses.append(torch.cat([x for _, x in heads], 1))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))
