"""What the speed of the operators for drafted tokens and for long contexts is measured on.

Every case is one call of an operator on a paged cache, with its tensors in
hand (torch.ops.mhcpre.*):

  draft   draft_attention: several new tokens per sequence over a paged cache,
          a tree of drafted tokens or a chain of them (a prompt's chunk);
  accept  draft_accept: the path of a tree that the model's own choices confirm;
  keep    cache_keep: the confirmed tokens' keys and values to the places after
          the context;
  bounds  cache_bounds: the smallest and largest key of every page, kept up with
          the cache;
  sparse  sparse_attention: one new token per sequence, over the pages of each kv
          head that the bounds rank highest.

The plain forms are elementary torch operations in 32 bits, rounded once at
the end.  Only the pages' scores are in 64 bits, in both forms and in the
definition: which page is the last one taken hangs on their last bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _draft(B, S, heads, kv_heads, d, length, page, dtype, tree=True, ragged=True, window=0):
    return dict(op="draft", B=B, S=S, heads=heads, kv_heads=kv_heads, d=d, length=length, page=page,
                dtype=dtype, tree=tree, ragged=ragged, window=window)


def _accept(B, S):
    return dict(op="accept", B=B, S=S)


def _keep(B, S, kept, kv_heads, d, page, dtype, slot_major=False):
    return dict(op="keep", B=B, S=S, kept=kept, kv_heads=kv_heads, d=d, page=page, dtype=dtype,
                slot_major=slot_major)


def _bounds(B, tokens, length, kv_heads, d, page, dtype):
    return dict(op="bounds", B=B, tokens=tokens, length=length, kv_heads=kv_heads, d=d, page=page,
                dtype=dtype)


def _sparse(B, heads, kv_heads, d, length, page, top, dtype, ragged=True):
    return dict(op="sparse", B=B, heads=heads, kv_heads=kv_heads, d=d, length=length, page=page,
                top=top, dtype=dtype, ragged=ragged)


def listed():
    return [
        # One user's chat, 1000 tokens in, with a small tree: latency counts.
        dict(_draft(1, 8, 32, 8, 128, 1000, 16, "bf16", ragged=False), name="draft_one"),
        # A server's step with drafts: sequences of all ages, trees of different sizes.
        dict(_draft(32, 32, 32, 8, 128, 8192, 64, "fp16"), name="draft_batch"),
        # Chunks of prompts behind what the cache holds, a sliding window, odd sizes.
        dict(_draft(3, 777, 24, 24, 96, 5000, 7, "fp16", tree=False, window=1111),
             name="draft_chunk_window"),
        # The largest: long documents, eight query heads to each of the cache's, large trees.
        dict(_draft(2, 64, 64, 8, 128, 65536, 64, "bf16"), name="draft_long"),
        # What the two steps confirm.
        dict(_accept(32, 32), name="accept_batch"),
        dict(_accept(1000, 256), name="accept_large"),
        # A few confirmed tokens of each tree to their places, in one layer's cache.
        dict(_keep(32, 32, 5, 8, 128, 64, "fp16"), name="keep_batch"),
        dict(_keep(500, 101, 17, 8, 128, 16, "bf16", True), name="keep_large"),
        # The bounds after a step of single tokens, and after prompts.
        dict(_bounds(64, 1, 8192, 8, 128, 64, "bf16"), name="bounds_step"),
        dict(_bounds(8, 8192, 16384, 8, 128, 16, "fp16"), name="bounds_prompts"),
        # One user's document of 131072 tokens, 64 pages of 64 for each head.
        dict(_sparse(1, 32, 8, 128, 131072, 64, 64, "bf16", False), name="sparse_one"),
        # A server's batch of documents, small pages.
        dict(_sparse(16, 64, 8, 128, 131072, 16, 256, "fp16"), name="sparse_batch"),
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def _pairs(c):
    """Scores of a draft case when every sequence has the longest's length."""
    return c["B"] * c["heads"] * c["S"] * c["length"]


def _padded(c):
    """Cache values of a case when every sequence has the longest's length."""
    return c["B"] * c["length"] * c["kv_heads"] * c["d"]


def _largest(op, size):
    return max(size(c) for c in listed() if c["op"] == op)


def draw(rng):
    op = rng.choice(("draft", "draft", "draft", "accept", "keep", "bounds", "sparse", "sparse"))
    dtype = rng.choice(("fp16", "bf16"))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 3, 4, 5, 8, 16))
    d = rng.choice((64, 96, 128, 128, 128, 192, 256))
    page = rng.choice((1, 7, 16, 16, 32, 64, 64, 128))
    while op == "draft":
        tree = rng.random() < 0.7
        S = _log(rng, 1, 256 if tree else 2048)
        length = _log(rng, S, 131072)
        c = _draft(_log(rng, 1, 64), S, heads, kv_heads, d, length, page, dtype, tree,
                   rng.random() < 0.8, _log(rng, 1, length) if rng.random() < 0.25 else 0)
        if (_pairs(c) * d <= _largest("draft", _pairs) * 64
                and _padded(c) <= _largest("draft", _padded)):
            return c
    if op == "accept":
        return _accept(_log(rng, 1, 1000), _log(rng, 1, 256))
    if op == "keep":
        S = _log(rng, 1, 256)
        B = _log(rng, 1, min(500, max(1, 500 * 101 * 8 * 128 // (S * kv_heads * d))))
        return _keep(B, S, rng.randint(1, min(S, 40)), kv_heads, d, page, dtype, rng.random() < 0.5)
    while op == "bounds":
        tokens = _log(rng, 1, 8192)
        c = _bounds(_log(rng, 1, 256), tokens, _log(rng, tokens, 32768), kv_heads, d, max(page, 7),
                    dtype)
        if _padded(c) <= _largest("bounds", _padded):
            return c
    while True:
        length, page = _log(rng, 1, 131072), max(page, 7)
        c = _sparse(_log(rng, 1, 64), heads, kv_heads, d, length, page,
                    _log(rng, 2, max(2, min(8192, length) // page + 2)), dtype, rng.random() < 0.8)
        if _padded(c) <= _largest("sparse", _padded) // 2:
            return c


def _lengths(case):
    """The cached tokens of a case's rows: all the longest, or spread from short ones (an idle row of
    length 0 among them in batches of more than 8) to the longest."""
    B, longest = case["B"], case["length"]
    if not case.get("ragged", True):
        return [longest] * B
    lengths = [max(1, round(longest * ((i + 1) / B) ** 2)) for i in range(B)]
    if B > 8:
        lengths[0] = 0
    return lengths


def _new(case):
    """New tokens of a case's rows, of the row of the same number in _lengths: most have all of them,
    some fewer."""
    most = case["S"] if case["op"] == "draft" else case["tokens"]
    return [min(n, max(1, most - i % 4 * most // 5)) for i, n in enumerate(_lengths(case))]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32):
    """Normal values in `dtype`, made in pieces so that a large cache needs little beside itself."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for r in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - r)
        flat[r:r + n] = torch.randn(n, generator=g, device="cuda")
    return out


def _cache(g, pages, page, kv_heads, d, dtype, slot_major=False):
    """A cache [pages, page, kv_heads, d]; in memory a head's slots of a page are contiguous, or
    (slot_major) a slot's heads."""
    if slot_major:
        return _normal(g, (pages, page, kv_heads, d), dtype)
    return _normal(g, (pages, kv_heads, page, d), dtype).transpose(1, 2)


def _table(g, counts, width, pages):
    """A page table int32 [rows, width]: distinct pages of the pool, in no order, then -1.  The
    pool's last page is nobody's."""
    counts = torch.tensor(counts, device="cuda")
    order = torch.randperm(pages - 1, generator=g, device="cuda")
    column = torch.arange(width, device="cuda")
    held = column < counts[:, None]
    at = (counts.cumsum(0) - counts)[:, None] + column
    return torch.where(held, order[at.clamp(max=pages - 2)], -1).int()


def _paged(g, case, lengths, slot_major=False):
    """Page table, lengths (rows in no order), a key and a value cache, and the rows' order."""
    kv_heads, d, page = (case[k] for k in ("kv_heads", "d", "page"))
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + sum(counts) // 16 + 2
    table = _table(g, counts, max(max(counts), 1), pages)
    order = torch.randperm(len(lengths), generator=g, device="cuda")
    s = {"op": case["op"], "page_table": table[order].contiguous(),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")[order].contiguous(),
         "k_cache": _cache(g, pages, page, kv_heads, d, DTYPES[case["dtype"]], slot_major)}
    return s, order


def _trees(g, B, S):
    """Parents int32 [B, S] of trees around node 0, most of them near the root."""
    node = torch.arange(S, device="cuda")
    near = torch.rand((B, S), generator=g, device="cuda") ** 2
    return torch.where(node > 0, (near * node).long().clamp(max=(node - 1).clamp(min=0)), -1).int()


def _prepare_draft(case, seed):
    g = _generator(seed)
    B, S, heads, d, dtype = case["B"], case["S"], case["heads"], case["d"], DTYPES[case["dtype"]]
    s, order = _paged(g, case, _lengths(case))
    s["v_cache"] = _normal(g, s["k_cache"].transpose(1, 2).shape, dtype).transpose(1, 2)
    s["q"] = (2 * _normal(g, (B, S, heads, d))).to(dtype)
    s["parents"] = _trees(g, B, S) if case["tree"] else None
    s["drafted"] = torch.tensor(_new(case), dtype=torch.int32, device="cuda")[order].contiguous()
    s.update(scale=d ** -0.5, window=case["window"])
    return s


def _prepare_accept(case, seed):
    g = _generator(seed)
    B, S = case["B"], case["S"]
    parents = _trees(g, B, S)
    # The model chooses one of the drafted tokens more often than not.  Siblings differ in their
    # tokens, but for a few.
    tokens = torch.randint(0, 32000, (B, S), generator=g, device="cuda")
    chosen = torch.randint(0, 32000, (B, S), generator=g, device="cuda")
    child = torch.where(torch.rand((B, S), generator=g, device="cuda") < 0.7, torch.arange(S, device="cuda"), 0)
    child = torch.zeros_like(child).scatter_reduce(1, parents.clamp(min=0).long(), child, "amax")
    chosen = torch.where(child > 0, tokens.gather(1, child), chosen)
    drafted = torch.randint(S - S // 4, S + 1, (B,), generator=g, device="cuda").int()
    lengths = drafted + torch.randint(0, 8192, (B,), generator=g, device="cuda").int()
    return {"op": "accept", "tokens": tokens, "parents": parents, "drafted": drafted,
            "chosen": chosen, "lengths": lengths}


def _kept(case):
    """Nodes on the confirmed path of each row of a keep case."""
    return [1 + (case["kept"] - 1) * (i % 7) // 6 for i in range(case["B"])]


def _prepare_keep(case, seed):
    g = _generator(seed)
    B, S = case["B"], case["S"]
    s, order = _paged(g, case, [S + 100 + i * 37 % 200 for i in range(B)], case["slot_major"])
    s["v_cache"] = _cache(g, s["k_cache"].shape[0], case["page"], case["kv_heads"], case["d"],
                          DTYPES[case["dtype"]], case["slot_major"])
    s["drafted"] = torch.full((B,), S, dtype=torch.int32, device="cuda")
    # Node 0 and a few of the others, ascending.
    rank = torch.rand((B, S), generator=g, device="cuda")
    rank[:, 0] = -1
    some = rank.argsort(1).argsort(1) < torch.tensor(_kept(case), device="cuda")[:, None]
    node = torch.arange(S, device="cuda")
    path = torch.where(some, node, S).sort(1).values
    s["path"] = torch.where(path < S, path, -1).int()
    return s


def _prepare_bounds(case, seed):
    g = _generator(seed)
    s, order = _paged(g, case, _lengths(case))
    pages, page, kv_heads, d = s["k_cache"].shape
    s["counts"] = torch.tensor(_new(case), dtype=torch.int32, device="cuda")[order].contiguous()
    s["tokens"] = case["tokens"]
    a = _normal(g, (pages, kv_heads, d), s["k_cache"].dtype)
    s["lo"], s["hi"] = a.abs().neg() - 1, a.abs() + 1
    return s


def _prepare_sparse(case, seed):
    g = _generator(seed)
    s, order = _paged(g, case, _lengths(case))
    k = s["k_cache"]
    pages, page, kv_heads, d = k.shape
    # Keys of a page have something in common, of some pages more than of others.
    topic = _normal(g, (pages, 1, kv_heads, d), k.dtype)
    topic *= torch.rand((pages, 1, 1, 1), generator=g, device="cuda").to(k.dtype)
    k += topic
    s["v_cache"] = _normal(g, k.transpose(1, 2).shape, k.dtype).transpose(1, 2)
    held = torch.zeros(pages, dtype=torch.long, device="cuda")  # tokens of each page
    column = torch.arange(s["page_table"].shape[1], device="cuda") * page
    inside = (s["lengths"][:, None] - column).clamp(0, page).long()
    at = torch.where(s["page_table"] >= 0, s["page_table"], pages - 1).long()
    held.scatter_(0, at.view(-1), inside.view(-1))
    there = (torch.arange(page, device="cuda") < held[:, None])[..., None, None]
    s["lo"] = torch.where(there, k, math.inf).amin(1)
    s["hi"] = torch.where(there, k, -math.inf).amax(1)
    s["q"] = (2 * _normal(g, (case["B"], case["heads"], d))).to(k.dtype)
    s.update(top=case["top"], first=1, last=1, scale=d ** -0.5)
    return s


_PREPARE = {"draft": _prepare_draft, "accept": _prepare_accept, "keep": _prepare_keep,
            "bounds": _prepare_bounds, "sparse": _prepare_sparse}


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _ancestors(parents):
    """Bool [B, S, S]: whether node j is node i or one of its ancestors."""
    B, S = parents.shape
    node = torch.arange(S, device=parents.device)
    step = (parents[:, :, None] == node) & (node < node[:, None])  # the parent
    reach = (step | torch.eye(S, dtype=torch.bool, device=parents.device)).float()
    for _ in range(max(1, (S - 1).bit_length())):  # paths of twice the length
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _plain_draft(s):
    q, table, lengths = s["q"], s["page_table"].long(), s["lengths"].long()
    B, S, heads, d = q.shape
    page, kv_heads = s["k_cache"].shape[1:3]
    L = table.shape[1] * page
    rows = table.clamp(min=0)
    drafted = torch.minimum(s["drafted"].long().clamp(0, S), lengths)
    context = lengths - drafted
    node, t = torch.arange(S, device=q.device), torch.arange(L, device=q.device)
    if s["parents"] is None:
        reach = (node <= node[:, None]).expand(B, S, S)
    else:
        reach = _ancestors(s["parents"])
    depth = reach.sum(2) - 1
    j = t - context[:, None]  # [B, L]: the key's node, or below 0
    seen = torch.where((j < 0)[:, None], True,
                       reach.gather(2, j.clamp(0, S - 1)[:, None].expand(B, S, L)))
    at = torch.where(j < 0, t, context[:, None] + depth.gather(1, j.clamp(0, S - 1)))  # positions
    if s["window"]:
        seen = seen & (at[:, None] > (context[:, None] + depth)[:, :, None] - s["window"])
    seen = seen & (t < lengths[:, None])[:, None] & (node < drafted[:, None])[:, :, None]
    seen = seen[:, None, None]  # [B, 1, 1, S, L]
    k = s["k_cache"].transpose(1, 2)[rows].float().permute(0, 2, 4, 1, 3).reshape(B, kv_heads, d, L)
    qs = q.float().view(B, S, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4)
    score = torch.matmul(qs.reshape(B, kv_heads, -1, d), k).view(B, kv_heads, -1, S, L) * s["scale"]
    del k
    score = torch.where(seen, score, -math.inf)
    top = score.amax(4, keepdim=True)
    score = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = score.sum(4, keepdim=True)
    v = s["v_cache"].transpose(1, 2)[rows].float().permute(0, 2, 1, 3, 4).reshape(B, kv_heads, L, d)
    out = torch.matmul(score.view(B, kv_heads, -1, L), v).view(B, kv_heads, -1, S, d)
    out = out / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    return (out.permute(0, 3, 1, 2, 4).reshape(B, S, heads, d).to(q.dtype),
            lse.permute(0, 3, 1, 2).reshape(B, S, heads))


def _plain_accept(s):
    tokens, parents, chosen = s["tokens"], s["parents"].long(), s["chosen"]
    B, S = tokens.shape
    node = torch.arange(S, device=tokens.device)
    drafted = torch.minimum(s["drafted"].clamp(0, S), s["lengths"].clamp(min=0)).long()
    there = node < drafted[:, None]
    child = (parents >= 0) & (parents < node) & there
    wanted = child & (chosen.gather(1, parents.clamp(0, S - 1)) == tokens)
    # Of a node's children with the wanted token the first one.
    twin = (parents[:, :, None] == parents[:, None]) & wanted[:, None] & (node < node[:, None])
    edge = (node == 0) & there | wanted & ~twin.any(2)
    # A node is on the path if all of its ancestors have such an edge.
    reach = _ancestors(torch.where(child, s["parents"], -1))
    on = ~(reach & ~edge[:, None]).any(2)
    path = torch.where(on, node, S).sort(1).values
    path = torch.where(path < S, path, -1)
    accepted = on.sum(1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])
    after = torch.where(accepted > 0, chosen.gather(1, last.clamp(min=0))[:, 0], -1)
    return (path.int(), accepted.int(), after,
            (s["lengths"].clamp(min=0) - drafted + accepted).int())


def _plain_keep(s):
    lengths, path, table = s["lengths"].long(), s["path"].long(), s["page_table"].long()
    B, S = path.shape
    N, page = s["k_cache"].shape[:2]
    first = (lengths - torch.minimum(s["drafted"].long(), lengths))[:, None]
    moved = path > torch.arange(S, device=path.device)
    # A row's other tokens: a slot of nobody's page onto itself.
    spare = (N - 1) * page

    def slot(t):
        return torch.where(moved, table.gather(1, t.clamp(min=0) // page) * page + t % page, spare)

    src = slot(torch.where(moved, first + path, 0))
    dst = slot(torch.where(moved, first + torch.arange(S, device=path.device), 0))
    for cache in (s["k_cache"], s["v_cache"]):
        cache[dst // page, dst % page] = cache[src // page, src % page]
    return s["k_cache"], s["v_cache"]


def _plain_bounds(s):
    table, lengths = s["page_table"].long(), s["lengths"].long()
    N, page = s["k_cache"].shape[:2]
    counts = torch.minimum(s["counts"].long().clamp(0, s["tokens"]), lengths)
    begin = lengths - counts
    column = begin[:, None] // page + torch.arange((s["tokens"] + page - 2) // page + 1, device=table.device)
    touched = (column * page < lengths[:, None]) & (counts > 0)[:, None]
    pages = table.gather(1, column.clamp(max=table.shape[1] - 1))
    pages = torch.where(touched & (pages >= 0), pages, N - 1)  # others: nobody's page
    t = column[..., None] * page + torch.arange(page, device=table.device)
    new = (t >= begin[:, None, None]) & (t < lengths[:, None, None]) & (pages < N - 1)[..., None]
    old = (column * page < begin[:, None]) | (pages == N - 1)
    new, old = new[..., None, None], old[..., None, None]
    k = s["k_cache"][pages].float()  # [B, columns, page, kv_heads, d]
    for bound, far, best in ((s["lo"], math.inf, torch.minimum), (s["hi"], -math.inf, torch.maximum)):
        kept = torch.where(old, bound[pages].float(), far)
        k_best = torch.where(new, k, far)
        k_best = k_best.amin(2) if far > 0 else k_best.amax(2)
        bound[pages] = best(kept, k_best).to(bound.dtype)
    return s["lo"], s["hi"]


def _plain_columns(s):
    """The pages that each kv head of a row takes: int32 [B, kv_heads, top], ascending, then -1."""
    q, table, lengths = s["q"], s["page_table"].long(), s["lengths"].long()
    B, heads, d = q.shape
    page, kv_heads = s["k_cache"].shape[1:3]
    W, top = table.shape[1], s["top"]
    q = q.double().view(B, kv_heads, heads // kv_heads, d)
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)  # [B, kv_heads, d]
    rows = table.clamp(min=0)
    score = torch.matmul(s["hi"][rows].double().permute(0, 2, 1, 3), up[..., None])
    score += torch.matmul(s["lo"][rows].double().permute(0, 2, 1, 3), down[..., None])
    score = score[..., 0]  # [B, kv_heads, W]
    column = torch.arange(W, device=q.device)
    held = ((lengths + page - 1) // page)[:, None]
    always = (column < s["first"]) | (column >= held - s["last"])
    score = torch.where(always[:, None], math.inf, score)
    there = ((column < held) & (table >= 0))[:, None].expand_as(score)
    score = torch.where(there, score, -math.inf)
    order = torch.sort(score, dim=2, descending=True, stable=True).indices[:, :, :top]
    taken = torch.where(there.gather(2, order), order, W).sort(2).values
    taken = torch.nn.functional.pad(taken, (0, top - taken.shape[2]), value=W)
    return torch.where(taken < W, taken, -1).int()


def _plain_sparse(s):
    q, table, lengths = s["q"], s["page_table"].long(), s["lengths"].long()
    B, heads, d = q.shape
    page, kv_heads = s["k_cache"].shape[1:3]
    columns = _plain_columns(s)
    top = columns.shape[2]
    column = columns.clamp(min=0).long()
    pages = table[:, None].expand(B, kv_heads, -1).gather(2, column).clamp(min=0)
    head = torch.arange(kv_heads, device=q.device)[:, None]
    t = column[..., None] * page + torch.arange(page, device=q.device)
    seen = ((columns >= 0)[..., None] & (t < lengths[:, None, None, None])).view(B, kv_heads, 1, top * page)
    k = s["k_cache"].transpose(1, 2)[pages, head].float().view(B, kv_heads, top * page, d)
    qs = q.float().view(B, kv_heads, heads // kv_heads, d)
    score = torch.matmul(k, qs.transpose(2, 3)).transpose(2, 3) * s["scale"]
    del k
    score = torch.where(seen, score, -math.inf)
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(most > -math.inf, most, 0.0))
    total = p.sum(3, keepdim=True)
    v = s["v_cache"].transpose(1, 2)[pages, head].float().view(B, kv_heads, top * page, d)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = most + torch.log(total)
    return out.view(B, heads, d).to(q.dtype), lse.view(B, heads), columns


_PLAIN = {"draft": _plain_draft, "accept": _plain_accept, "keep": _plain_keep,
          "bounds": _plain_bounds, "sparse": _plain_sparse}


_ops = None


def _own(s):
    global _ops
    if _ops is None:
        import __graft_entry__

        __graft_entry__.load_package().torch_ops()
        _ops = torch.ops.mhcpre
    ops = _ops
    if s["op"] == "draft":
        return ops.draft_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                   s["drafted"], s["parents"], s["scale"], s["window"])
    if s["op"] == "accept":
        return ops.draft_accept(s["tokens"], s["parents"], s["drafted"], s["chosen"], s["lengths"])
    if s["op"] == "keep":
        ops.cache_keep(s["k_cache"], s["v_cache"], s["page_table"], s["lengths"], s["drafted"], s["path"])
        return s["k_cache"], s["v_cache"]
    if s["op"] == "bounds":
        ops.cache_bounds(s["k_cache"], s["page_table"], s["lengths"], s["counts"], s["lo"], s["hi"],
                         s["tokens"])
        return s["lo"], s["hi"]
    return ops.sparse_attention(s["q"], s["k_cache"], s["v_cache"], s["lo"], s["hi"], s["page_table"],
                                s["lengths"], s["top"], s["first"], s["last"], s["scale"])


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def work(case):
    op, B = case["op"], case["B"]
    if op == "accept":  # tokens and choices in 64 bits; parents, path; a few numbers a row
        return {"bytes": B * case["S"] * (8 + 8 + 4 + 4) + 24 * B, "flops": 0}
    page, kv_heads, d = (case[k] for k in ("page", "kv_heads", "d"))
    row = 2 * kv_heads * d  # bytes of a token in one cache
    if op == "keep":
        moved = sum(_kept(case)) - B
        return {"bytes": 2 * 2 * moved * row + 4 * B * case["S"] + 8 * B, "flops": 0}
    lengths = _lengths(case)
    if op == "bounds":
        counts = _new(case)
        touched = sum(-(-n // page) - (n - c) // page for n, c in zip(lengths, counts))
        joined = sum(c > 0 and (n - c) % page > 0 for n, c in zip(lengths, counts))
        return {"bytes": sum(counts) * row + 2 * (touched + joined) * row + 4 * touched + 8 * B,
                "flops": 2 * sum(counts) * kv_heads * d}
    heads = case["heads"]
    if op == "draft":
        S, new, window = case["S"], _new(case), case["window"] or 1 << 40
        # What a tree's nodes see of each other is counted as themselves only.
        tokens = sum(min(n, window + c - 1) for n, c in zip(lengths, new) if c)
        if case["tree"]:
            pairs = sum(c * min(n - c + 1, window) for n, c in zip(lengths, new))
        else:
            pairs = sum(min(n - c + i + 1, window) for n, c in zip(lengths, new) for i in range(c))
        size = 2 * tokens * row + 2 * B * S * heads * d * 2 + 4 * B * S * heads + 4 * tokens // page
        return {"bytes": size + (4 * B * S if case["tree"] else 0) + 8 * B, "flops": 4 * pairs * heads * d}
    held = [-(-n // page) for n in lengths]
    tokens = sum(min(n, case["top"] * page) for n in lengths)
    size = 2 * sum(held) * row + 4 * sum(held)  # both bounds and the table
    size += 2 * tokens * row + 2 * 2 * B * heads * d + 4 * B * heads + 4 * B * kv_heads * case["top"]
    return {"bytes": size, "flops": 4 * sum(held) * kv_heads * d + 4 * tokens * heads * d}


def _exact_draft(s):
    q, k_cache, v_cache = s["q"], s["k_cache"], s["v_cache"]
    B, S, heads, d = q.shape
    page, kv_heads = k_cache.shape[1:3]
    group = heads // kv_heads
    out = torch.zeros(B, S, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((B, S, heads), -math.inf, dtype=torch.float64, device=q.device)
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["drafted"].tolist())):
        c = min(c, n)
        if not c:
            continue
        parents = list(range(-1, c - 1)) if s["parents"] is None else s["parents"][b].tolist()
        see = torch.zeros(c, n, dtype=torch.bool)
        for i in range(c):
            trail, j = [], i
            while j >= 0:
                trail.append(n - c + j)
                j = parents[j]
            back = len(trail)  # tokens of the drafts that it sees; before them the context
            seen = trail if not s["window"] else trail[:s["window"]]
            from_ = 0 if not s["window"] else max(0, n - c - max(0, s["window"] - back))
            see[i, from_:n - c] = True
            see[i, seen] = True
        see = see.to(q.device)
        t = torch.arange(n, device=q.device)
        at = s["page_table"][b].long()[t // page]
        for h in range(kv_heads):
            mine = slice(h * group, (h + 1) * group)
            x = q[b, :c, mine].double().reshape(c * group, d)
            score = x @ k_cache[at, t % page, h].double().T.contiguous() * s["scale"]
            score = score.view(c, group, n).masked_fill(~see[:, None], -math.inf)
            lse[b, :c, mine] = torch.logsumexp(score, 2)
            p = torch.softmax(score, 2).view(c * group, n)
            out[b, :c, mine] = (p @ v_cache[at, t % page, h].double()).view(c, group, d)
    return out, lse


def _exact_keep(s):
    k, v, page = s["k_cache"].double(), s["v_cache"].double(), s["k_cache"].shape[1]
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["drafted"].tolist())):
        t = s["path"][b].long()
        src = n - min(c, n) + t[t >= 0]
        dst = n - min(c, n) + torch.arange(len(src), device=k.device)
        pages = s["page_table"][b].long()
        for cache in (k, v):  # (the right side is read whole before any is written)
            cache[pages[dst // page], dst % page] = cache[pages[src // page], src % page]
    return k, v


def _exact_bounds(s):
    lo, hi = s["lo"].double(), s["hi"].double()
    page = s["k_cache"].shape[1]
    for b, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
        c = min(c, n)
        if not c:
            continue
        t = torch.arange(n - c, n, device=lo.device)
        k = s["k_cache"][s["page_table"][b].long()[t // page], t % page].double()
        columns = torch.arange((n - c) // page, (n - 1) // page + 1, device=lo.device)
        pages = s["page_table"][b].long()[columns]
        at = (t // page - columns[0])[:, None, None].expand_as(k)
        fresh = columns * page >= n - c
        for bound, kind, far in ((lo, "amin", math.inf), (hi, "amax", -math.inf)):
            begin = torch.where(fresh[:, None, None], far, bound[pages])
            bound[pages] = begin.scatter_reduce(0, at, k, kind)
    return lo, hi


def _exact_sparse(s):
    q, k_cache, v_cache = s["q"], s["k_cache"], s["v_cache"]
    B, heads, d = q.shape
    page, kv_heads = k_cache.shape[1:3]
    group, top = heads // kv_heads, s["top"]
    out = torch.zeros(B, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((B, heads), -math.inf, dtype=torch.float64, device=q.device)
    columns = torch.full((B, kv_heads, top), -1, dtype=torch.int32, device=q.device)
    for b, n in enumerate(s["lengths"].tolist()):
        held = -(-n // page)
        pages = s["page_table"][b, :held].long()
        for h in range(kv_heads if n else 0):
            mine = slice(h * group, (h + 1) * group)
            x = q[b, mine].double()
            low, high = s["lo"][pages, h].double(), s["hi"][pages, h].double()
            bound = torch.zeros(held, dtype=torch.float64, device=q.device)
            for y in x:
                bound += torch.maximum(y * low, y * high).sum(1)
            bound[:s["first"]] = math.inf
            bound[max(0, held - s["last"]):] = math.inf
            rank = torch.argsort(bound, descending=True, stable=True)[:top].sort().values
            columns[b, h, :len(rank)] = rank.int()
            t = (rank[:, None] * page + torch.arange(page, device=q.device)).view(-1)
            t = t[t < n]
            at = pages[t // page]
            score = x @ k_cache[at, t % page, h].double().T.contiguous() * s["scale"]
            lse[b, mine] = torch.logsumexp(score, 1)
            out[b, mine] = torch.softmax(score, 1) @ v_cache[at, t % page, h].double()
    return out, lse, columns


def exact(case, seed):
    """In 64 bits; nothing for what chooses, whose outputs are whole numbers."""
    kind = {"draft": _exact_draft, "keep": _exact_keep, "bounds": _exact_bounds,
            "sparse": _exact_sparse}.get(case["op"])
    return kind(prepare(case, seed)) if kind else None
