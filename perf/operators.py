"""What the serving operators' speed is measured on.

Every case is one call of an operator that a serving step makes beside
MhcPre, with its tensors in hand (torch.ops.mhcpre.*):

  attention  paged_attention: one new token per sequence over a paged cache;
  rope       qk_norm_rope: norms of queries and keys per head and the rotation,
             on views of one fused projection's output; or with the keys and
             values written into the cache's pages (qk_norm_rope_append);
  update     cache_update: a step's page table (keep, fork, free, extend);
  compact    cache_compact: the moves that bring the pages in use to the front;
  copy       cache_copy_pages: page contents, for forks and compaction.

The plain forms are elementary torch operations in 32 bits, rounded once at
the end.  Only the rotation's angle is a product in 64 bits, in both forms and
in the definition: at position 10^5 a product in 32 bits is off by 10^-2 rad.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attention(B, heads, kv_heads, d, length, page, dtype, ragged=True, window=0):
    return dict(op="attention", B=B, heads=heads, kv_heads=kv_heads, d=d, length=length, page=page,
                dtype=dtype, ragged=ragged, window=window)


def _rope(T, heads, kv_heads, d, rot, dtype, append, norm=True, interleaved=False, stretch=1.0,
          page=64, start=0):
    return dict(op="rope", T=T, heads=heads, kv_heads=kv_heads, d=d, rot=rot, dtype=dtype,
                append=append, norm=norm, interleaved=interleaved, stretch=stretch, page=page,
                start=start)


def _tables(op, rows, width, pages, page, filled, tokens=1):
    return dict(op=op, rows=rows, width=width, pages=pages, page=page, filled=filled, tokens=tokens)


def _copy(moved, kv_heads, d, page, dtype, slot_major=False):
    return dict(op="copy", moved=moved, kv_heads=kv_heads, d=d, page=page, dtype=dtype,
                slot_major=slot_major)


def listed():
    return [
        # One user's chat, 1000 tokens in: latency and the join count.
        dict(_attention(1, 32, 8, 128, 1000, 16, "bf16", False), name="attention_one"),
        # The usual serving step: a decode batch of sequences of all ages.
        dict(_attention(64, 32, 8, 128, 8192, 64, "fp16"), name="attention_batch"),
        # No shared heads, odd batch, page and head sizes, a sliding window.
        dict(_attention(13, 24, 24, 96, 5000, 7, "fp16", window=1111), name="attention_odd_window"),
        # The largest: long documents, eight query heads to each of the cache's.
        dict(_attention(4, 64, 8, 128, 131072, 64, "bf16"), name="attention_long"),
        # A prefill chunk far into a stretched context: part of the head, neighbouring pairs.
        dict(_rope(8192, 64, 8, 128, 64, "fp16", False, interleaved=True, stretch=4.0,
                   start=100000), name="rope_prefill"),
        # A decode step's new tokens into the cache.
        dict(_rope(64, 32, 8, 128, 128, "bf16", True), name="rope_append_decode"),
        # Page tables of a small server's step, and of a large one's with prompts and small pages.
        dict(_tables("update", 64, 128, 4096, 64, 0.75), name="update_small"),
        dict(_tables("update", 1000, 2048, 200001, 16, 0.6, tokens=16), name="update_large"),
        # Compaction's plan for the same two pools.
        dict(_tables("compact", 64, 128, 4096, 64, 0.5), name="compact_small"),
        dict(_tables("compact", 1000, 2048, 200001, 16, 0.6), name="compact_large"),
        # Contents: the partial pages of a few forks, and a pool's compaction.
        dict(_copy(6, 8, 128, 16, "bf16", True), name="copy_forks"),
        dict(_copy(2500, 8, 128, 64, "fp16"), name="copy_compaction"),
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def _padded(c):
    """Cache values of an attention case when every sequence has the longest's length."""
    return c["B"] * c["length"] * c["kv_heads"] * c["d"]


def draw(rng):
    largest = max(_padded(c) for c in listed() if c["op"] == "attention")
    op = rng.choice(("attention", "attention", "attention", "rope", "rope", "update", "compact",
                     "copy"))
    dtype = rng.choice(("fp16", "bf16"))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 3, 4, 5, 8, 16))
    d = rng.choice((64, 96, 128, 128, 128, 192, 256))
    page = rng.choice((1, 7, 16, 16, 32, 64, 64, 128))
    while op == "attention":
        length = _log(rng, 1, 131072)
        c = _attention(_log(rng, 1, 512), heads, kv_heads, d, length, page, dtype,
                       rng.random() < 0.8, _log(rng, 1, length) if rng.random() < 0.25 else 0)
        if _padded(c) <= largest // 2:
            return c
    if op == "rope":
        T = _log(rng, 1, min(16384, 8192 * 72 * 128 // ((heads + kv_heads) * d)))
        return _rope(T, heads, kv_heads, d, rng.choice((d, d, d // 2, 32)), dtype,
                     rng.random() < 0.6, rng.random() < 0.7, rng.random() < 0.4,
                     rng.choice((1.0, 1.0, 8.0)), page, _log(rng, 1, 500000))
    if op == "copy":
        moved = _log(rng, 1, max(2, 2500 * 8 * 128 * 64 // (kv_heads * d * page)))
        return _copy(min(moved, 20000), kv_heads, d, page, dtype, rng.random() < 0.5)
    return _tables(op, _log(rng, 4, 1000), _log(rng, 4, 2048), _log(rng, 64, 200001), page,
                   rng.uniform(0.1, 0.9), rng.choice((1, 1, 1, 5, 64)))


def _lengths(case):
    """An attention case's lengths: all the longest, or spread from short ones (an idle row of
    length 0 among them in batches of more than 8) to the longest."""
    B, longest = case["B"], case["length"]
    if not case["ragged"]:
        return [longest] * B
    lengths = [max(1, round(longest * ((i + 1) / B) ** 2)) for i in range(B)]
    if B > 8:
        lengths[0] = 0
    return lengths


def _row_pages(case):
    """Pages that each row of a page table holds, short rows to long ones, `filled` of the pool."""
    rows = case["rows"]
    total = sum((i + 1) ** 2 for i in range(rows))
    room = case["filled"] * case["pages"]
    return [min(case["width"], int(room * (i + 1) ** 2 / total)) for i in range(rows)]


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
    """A page table int32 [rows, width]: distinct pages of the pool, in no order, then -1."""
    counts = torch.tensor(counts, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda")
    column = torch.arange(width, device="cuda")
    held = column < counts[:, None]
    at = (counts.cumsum(0) - counts)[:, None] + column
    return torch.where(held, order[at.clamp(max=pages - 1)], -1).int()


def _prepare_attention(case, seed):
    g = _generator(seed)
    B, heads, kv_heads, d, page = (case[k] for k in ("B", "heads", "kv_heads", "d", "page"))
    dtype = DTYPES[case["dtype"]]
    lengths = _lengths(case)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + sum(counts) // 16 + 1
    table = _table(g, counts, max(max(counts), 1), pages)
    order = torch.randperm(B, generator=g, device="cuda")
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return {"op": "attention", "q": (2 * _normal(g, (B, heads, d))).to(dtype),
            "k_cache": _cache(g, pages, page, kv_heads, d, dtype),
            "v_cache": _cache(g, pages, page, kv_heads, d, dtype), "page_table": table[order].contiguous(),
            "lengths": lengths[order].contiguous(), "scale": d ** -0.5, "window": case["window"]}


def _prepare_rope(case, seed):
    g = _generator(seed)
    T, heads, kv_heads, d, rot, page = (case[k] for k in ("T", "heads", "kv_heads", "d", "rot", "page"))
    dtype = DTYPES[case["dtype"]]
    qkv = _normal(g, (T, (heads + 2 * kv_heads) * d), dtype)  # the fused projection's output
    q, k, v = qkv.split([heads * d, kv_heads * d, kv_heads * d], 1)
    stretch = case["stretch"]
    inv_freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot) / stretch
    if case["append"]:  # tokens of many sequences, each at its own position
        positions = torch.randint(0, case["start"] + 8192, (T,), generator=g, device="cuda")
    else:  # a chunk of one sequence
        positions = case["start"] + torch.arange(T, device="cuda")
    s = {"op": "rope", "append": case["append"], "q": q.view(T, heads, d), "k": k.view(T, kv_heads, d),
         "v": v.view(T, kv_heads, d), "positions": positions, "inv_freq": inv_freq, "eps": EPS,
         "interleaved": case["interleaved"], "amplitude": 1 + 0.1 * math.log(stretch),
         "q_weight": 1 + 0.1 * _normal(g, (d,)) if case["norm"] else None,
         "k_weight": 1 + 0.1 * _normal(g, (d,)) if case["norm"] else None}
    if case["append"]:
        pages = -(-T // page) + 3
        order = torch.randperm(pages * page, generator=g, device="cuda")
        slots, spare = order[:T].clone(), order[T].clone()
        if T > 20:  # padding of a batch
            slots[::19] = -1
        s.update(slots=slots, spare=spare, k_cache=_cache(g, pages, page, kv_heads, d, dtype),
                 v_cache=_cache(g, pages, page, kv_heads, d, dtype))
    return s


def _prepare_tables(case, seed):
    g = _generator(seed)
    R, W, N, page, tokens = (case[k] for k in ("rows", "width", "pages", "page", "tokens"))
    counts = _row_pages(case)
    table = _table(g, counts, W, N)
    slack = torch.randint(0, page, (R,), generator=g, device="cuda")
    lengths = (torch.tensor(counts, device="cuda") * page - slack).clamp(min=0)
    order = torch.randperm(R, generator=g, device="cuda")
    s = {"op": case["op"], "page_table": table[order].contiguous(), "lengths": lengths[order].int(),
         "pages": N, "page": page, "tokens": tokens}
    if case["op"] == "update":
        # Most rows go on; one in ten goes on from another row (a beam, a shared prompt), one in
        # twenty ends.  Nearly all get a token, some a prompt's chunk.
        kind = torch.rand(R, generator=g, device="cuda")
        row = torch.arange(R, device="cuda")
        other = torch.randint(0, R, (R,), generator=g, device="cuda")
        s["parents"] = torch.where(kind < 0.1, other, torch.where(kind < 0.15, -1, row)).int()
        add = torch.randint(0, tokens + 1, (R,), generator=g, device="cuda")
        s["counts"] = torch.where(torch.rand(R, generator=g, device="cuda") < 0.8, 1, add).int()
    return s


def _prepare_copy(case, seed):
    g = _generator(seed)
    moved, kv_heads, d, page = (case[k] for k in ("moved", "kv_heads", "d", "page"))
    dtype = DTYPES[case["dtype"]]
    pages = 2 * moved + moved // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda").int()
    src, dst = order[:moved].clone(), order[moved:2 * moved].clone()
    if moved > 4:  # rows that need no copy
        src[::5] = -1
        dst[::5] = -1
    return {"op": "copy", "src": src, "dst": dst, "spare": order[2 * moved].clone(),
            "k_cache": _cache(g, pages, page, kv_heads, d, dtype, case["slot_major"]),
            "v_cache": _cache(g, pages, page, kv_heads, d, dtype, case["slot_major"])}


_PREPARE = {"attention": _prepare_attention, "rope": _prepare_rope, "update": _prepare_tables,
            "compact": _prepare_tables, "copy": _prepare_copy}


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _plain_attention(s):
    q, table, lengths = s["q"], s["page_table"].long(), s["lengths"]
    N, page, kv_heads, d = s["k_cache"].shape
    B, heads, _ = q.shape
    L = table.shape[1] * page
    rows = table.clamp(min=0)
    k = s["k_cache"].transpose(1, 2)[rows].float()  # [B, W, kv_heads, page, d]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, kv_heads, d, L)
    score = torch.matmul(q.float().view(B, kv_heads, heads // kv_heads, d), k) * s["scale"]
    del k
    t = torch.arange(L, device=q.device)
    seen = t < lengths[:, None]
    if s["window"]:
        seen = seen & (t >= lengths[:, None] - s["window"])
    seen = seen.view(B, 1, 1, L)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(3, keepdim=True)
    v = s["v_cache"].transpose(1, 2)[rows].float().permute(0, 2, 1, 3, 4).reshape(B, kv_heads, L, d)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    return out.view(B, heads, d).to(q.dtype), lse.view(B, heads)


def _rotated(x, weight, s, cos, sin):
    """Norm (with a weight) and rotation of x [T, heads, d] in the type of cos and sin."""
    x = x.to(cos.dtype)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + s["eps"]) * weight.to(cos.dtype)
    rot = 2 * cos.shape[2]
    turned, rest = x[..., :rot], x[..., rot:]
    if s["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
    ya, yb = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((ya, yb), 3).flatten(2) if s["interleaved"] else torch.cat((ya, yb), 2)
    return torch.cat((turned, rest), 2)


def _plain_rope(s):
    angle = torch.remainder(s["positions"].double()[:, None] * s["inv_freq"], 2 * math.pi).float()
    cos = (torch.cos(angle) * s["amplitude"])[:, None]
    sin = (torch.sin(angle) * s["amplitude"])[:, None]
    q = _rotated(s["q"], s["q_weight"], s, cos, sin).to(s["q"].dtype)
    k = _rotated(s["k"], s["k_weight"], s, cos, sin).to(s["k"].dtype)
    if not s["append"]:
        return q, k
    page = s["k_cache"].shape[1]
    # A row without a slot writes to a slot of nobody's what that holds.
    slot = s["slots"]
    on, at = (slot >= 0)[:, None, None], torch.where(slot >= 0, slot, s["spare"])
    for cache, rows in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        cache[at // page, at % page] = torch.where(on, rows, cache[at // page, at % page])
    return q, s["k_cache"], s["v_cache"]


def _base(table, lengths, N, page):
    """A table's valid entries of the pages that the lengths hold (others -1), their count."""
    R, W = table.shape
    held = (lengths + page - 1) // page
    column = torch.arange(W, device=table.device)
    good = (column < held[:, None]) & (table >= 0) & (table < N)
    return torch.where(good, table, -1), held, column


def _ranked(mask, size):
    """The places where mask is true, ascending, in `size` entries (the rest -1)."""
    rank = torch.cumsum(mask, 0) - 1
    at = torch.where(mask & (rank < size), rank, size)
    out = torch.full((size + 1,), -1, dtype=torch.long, device=mask.device)
    out.scatter_(0, at, torch.arange(mask.numel(), device=mask.device))
    return out[:size]


def _plain_update(s):
    N, page, tokens = s["pages"], s["page"], s["tokens"]
    table, parents = s["page_table"].long(), s["parents"].long()
    R, W = table.shape
    alive = (parents >= 0) & (parents < R)
    old = s["lengths"].long().clamp(0, W * page)
    length = torch.where(alive, old[parents.clamp(0, R - 1)], 0)
    table, held, column = _base(table[parents.clamp(0, R - 1)], length, N, page)
    refs = torch.zeros(N + W, dtype=torch.long, device=table.device)  # absent entries: W places
    refs.scatter_add_(0, torch.where(table >= 0, table, N + column).view(-1),
                      torch.ones_like(table).view(-1))
    add = s["counts"].long().clamp(0, tokens)
    grown = (length + add + page - 1) // page
    last = table.gather(1, (held - 1).clamp(min=0)[:, None])[:, 0]
    fits = (add > 0) & (grown <= W)
    private = fits & (length % page != 0) & (last >= 0) & (refs[last.clamp(min=0)] > 1)
    need = torch.where(fits, private + grown - held, 0)
    upto = torch.cumsum(need, 0)
    free = refs[:N] == 0
    served = fits & ((need == 0) | (upto <= free.sum()))
    order = _ranked(free, N)
    first = upto - need
    dst = torch.where(served & private, order[first.clamp(max=N - 1)], -1)
    src = torch.where(served & private, last, -1)
    at = (first + private)[:, None] + column - held[:, None]
    new = served[:, None] & (column >= held[:, None]) & (column < grown[:, None])
    table = torch.where(new, order[at.clamp(0, N - 1)], table)
    swap = (served & private)[:, None] & (column == held[:, None] - 1)
    table = torch.where(swap, dst[:, None], table)
    granted = torch.where(served, add, 0)
    i = torch.arange(tokens, device=table.device)
    t = length[:, None] + i
    where = table.gather(1, (t // page).clamp(max=W - 1))
    slots = torch.where((i < granted[:, None]) & (where >= 0), where * page + t % page, -1)
    return table.int(), (length + granted).int(), slots, granted.int(), src.int(), dst.int()


def _plain_compact(s):
    N, page = s["pages"], s["page"]
    R, W = s["page_table"].shape
    table, _, _ = _base(s["page_table"].long(), s["lengths"].long().clamp(0, W * page), N, page)
    used = torch.zeros(N + 1, dtype=torch.bool, device=table.device)
    used.scatter_(0, torch.where(table >= 0, table, N).view(-1), True)
    used = used[:N]
    count = used.sum()
    index = torch.arange(N, device=table.device)
    moves = used & (index >= count)
    src = _ranked(moves, N // 2)
    dst = torch.where(src >= 0, _ranked(~used & (index < count), N // 2), -1)
    rank = (torch.cumsum(moves, 0) - 1).clamp(min=0)
    to = torch.where(moves, torch.cat((dst, dst.new_zeros(1)))[rank], index)
    table = torch.where(table >= 0, to[table.clamp(min=0)], -1)
    return table.int(), src.int(), dst.int(), count.int().view(1)


def _plain_copy(s):
    # A pair of -1 writes to a page of nobody's what that holds.
    on = (s["src"] >= 0) & (s["dst"] >= 0)
    src = torch.where(on, s["src"], s["spare"]).long()
    dst = torch.where(on, s["dst"], s["spare"]).long()
    for cache in (s["k_cache"], s["v_cache"]):
        cache[dst] = cache[src]
    return s["k_cache"], s["v_cache"]


_PLAIN = {"attention": _plain_attention, "rope": _plain_rope, "update": _plain_update,
          "compact": _plain_compact, "copy": _plain_copy}


_ops = None


def _own(s):
    global _ops
    if _ops is None:
        import __graft_entry__

        __graft_entry__.load_package().torch_ops()
        _ops = torch.ops.mhcpre
    ops = _ops
    if s["op"] == "attention":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                   s["scale"], s["window"])
    if s["op"] == "update":
        return ops.cache_update(s["page_table"], s["lengths"], s["parents"], s["counts"], s["pages"],
                                s["page"], s["tokens"])
    if s["op"] == "compact":
        return ops.cache_compact(s["page_table"], s["lengths"], s["pages"], s["page"])
    if s["op"] == "copy":
        ops.cache_copy_pages(s["k_cache"], s["v_cache"], s["src"], s["dst"])
        return s["k_cache"], s["v_cache"]
    if not s["append"]:
        return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"],
                                s["k_weight"], s["eps"], s["interleaved"], s["amplitude"])
    q = ops.qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["slots"],
                                s["k_cache"], s["v_cache"], s["q_weight"], s["k_weight"], s["eps"],
                                s["interleaved"], s["amplitude"])
    return q, s["k_cache"], s["v_cache"]


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


def work(case):
    if case["op"] == "attention":
        window = case["window"] or case["length"]
        tokens = sum(min(n, window) for n in _lengths(case))
        pages = sum(-(-min(n, window) // case["page"]) for n in _lengths(case))
        B, heads, kv_heads, d = (case[k] for k in ("B", "heads", "kv_heads", "d"))
        # the cache, q and out, lse, the table's entries and the lengths
        size = 2 * tokens * kv_heads * d * 2 + 2 * B * heads * d * 2 + 4 * B * heads + 4 * pages + 4 * B
        return {"bytes": size, "flops": 4 * tokens * heads * d}
    if case["op"] == "rope":
        T, heads, kv_heads, d, rot = (case[k] for k in ("T", "heads", "kv_heads", "d", "rot"))
        values = T * (heads + kv_heads) * d
        size = 2 * 2 * values + 8 * T + 4 * rot + (8 * d if case["norm"] else 0)
        if case["append"]:
            size += 2 * 2 * T * kv_heads * d + 8 * T
        return {"bytes": size, "flops": (4 if case["norm"] else 0) * values + 3 * T * (heads + kv_heads) * rot}
    if case["op"] == "copy":
        pairs = case["moved"] - (-(-case["moved"] // 5) if case["moved"] > 4 else 0)
        size = 2 * 2 * pairs * case["page"] * case["kv_heads"] * case["d"] * 2 + 8 * case["moved"]
        return {"bytes": size, "flops": 0}
    R, W, N = case["rows"], case["width"], case["pages"]
    size = 4 * sum(_row_pages(case)) + 4 * R * W + 4 * R  # entries held, the new table, the lengths
    if case["op"] == "update":
        size += 4 * R * (2 + 4) + 8 * R * case["tokens"]
    else:
        size += 4 * 2 * (N // 2) + 4
    return {"bytes": size, "flops": 0}


def _exact_attention(s):
    q, k_cache, v_cache = s["q"], s["k_cache"], s["v_cache"]
    B, heads, d = q.shape
    page, kv_heads = k_cache.shape[1:3]
    out = torch.zeros(B, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((B, heads), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["lengths"].tolist()):
        t = torch.arange(max(0, n - s["window"]) if s["window"] else 0, n, device=q.device)
        if not t.numel():
            continue
        at = s["page_table"][b].long()[t // page]
        for h in range(kv_heads):
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            score = q[b, group].double() @ k_cache[at, t % page, h].double().T.contiguous() * s["scale"]
            lse[b, group] = torch.logsumexp(score, 1)
            out[b, group] = torch.softmax(score, 1) @ v_cache[at, t % page, h].double()
    return out, lse


def _exact_rope(s):
    rot = 2 * s["inv_freq"].numel()
    turn = torch.polar(torch.full((), s["amplitude"], dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["inv_freq"])[:, None]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + s["eps"]) * weight.double()
        y = x.clone()
        places = torch.arange(rot, device="cuda")
        one, two = (places[0::2], places[1::2]) if s["interleaved"] else places.view(2, -1)
        z = torch.complex(x[..., one], x[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        return y

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    if not s["append"]:
        return q, k
    caches = []
    for cache, rows in ((s["k_cache"], k), (s["v_cache"], s["v"].double())):
        cache = cache.double()
        on = s["slots"] >= 0
        slot, page = s["slots"][on], cache.shape[1]
        cache[slot // page, slot % page] = rows[on]
        caches.append(cache)
    return q, caches[0], caches[1]


def exact(case, seed):
    """In 64 bits; nothing for the page operators, whose outputs are whole numbers and copies."""
    if case["op"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["op"] == "rope":
        return _exact_rope(prepare(case, seed))
    return None
