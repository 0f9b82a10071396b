"""Plain 64-bit implementations of the operators for drafted tokens and selected pages, and their bounds."""
from __future__ import annotations

import math

import torch

from serve_ref import ROUND, TINY


def attend(q, k, v, scale, dtype):
    """(out, lse, bound of out, bound of lse) of query heads q [G, d] over keys and values [n, d], in 64 bits.

    The bounds: a score of d products, its scaling and its difference from the maximum are off by at most (d + 4)
    roundings of scale * sum |q_i k_i| and one of |s - max|; exp and log by four roundings; sums of n terms by n
    roundings of the sum of magnitudes; weights are held in 16 bits at least (2^-16); the last rounding is the type's."""
    q, k, v = q.double(), k.double(), v.double()
    eps = ROUND[torch.float32]
    s = q @ k.T * scale
    off = (q.shape[1] + 4) * eps * abs(scale) * (q.abs() @ k.abs().T)
    top = s.amax(1, keepdim=True)
    off = off + off.amax(1, keepdim=True) + 2 * eps * (s - top).abs() + 8 * eps
    p = torch.softmax(s, 1)
    rel = (p * off).sum(1, keepdim=True) + (k.shape[0] + 8) * eps
    out, lse = p @ v, torch.logsumexp(s, 1)
    out_bound = (p * off) @ v.abs() + (rel + 2.0 ** -16) * (p @ v.abs())
    lse_bound = rel[:, 0] + 4 * eps * (1 + lse.abs()) + 2 * eps * top[:, 0].abs()
    u = ROUND[dtype]
    return out, lse, out_bound * (1 + u) + u * out.abs() + TINY[dtype], lse_bound



def paths(parents, n):
    """Each node's ancestors from the root to itself; parents: a list, or None for a chain."""
    out = []
    for i in range(n):
        p = i - 1 if parents is None else parents[i]
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def new_tokens(lengths, drafted, S, most):
    """(c, n) of every row."""
    out = []
    for L, m in zip(lengths, drafted):
        L = min(max(L, 0), most)
        n = min(max(m, 0), S, L)
        out.append((L - n, n))
    return out


def draft_attention(q, k_cache, v_cache, table, lengths, drafted, parents, scale, window=0):
    """(out, lse, bound of out, bound of lse), node by node."""
    q, table, k_cache, v_cache = q.cpu(), table.cpu().long(), k_cache.cpu(), v_cache.cpu()
    B, S, heads, d = q.shape
    pages, page, kv_heads, _ = k_cache.shape
    group = heads // kv_heads
    out, out_bound = (torch.zeros(B, S, heads, d, dtype=torch.float64) for _ in range(2))
    lse = torch.full((B, S, heads), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    for b, (c, n) in enumerate(new_tokens(lengths.tolist(), drafted.tolist(), S, table.shape[1] * page)):
        for i, path in enumerate(paths(None if parents is None else parents[b].tolist(), n)):
            at = c + len(path) - 1
            low = max(0, at - window + 1) if window else 0
            t = torch.tensor(list(range(min(low, c), c)) + [c + j for r, j in enumerate(path) if c + r >= low],
                             dtype=torch.long)
            g = table[b, t // page]
            seen = (g >= 0) & (g < pages)
            t, g = t[seen], g[seen]
            if not t.numel():
                continue
            for h in range(kv_heads):
                mine = slice(h * group, (h + 1) * group)
                got = attend(q[b, i, mine], k_cache[g, t % page, h], v_cache[g, t % page, h], scale, q.dtype)
                for to, value in zip((out, lse, out_bound, lse_bound), got):
                    to[b, i, mine] = value
    return out, lse, out_bound, lse_bound


def draft_accept(tokens, parents, drafted, chosen, lengths):
    """On Python lists; (path, accepted, next, new lengths)."""
    out = ([], [], [], [])
    for b, (row, want) in enumerate(zip(tokens, chosen)):
        L = max(lengths[b], 0)
        n = min(max(drafted[b], 0), len(row), L)
        path = [0] if n else []
        while path:
            children = [j for j in range(path[-1] + 1, n)
                        if (j - 1 if parents is None else parents[b][j]) == path[-1] and row[j] == want[path[-1]]]
            if not children:
                break
            path.append(children[0])
        for o, v in zip(out, (path + [-1] * (len(row) - len(path)), len(path), want[path[-1]] if path else -1,
                              L - n + len(path))):
            o.append(v)
    return out


def cache_keep(k_cache, v_cache, table, lengths, drafted, path):
    """On copies of the caches (on the host)."""
    k, v = k_cache.cpu().clone(), v_cache.cpu().clone()
    pages, page = k.shape[:2]
    S = path.shape[1]
    for b, (c, n) in enumerate(new_tokens(lengths.tolist(), drafted.tolist(), S, table.shape[1] * page)):
        before = -1
        for x, node in enumerate(path[b].tolist()):
            if not before < node < n:
                break
            before = node
            src, dst = (int(table[b, (c + y) // page]) for y in (node, x))
            if 0 <= src < pages and 0 <= dst < pages:
                for cache in (k, v):
                    cache[dst, (c + x) % page] = cache[src, (c + node) % page]
    return k, v


def cache_bounds(k_cache, table, lengths, counts, lo, hi, tokens):
    """On copies of lo and hi (on the host), in 64 bits."""
    k, lo, hi = k_cache.cpu().double(), lo.cpu().double(), hi.cpu().double()
    pages, page = k.shape[:2]
    for b, (begin, n) in enumerate(new_tokens(lengths.tolist(), counts.tolist(), tokens, table.shape[1] * page)):
        for column in range(begin // page, -(-(begin + n) // page) if n else 0):
            g = int(table[b, column])
            if not 0 <= g < pages:
                continue
            first, last = max(begin - column * page, 0), min(begin + n - column * page, page)
            low, high = (torch.cat((k[g, first:last], x[g][None])) if first else k[g, first:last] for x in (lo, hi))
            nan = torch.isnan(low).any(0) | torch.isnan(high).any(0)
            lo[g], hi[g] = (torch.where(nan, math.nan, x) for x in (low.amin(0), high.amax(0)))
    return lo, hi


def sparse_columns(q, lo, hi, table, lengths, page, top, first, last):
    """The columns that every kv head of every row takes, ascending, as lists."""
    q, lo, hi, table = q.cpu().double(), lo.cpu().double(), hi.cpu().double(), table.cpu().tolist()
    pages, kv_heads = lo.shape[:2]
    group = q.shape[1] // kv_heads
    out = []
    for b, L in enumerate(lengths.tolist()):
        L = min(max(L, 0), len(table[b]) * page)
        held = -(-L // page)
        rows = []
        for h in range(kv_heads):
            x = q[b, h * group:(h + 1) * group]
            up, down = torch.where(x < 0, 0.0, x).sum(0), torch.where(x > 0, 0.0, x).sum(0)
            ranks = []
            for c in range(held):
                g = table[b][c]
                if not 0 <= g < pages:
                    continue
                score = float(up @ hi[g, h] + down @ lo[g, h])
                # (always, then NaN, then by score; ties to the lower column)
                ranks.append((0 if c < first or c >= held - last else 1, 0 if math.isnan(score) else 1,
                              0.0 if math.isnan(score) else -score, c))
            rows.append(sorted(r[3] for r in sorted(ranks)[:top]))
        out.append(rows)
    return out


def sparse_attention(q, k_cache, v_cache, lo, hi, table, lengths, top, first, last, scale):
    """(out, lse, bound of out, bound of lse, columns int32 [B, kv_heads, top])."""
    page, kv_heads = k_cache.shape[1:3]
    taken = sparse_columns(q, lo, hi, table, lengths, page, top, first, last)
    q, table, k_cache, v_cache = q.cpu(), table.cpu(), k_cache.cpu(), v_cache.cpu()
    B, heads, d = q.shape
    group = heads // kv_heads
    out, out_bound = (torch.zeros(B, heads, d, dtype=torch.float64) for _ in range(2))
    lse = torch.full((B, heads), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    columns = torch.full((B, kv_heads, top), -1, dtype=torch.int32)
    for b, L in enumerate(lengths.tolist()):
        L = min(max(L, 0), table.shape[1] * page)
        for h in range(kv_heads):
            columns[b, h, :len(taken[b][h])] = torch.tensor(taken[b][h], dtype=torch.int32)
            t = torch.tensor([c * page + x for c in taken[b][h] for x in range(page) if c * page + x < L],
                             dtype=torch.long)
            if not t.numel():
                continue
            g, mine = table[b].long()[t // page], slice(h * group, (h + 1) * group)
            got = attend(q[b, mine], k_cache[g, t % page, h], v_cache[g, t % page, h], scale, q.dtype)
            for to, value in zip((out, lse, out_bound, lse_bound), got):
                to[b, mine] = value
    return out, lse, out_bound, lse_bound, columns
