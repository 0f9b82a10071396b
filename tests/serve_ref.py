"""Plain 64-bit implementations of the serving operators, and their bounds."""
from __future__ import annotations

import math

import torch

# Unit roundoff of a rounding to the type: half its spacing at 1.
ROUND = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}
# Spacing of the type's smallest values (an absolute rounding error of half of it).
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def attention(q, k_cache, v_cache, table, lengths, scale, window=0):
    """(out, lse, bound of out, bound of lse) in 64 bits, one query head after the other.

    The bounds: a score of d products, its scaling and its difference from the
    maximum are off by at most (d + 4) roundings of scale * sum |q_i k_i| and
    one of |s - max|; exp and log by four roundings; sums of n terms by n
    roundings of the sum of magnitudes; weights are held in 16 bits at least
    (2^-16); the last rounding is the type's."""
    q, table, lengths = q.cpu(), table.cpu(), lengths.cpu()
    k_cache, v_cache = k_cache.cpu(), v_cache.cpu()
    B, heads, d = q.shape
    pages, page, kv_heads, _ = k_cache.shape
    W = table.shape[1]
    out = torch.zeros(B, heads, d, dtype=torch.float64)
    lse = torch.full((B, heads), -math.inf, dtype=torch.float64)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    eps = ROUND[torch.float32]
    for b in range(B):
        L = min(max(int(lengths[b]), 0), W * page)
        t = torch.arange(max(0, L - window) if window else 0, L)
        at = table[b].long()[t // page]
        seen = (at >= 0) & (at < pages)
        t, at = t[seen], at[seen]
        if not t.numel():
            continue
        for h in range(kv_heads):
            group = slice(h * (heads // kv_heads), (h + 1) * (heads // kv_heads))
            k, v = k_cache[at, t % page, h].double(), v_cache[at, t % page, h].double()
            qh = q[b, group].double()
            s = qh @ k.T * scale
            off = (d + 4) * eps * abs(scale) * (qh.abs() @ k.abs().T)
            top = s.amax(1, keepdim=True)
            off = (off + off.amax(1, keepdim=True) + 2 * eps * (s - top).abs() + 8 * eps)
            # (a key whose weight is 0 in 32 bits has no error to speak of)
            p = torch.softmax(s, 1)
            rel = (p * off).sum(1, keepdim=True) + (len(t) + 8) * eps
            out[b, group] = p @ v
            lse[b, group] = torch.logsumexp(s, 1)
            out_bound[b, group] = (p * off) @ v.abs() + (rel + 2.0 ** -16) * (p @ v.abs())
            lse_bound[b, group] = rel[:, 0] + 4 * eps * (1 + lse[b, group].abs())
    u = ROUND[q.dtype]
    out_bound = out_bound * (1 + u) + u * out.abs() + TINY[q.dtype]
    return out, lse, out_bound, lse_bound


def norm_rope(x, weight, positions, inv_freq, eps, interleaved, amplitude):
    """(y, bound): the norm and rotation of x [T, heads, d] in 64 bits.  The
    bound: d + 8 roundings in the norm, six in the rotation, sine and cosine off
    by 2^-18, then the type's rounding."""
    x, positions = x.cpu(), positions.cpu().double()
    y = x.double()
    d = x.shape[2]
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(2, keepdim=True) + eps) * weight.cpu().double()
    slack = (d + 8) * ROUND[torch.float32] * y.abs()
    if inv_freq is not None and inv_freq.numel():
        freq = inv_freq.cpu().double()
        half = freq.numel()
        angle = (positions[:, None] * freq)[:, None]
        c, s = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
        i = torch.arange(half)
        one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b, ea, eb = y[..., one], y[..., two], slack[..., one], slack[..., two]
        y, slack = y.clone(), slack.clone()
        y[..., one], y[..., two] = a * c - b * s, a * s + b * c
        trig = (2.0 ** -18 + 6 * ROUND[torch.float32]) * abs(amplitude) * (a.abs() + b.abs())
        slack[..., one] = ea * c.abs() + eb * s.abs() + trig
        slack[..., two] = ea * s.abs() + eb * c.abs() + trig
    u = ROUND[x.dtype]
    return y, slack * (1 + u) + u * y.abs() + TINY[x.dtype]


def _held(table, lengths, page, r, pages):
    W = len(table[r])
    n = min(max(lengths[r], 0), W * page)
    return [p if 0 <= p < pages else -1 for p in table[r][:-(-n // page)]], n


def update(table, lengths, parents, counts, pages, page, tokens):
    """cache_update on Python lists; (table, lengths, slots, granted, src, dst)."""
    R, W = len(table), len(table[0]) if table else 0
    rows, refs = [], [0] * pages
    for r in range(R):
        p = parents[r]
        held, n = _held(table, lengths, page, p, pages) if 0 <= p < R else ([], 0)
        rows.append((held, n))
        for g in held:
            if g >= 0:
                refs[g] += 1
    free = [g for g in range(pages) if refs[g] == 0]
    asked = 0
    out = ([], [], [], [], [], [])
    for r, (held, n) in enumerate(rows):
        held = list(held)
        add = min(max(counts[r], 0), tokens)
        grown = -(-(n + add) // page)
        src = dst = -1
        slots = []
        if add > 0 and grown <= W:
            copy = n % page != 0 and held[-1] >= 0 and refs[held[-1]] > 1
            need = copy + grown - len(held)
            asked += need
            if need == 0 or asked <= len(free):
                mine = free[asked - need:asked]
                if copy:
                    src, dst = held[-1], mine[0]
                    held[-1] = dst
                held += mine[copy:]
                for t in range(n, n + add):
                    g = held[t // page]
                    slots.append(g * page + t % page if g >= 0 else -1)
        granted = len(slots)
        for o, v in zip(out, (held + [-1] * (W - len(held)), n + granted, slots + [-1] * (tokens - granted),
                              granted, src, dst)):
            o.append(v)
    return out


def compact(table, lengths, pages, page):
    """cache_compact on Python lists; (table, src, dst, used)."""
    rows = [_held(table, lengths, page, r, pages)[0] for r in range(len(table))]
    used = sorted({g for row in rows for g in row if g >= 0})
    U = len(used)
    src = [g for g in used if g >= U]
    dst = sorted(set(range(U)) - set(used))[:len(src)]
    to = dict(zip(src, dst))
    pad = [-1] * (pages // 2 - len(src))
    return ([[to.get(g, g) for g in row] + [-1] * (len(table[r]) - len(row)) for r, row in enumerate(rows)],
            src + pad, dst + pad, [U])
