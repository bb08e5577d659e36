"""The operators on a paged key/value cache in 64 bits, request by request (the
oracle of ``flashmap_b200.cache_ops``).  Tensors are on the CPU."""

from __future__ import annotations

import math

import torch


def rows_of(pool: torch.Tensor, table: torch.Tensor, length: int) -> torch.Tensor:
    """(length, kv_heads, head_dim) rows of one request in fp64."""
    j = torch.arange(length)
    return pool.float().double()[table[j // pool.shape[2]].long(), :, j % pool.shape[2]]


def visible(positions: torch.Tensor, length: int, window: int, sinks: int) -> torch.Tensor:
    """(rows, length): whether the row at each position sees each key."""
    j, p = torch.arange(length)[None], positions[:, None]
    ok = j <= p
    return ok & ((p - j < window) | (j < sinks)) if window > 0 else ok


def attend(q, k, v, seen, scale: float):
    """One head: q (rows, D), k and v (n, D), seen (rows, n), fp64.  Returns the
    outputs, the weights, and sum |w| |v|, which errors scale with."""
    s = (q @ k.T) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((s.shape[0], 1), -math.inf, dtype=s.dtype)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    e = e.masked_fill(~seen, 0.0)
    total = e.sum(-1, keepdim=True)
    w = e / torch.where(total == 0, 1.0, total)
    vs = torch.where(seen.any(0)[:, None], v, 0.0)  # what no row sees takes no part
    return w @ vs, w, w @ vs.abs()


def window_attention(q, k_pool, v_pool, cu, lengths, table, scale, window=0, sinks=0, descales=None):
    """(out, scale of out, weights): q (tokens, heads, D); weights[r] (heads, rows, length)."""
    T, H, D = q.shape
    KH = k_pool.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    weights = []
    for r, L in enumerate(lengths):
        a, b = int(cu[r]), int(cu[r + 1])
        k, v = rows_of(k_pool, table[r], L), rows_of(v_pool, table[r], L)
        if descales is not None:
            k = k * descales[0, r].double()[None, :, None]
            v = v * descales[1, r].double()[None, :, None]
        seen = visible(torch.arange(L - (b - a), L), L, window, sinks)
        per = []
        for h in range(H):
            c = h // (H // KH)
            out[a:b, h], w, mag[a:b, h] = attend(q[a:b, h].double(), k[:, c], v[:, c], seen, scale)
            per.append(w)
        weights.append(torch.stack(per))
    return out, mag, weights


def decode_attention(q, k_pool, v_pool, lengths, table, scale, window=0, sinks=0, descales=None):
    """(out, scale of out, gathered weights per request (kv_heads, length)) of one new token each."""
    KH = k_pool.shape[1]
    cu = torch.tensor([0] + [1 if L > 0 else 0 for L in lengths]).cumsum(0)
    rows = [r for r, L in enumerate(lengths) if L > 0]
    o, m, w = window_attention(q[rows], k_pool, v_pool, cu, lengths, table, scale, window, sinks, descales)
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    out[rows], mag[rows] = o, m
    sums = [x.sum(1).view(KH, q.shape[1] // KH, x.shape[-1]).sum(1) for x in w]
    return out, mag, sums


def evict(sums, lengths, budget: int, sinks: int, recent: int):
    """kept[r][h]: the positions that stay, in order."""
    kept = []
    for r, L in enumerate(lengths):
        per = []
        for h in range(sums.shape[1]):
            if L <= budget:
                per.append(list(range(L)))
                continue
            middle = range(sinks, L - recent)
            row = sums[r, h].tolist()
            order = sorted(middle, key=lambda j: (row[j] != row[j], -row[j] if row[j] == row[j] else 0.0, j))
            per.append(sorted(list(range(sinks)) + list(range(L - recent, L)) + order[: budget - sinks - recent]))
        kept.append(per)
    return kept
