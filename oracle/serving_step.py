"""Appending to a paged cache, 4-bit cache rows and token log probabilities (the
oracle of ``cache_ops.append_paged_context``, of the 4-bit attentions' caches
and of ``ops.token_logprobs``).  Tensors are on the CPU."""

from __future__ import annotations

import math

import torch

#: magnitudes of the e2m1 codes 0 .. 7; code + 8 is the negative
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP8 = torch.float8_e4m3fn


def values4(codes: torch.Tensor, factors: torch.Tensor) -> torch.Tensor:
    """fp64 values (..., D) of codes (..., D / 2) and factors (..., D / 16)."""
    signed = torch.tensor(E2M1 + tuple(-c for c in E2M1), dtype=torch.float64)
    c = signed[torch.stack([codes & 15, codes >> 4], -1).long()].flatten(-2)
    return (c.unflatten(-1, (-1, 16)) * factors.float().double()[..., None]).flatten(-2)


def quantise4(x: torch.Tensor):
    """(codes, factors) of rows (..., D), by the distance to every code; quotients in x's own type."""
    g = x.unflatten(-1, (-1, 16))
    top = torch.where(torch.isnan(g).any(-1), math.nan, g.abs().amax(-1)).to(x.dtype)
    factors = (top / 6).clamp(max=448.0).float().to(FP8)
    f = factors.float().to(x.dtype)[..., None]
    y = torch.where(f == 0, 0.0, g.abs() / f)
    grid = torch.tensor(E2M1, dtype=torch.float64)
    far = (y.double().clamp(max=6.0)[..., None] - grid).abs()
    low = far.argmin(-1)  # the lower of two as near
    high = (low + 1).clamp(max=7)
    tie = far.gather(-1, low[..., None])[..., 0] == far.gather(-1, high[..., None])[..., 0]
    code = torch.where(tie & (low % 2 == 1), high, low)
    code = torch.where(torch.isnan(y), 0, code) + 8 * torch.signbit(g)
    code = code.flatten(-2).unflatten(-1, (-1, 2)).to(torch.uint8)
    return code[..., 0] | code[..., 1] << 4, factors


def rotate(x: torch.Tensor, cos_sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x (tokens, heads, D) by cos_sin (tokens, rotary / 2, 2), each product and sum in x's type."""
    n = 2 * cos_sin.shape[1]
    out = x.clone()
    for i in range(n // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n // 2)
        c, s = cos_sin[:, i, 0].to(x.dtype)[:, None], cos_sin[:, i, 1].to(x.dtype)[:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def token_logprobs(logits: torch.Tensor, tokens, top_k: int, temperature: float):
    """fp64 (logprobs, entropy, ids, their logprobs) of rows (rows, V), one row after the other."""
    lps, ents, ids, tops = [], [], [], []
    for row, t in zip(logits.double() / temperature, tokens):
        order = sorted(range(row.numel()), key=lambda i: (-row[i].item(), i))[:top_k] if row.numel() < 4096 else \
            torch.sort(row, descending=True, stable=True).indices[:top_k].tolist()
        if (row == -math.inf).all():
            lp, ent = torch.full_like(row, -math.inf), torch.zeros((), dtype=torch.float64)
        else:
            d = row - row.max()  # first: rows of 1e38 leave no place for a logarithm
            lp = d - d.exp().sum().log()
            ent = -torch.where(lp == -math.inf, 0.0, lp.exp() * lp).sum()
        lps.append(lp[t] if 0 <= t < row.numel() else torch.tensor(-math.inf, dtype=torch.float64))
        ents.append(ent)
        ids.append(torch.tensor(order, dtype=torch.int64))
        tops.append(lp[order] if top_k else lp[:0])
    return torch.stack(lps), torch.stack(ents), torch.stack(ids), torch.stack(tops)
