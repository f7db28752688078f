"""Float64 restatement of token sampling: probabilities, filters and the
inverse of the running sum, one row at a time."""

from __future__ import annotations

import torch


def row(logits, uniform, temperature, top_k, top_p, min_p, slack=0.0):
    """Kept probabilities (vocabulary order, unnormalised), as a pair: the set
    kept with each limit tightened and with each limit widened by the relative
    `slack`, for comparisons in the presence of rounding."""
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), torch.tensor(-torch.inf, dtype=torch.float64), x)
    if not temperature > 0:
        top_k, temperature = 1, 1.0
    p = torch.where(x == x.max(), torch.ones_like(x), torch.exp((x - x.max()) / temperature))
    order = torch.argsort(-p, stable=True)
    sets = []
    for sign in (-1, 1):
        s = p[order]
        keep = torch.arange(x.numel()) < (top_k if top_k > 0 else x.numel())
        if sign > 0 and top_k > 1:
            # (a token that rounding makes equal to the last one kept may take its place)
            keep |= s >= s[min(top_k, x.numel()) - 1] * (1 - slack)
        s = s * keep
        if top_p < 1:
            before = torch.cumsum(s, 0) - s
            keep &= (before < top_p * s.sum() * (1 + sign * slack)) | (torch.arange(x.numel()) == 0)
        keep &= (s >= min_p * (1 - sign * slack)) | (torch.arange(x.numel()) == 0)
        sets.append(torch.zeros_like(p).scatter(0, order, p[order] * keep))
    return sets
