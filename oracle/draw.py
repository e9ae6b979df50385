"""The filtered draw from given uniform numbers, in 64 bits, one row at a time."""

from __future__ import annotations

import math

import torch


def draw_row(logits: torch.Tensor, u: float, temperature: float, top_k: int = 0, top_p: float = 1.0,
             min_p: float = 0.0) -> int:
    raw = logits.float().cpu()
    if not temperature > 0:
        return int(torch.argmax(raw))
    l = raw.double().nan_to_num(-math.inf, math.inf, -math.inf)
    top = l.max().item()
    if top == -math.inf:
        return int(torch.argmax(torch.where(raw.isnan(), -math.inf, raw)))
    if top == math.inf:
        w = (l == math.inf).double()
    else:
        w = torch.exp((l - top) / temperature)
        w = torch.where(l == top, 1.0, w)
    order = torch.argsort(l, descending=True, stable=True)
    n = len(order) if top_k <= 0 else min(top_k, len(order))
    ws = w[order]
    if min_p > 0:
        n = min(n, int((ws >= min(min_p, 1.0)).sum()))
    n = max(n, 1)
    if top_p < 1:
        before = torch.cumsum(ws[:n], 0) - ws[:n]
        n = max(1, int((before < top_p * ws[:n].sum()).sum()))
    kept = torch.zeros_like(w)
    kept[order[:n]] = ws[:n]
    cum = torch.cumsum(kept, 0)
    hit = (cum > u * cum[-1]).nonzero()
    return int(hit[0]) if len(hit) else int(order[:n].max())
