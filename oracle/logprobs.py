"""Oracle of the token log-probabilities (test infrastructure), in 64 bits."""
from __future__ import annotations

import math

import torch


def token_logprobs(logits, tokens, top_k=0, temperature=1.0, suppress=None):
    """(logprobs, entropy, top_logprobs float64, top_ids int64) of logits [R, V]."""
    R, V = logits.shape
    x = logits.detach().cpu().double()
    if suppress is not None:
        x = x.masked_fill(suppress.cpu()[None], -math.inf)
    lp, ent, tops, ids = [], [], [], []
    for r in range(R):
        p = torch.log_softmax(x[r] / temperature, 0)
        if not bool((x[r] > -math.inf).any()) and not bool(torch.isnan(x[r]).any()):
            p = torch.full((V,), -math.inf, dtype=torch.float64)
        t = int(tokens[r])
        lp.append(float(p[t]) if 0 <= t < V else math.nan)
        ent.append(float(-(torch.where(p == -math.inf, torch.zeros_like(p), p.exp() * p)).sum()))
        order = torch.sort(x[r], descending=True, stable=True).indices[:top_k]     # ties keep the lower index first
        ids.append(order)
        tops.append(p[order])
    stack = lambda v, dt: torch.stack(v) if R else torch.zeros(0, top_k, dtype=dt)  # noqa: E731
    return torch.tensor(lp, dtype=torch.float64), torch.tensor(ent, dtype=torch.float64), stack(tops, torch.float64), stack(ids, torch.int64)
