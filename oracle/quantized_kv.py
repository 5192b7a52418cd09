"""Oracle of the 4-bit KV cache (test infrastructure): quantisation, values and attention in 64 bits, on any device.

A group of 64 channels is stored as scale = max/15 - min/15 and bias = min, both in the cache's type, and codes
round((x - bias) / scale) in 0..15; the divisions are single-precision IEEE operations, which the codes are defined by.
"""
from __future__ import annotations

import math

import torch

GROUP = 64


def quantise(x: torch.Tensor):
    """x [..., D] -> (codes int32 [..., D/8], scales, biases [..., D/64])."""
    g = x.float().unflatten(-1, (-1, GROUP))
    fine = torch.isfinite(g).all(-1)
    lo, hi = g.amin(-1), g.amax(-1)
    n15 = torch.full_like(hi, 15)   # a tensor: torch on a GPU multiplies by the rounded reciprocal of a number
    scale = torch.where(fine, hi / n15 - lo / n15, torch.nan).to(x.dtype)
    bias = torch.where(fine, lo, torch.nan).to(x.dtype)
    s = scale.float()[..., None]
    n = torch.where(s > 0, torch.round((g - bias.float()[..., None]) / s), torch.zeros_like(g)).nan_to_num(0).clamp(0, 15)
    n = n.to(torch.int64).flatten(-2).unflatten(-1, (-1, 8))
    words = (n << (4 * torch.arange(8, device=x.device))).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32), scale, bias


def values(codes, scales, biases, dtype=torch.float64) -> torch.Tensor:
    """[..., D] of what the codes stand for."""
    n = (codes.to(torch.int64)[..., None] >> (4 * torch.arange(8, device=codes.device))) & 15
    n = n.flatten(-2).unflatten(-1, (-1, GROUP)).to(dtype)
    return (n * scales.to(dtype)[..., None] + biases.to(dtype)[..., None]).flatten(-2)


def sdpa(q, k_cache, v_cache, scale, lengths, mask=None, max_length=None):
    """float64 [B, Hq, T, D]; hidden positions are left out of the sums, not multiplied by zero."""
    B, Hq, T, D = q.shape
    cap = k_cache[0].shape[2]
    Hk = k_cache[0].shape[1]
    n_max = cap if max_length is None else max_length
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=q.device)
    if mask is not None:
        mask = mask.expand(B, Hq, T, n_max)
    for b in range(B):
        n = int(lengths[b])
        for h in range(Hk):
            k, v = (values(*[p[b, h] for p in c]) for c in (k_cache, v_cache))
            for t in range(T):
                top = min(n, n_max, n - T + t + 1)
                if top <= 0:
                    continue
                for hq in range(h * (Hq // Hk), (h + 1) * (Hq // Hk)):
                    x = k[:top] @ q[b, hq, t].double() * scale
                    keep = torch.ones(top, dtype=torch.bool, device=q.device)
                    if mask is not None:
                        m = mask[b, hq, t, :top]
                        if m.dtype == torch.bool:
                            keep = m
                        else:
                            keep = m != -math.inf
                            x = x + m.double()
                    if bool(keep.any()):
                        out[b, hq, t] = torch.softmax(x[keep], 0) @ v[:top][keep]
    return out
