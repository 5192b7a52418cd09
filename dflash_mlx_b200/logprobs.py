"""Log-probabilities of given tokens, with the entropy and the most likely alternatives of every row of logits: what a server
reports beside the greedy token, and what accepting drafted tokens by probability starts from (the greedy counterpart is
``greedy_tokens_with_mask``, dflash_mlx/runtime.py:90-98).  One launch of libdflash_b200 per call; no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib

_c = ctypes
_vp, _i32, _f32 = _c.c_void_p, _c.c_int, _c.c_float
_declared = False
MAX_TOP_K = 32


def _ensure_declared():
    global _declared
    if _declared:
        return
    _lib.declare("dflash_token_logprobs", _i32, [_vp, _c.c_longlong, _vp, _vp, _f32] + [_vp] * 4 + [_i32] * 4 + [_vp])
    _declared = True


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # float32 [...]: log p of the given token
    entropy: torch.Tensor         # float32 [...]: -sum p log p, in nats
    top_logprobs: torch.Tensor    # float32 [..., top_k], highest first
    top_ids: torch.Tensor         # int32 [..., top_k], ties to the lower id


def token_logprobs(logits, tokens, *, top_k: int = 0, temperature: float = 1.0,
                   suppress: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """``logits`` ``[..., V]`` (bf16, fp16 or fp32); ``tokens`` ``[...]`` (int32 or int64); p = softmax(logits / temperature).

    ``top_k`` (0..min(32, V)) alternatives per row.  ``suppress`` (bool ``[V]``): those tokens have probability 0.  A token
    outside ``[0, V)`` has the log-probability NaN.  A row with nothing but ``-inf`` yields ``-inf`` and the entropy 0; a row
    that holds a NaN or ``+inf`` yields NaN.  Rows are read in place when the last dimension is contiguous and the others
    collapse to one stride.
    """
    _ensure_declared()
    dev = _lib.require_cuda(logits, tokens, suppress)
    if logits.ndim < 1:
        raise ValueError("logits must be [..., V]")
    V = logits.shape[-1]
    rows = tuple(logits.shape[:-1])
    if tuple(tokens.shape) != rows:
        raise ValueError(f"tokens must have logits' leading shape {rows}, got {tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    code = _lib.dtype_code(logits.dtype)
    top_k = int(top_k)
    if V < 1 or not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"top_k={top_k} outside 0..min({MAX_TOP_K}, V={V})")
    temperature = float(temperature)
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if suppress is not None:
        if suppress.dtype != torch.bool or tuple(suppress.shape) != (V,):
            raise ValueError(f"suppress must be a bool tensor [V] = {(V,)}")
        suppress = suppress.contiguous().view(torch.uint8)
    if logits.ndim == 2 and logits.stride(1) == 1 and logits.stride(0) >= V:
        x = logits
    else:
        x = logits.reshape(-1, V) if logits.ndim > 1 else logits.view(1, V)
        if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < V):
            x = x.contiguous()
    R = x.shape[0]
    ids = tokens.reshape(-1)
    if ids.dtype == torch.int64:      # ids beyond int32 must not wrap into the vocabulary
        ids = ids.clamp(-1, V).to(torch.int32)
    ids = ids.contiguous()
    out = torch.empty(2, R, dtype=torch.float32, device=dev)
    tops = torch.empty(R, top_k, dtype=torch.float32, device=dev)
    top_ids = torch.empty(R, top_k, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        st = _lib.lib().dflash_token_logprobs(
            x.data_ptr(), x.stride(0) if R > 1 else V, ids.data_ptr(), _lib.ptr(suppress), temperature, out[0].data_ptr(),
            out[1].data_ptr(), tops.data_ptr() if top_k else 0, top_ids.data_ptr() if top_k else 0, R, V, top_k, code,
            _lib.stream_ptr(dev))
    _lib.check(st, "dflash_token_logprobs")
    return TokenLogprobs(out[0].view(rows), out[1].view(rows), tops.view(*rows, top_k), top_ids.view(*rows, top_k))
