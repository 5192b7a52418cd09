"""Log-probabilities of given tokens, with the entropy and the most likely alternatives of every row of logits: what a server
reports beside the greedy token, and what accepting drafted tokens by probability starts from (the greedy counterpart is
``greedy_tokens_with_mask``, dflash_mlx/runtime.py:90-98).  One launch of libdflash_b200 per call; no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # float32 [...]: log p of the given token
    entropy: torch.Tensor         # float32 [...]: -sum p log p, in nats
    top_logprobs: torch.Tensor    # float32 [..., top_k], highest first
    top_ids: torch.Tensor         # int32 [..., top_k], ties to the lower id


def token_logprobs(logits, tokens, *, top_k: int = 0, temperature: float = 1.0,
                   suppress: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """``logits`` ``[..., V]`` (bf16, fp16 or fp32); ``tokens`` ``[...]`` (int32 or int64); p = softmax(logits / temperature),
    ``temperature`` from 1e-30 to 1e38.

    ``top_k`` (0..min(32, V)) alternatives per row.  ``suppress`` (bool ``[V]``): those tokens have probability 0.  A token
    outside ``[0, V)`` has the log-probability NaN.  A row with nothing but ``-inf`` yields ``-inf`` and the entropy 0; a row
    that holds a NaN or ``+inf`` yields NaN.  Rows are read in place when the last dimension is contiguous and the others
    collapse to one stride.
    """
    return TokenLogprobs(*(_lib._native or _lib.native()).token_logprobs(logits, tokens, top_k, temperature, suppress))
