"""The 4-bit KV cache: quantising keys and values as they are written, reading them back, and attention over the codes.

The reference hands its attention whatever cache mlx-lm made, a quantised one among them (dflash_mlx/runtime.py:671-676); its
own 16-row attention takes dense keys and values only (dflash_mlx/kernels.py:658-761).  Here the cache stays in 4 bits: one side
(keys or values) is a tuple ``(codes, scales, biases)`` in the layout of the packed weights - ``codes`` int32
``[B, Hk, capacity, D/8]`` (nibble i of word j is channel 8j+i), ``scales`` and ``biases`` ``[B, Hk, capacity, D/64]`` in the
model's type; a channel stands for ``code * scale + bias``.  All compute is in libdflash_b200 (sm_100a).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

GROUP = 64


class QuantizedKV(NamedTuple):
    """One side of a cache."""
    codes: torch.Tensor
    scales: torch.Tensor
    biases: torch.Tensor


def allocate(batch: int, kv_heads: int, capacity: int, head_dim: int, *, dtype=torch.bfloat16,
             device="cuda") -> Tuple[QuantizedKV, QuantizedKV]:
    """Zero-filled key and value sides of a cache."""
    if head_dim not in (128, 256):
        raise ValueError(f"D={head_dim} is not supported (need 128 or 256)")
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported dtype {dtype}")

    def side():
        z = lambda n, dt: torch.zeros(batch, kv_heads, capacity, n, dtype=dt, device=device)  # noqa: E731
        return QuantizedKV(z(head_dim // 8, torch.int32), z(head_dim // GROUP, dtype), z(head_dim // GROUP, dtype))
    return side(), side()


def quantized_kv_write(keys, values, k_cache, v_cache, offsets, *, counts: Optional[torch.Tensor] = None) -> None:
    """Quantises ``keys`` / ``values`` ``[B, Hk, T, D]`` into positions ``offsets[b] + t`` of the cache, in place.

    ``offsets`` int32 ``[B]`` on the device (a captured graph replays at any position); ``counts`` int32 ``[B]``: only the first
    ``counts[b]`` rows of sequence ``b`` are stored (a padded batch).  Per 64 channels: scale = max/15 - min/15 and bias = min in
    the cache's type, code = round((x - bias) / scale) in 0..15 (the layout of ``mx.quantize``, not its codes).  A group that
    holds a NaN or infinity reads back as NaN.  Rows outside the capacity are not stored and set the device error word, which
    ``check_device_error`` raises.  A cache whose sequences, heads or sides share memory is refused.
    """
    (_lib._native or _lib.native()).kv4_write(keys, values, *k_cache, *v_cache, offsets, counts)


def quantized_kv_read(k_cache, v_cache, start: Union[int, torch.Tensor], length: int):
    """Dense keys and values ``[B, Hk, length, D]`` of positions ``start .. start + length - 1`` in the cache's type.  ``start``
    is an int, or an int32 tensor ``[B]`` on the device; positions outside the capacity read as zero."""
    return (_lib._native or _lib.native()).kv4_read(*k_cache, *v_cache, start, length)


def quantized_kv_sdpa(queries, k_cache, v_cache, scale: float, lengths: Union[int, torch.Tensor],
                      mask: Optional[torch.Tensor] = None, *, max_length: Optional[int] = None, num_splits: int = 0):
    """Softmax attention of ``queries`` ``[B, Hq, T, D]``, T >= 1 (a token, a verify block, a chunk of a prompt), over the cache.

    ``lengths``: positions every sequence holds, the T queries' own among them - an int, or an int32 tensor ``[B]`` read on
    the device.  Row ``t`` of sequence ``b`` sees position ``n`` iff ``n <= lengths[b] - T + t`` (and ``n < lengths[b]``).
    ``max_length`` (default: the int, or the capacity) bounds the lengths: positions from it on are not read.  ``mask`` is a bool
    (False hides) or additive (the queries' dtype or float32; -inf hides) tensor that broadcasts to ``[B, Hq, T, max_length]``;
    it is read in place.  Returns ``[B, Hq, T, D]``; a row that sees nothing is zero.  Hidden keys and values change no bit of a
    row, whatever they hold; a visible value with a scale or bias that is not finite makes its row NaN.  ``num_splits`` fixes the
    number of key ranges (0: from the SM count).
    """
    return (_lib._native or _lib.native()).kv4_sdpa(queries, *k_cache, *v_cache, scale, lengths, mask, max_length, num_splits)


def check_device_error(device, where: str) -> None:
    """Reads (and clears) the status word of ``device`` after a synchronisation and raises ``DFlashError`` where a call was not carried
    out: rows of a write outside the capacity (code 61), a wait inside the attention that ran out (62)."""
    index = torch.device(device).index
    code = _lib.lib().dflash_device_error(torch.cuda.current_device() if index is None else index)
    if code != 0:
        what = {61: "rows outside the cache's capacity were not written",
                62: "an attention kernel abandoned a bounded wait; the results of the last calls are not valid"}
        raise _lib.DFlashError(f"{where}: device error word {code & 0xFF} (detail {code >> 8}): "
                               + what.get(code & 0xFF, "a kernel refused its operands or abandoned a bounded wait"))


class QuantizedKVCache:
    """One attention layer's cache in 4 bits, with the positions of its sequences on the device.

    ``update`` quantises a block of new keys and values behind what the cache holds, ``attend`` lets the same block's queries
    attend, ``commit`` moves the positions on - by the whole block after a prompt chunk or a token, by the accepted length after
    a verify block, which rolls the rest back (rows behind the position are overwritten by the next block).
    """

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, *, dtype=torch.bfloat16, device="cuda"):
        self.keys, self.values = allocate(batch, kv_heads, capacity, head_dim, dtype=dtype, device=device)
        self.capacity = capacity
        self.offsets = torch.zeros(batch, dtype=torch.int32, device=device)

    def update(self, keys, values, counts: Optional[torch.Tensor] = None) -> None:
        quantized_kv_write(keys, values, self.keys, self.values, self.offsets, counts=counts)

    def attend(self, queries, scale: float, mask: Optional[torch.Tensor] = None, *, max_length: Optional[int] = None):
        """Attention of the block written last: its rows see the positions before it and, causally, each other."""
        return quantized_kv_sdpa(queries, self.keys, self.values, scale, self.offsets + queries.shape[2], mask, max_length=max_length)

    def commit(self, accepted: Union[int, torch.Tensor]) -> None:
        """Positions += accepted (an int, or int32 ``[B]`` on the device)."""
        self.offsets += accepted

    def check_device_error(self, where: str) -> None:
        """Reads (and clears) the device's status word - a row that ``update`` could not place inside the capacity, a kernel that
        gave up on a bounded wait - and raises.  Synchronises the device: called where the host synchronises anyway."""
        check_device_error(self.offsets.device, where)

    def read(self, start: Union[int, torch.Tensor], length: int):
        return quantized_kv_read(self.keys, self.values, start, length)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (*self.keys, *self.values))
