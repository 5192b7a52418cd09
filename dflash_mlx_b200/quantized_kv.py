"""The 4-bit KV cache: quantising keys and values as they are written, reading them back, and attention over the codes.

The reference hands its attention whatever cache mlx-lm made, a quantised one among them (dflash_mlx/runtime.py:671-676); its
own 16-row attention takes dense keys and values only (dflash_mlx/kernels.py:658-761).  Here the cache stays in 4 bits: one side
(keys or values) is a tuple ``(codes, scales, biases)`` in the layout of the packed weights - ``codes`` int32
``[B, Hk, capacity, D/8]`` (nibble i of word j is channel 8j+i), ``scales`` and ``biases`` ``[B, Hk, capacity, D/64]`` in the
model's type; a channel stands for ``code * scale + bias``.  All compute is in libdflash_b200 (sm_100a).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

_c = ctypes
_vp, _i32, _f32, _ll = _c.c_void_p, _c.c_int, _c.c_float, _c.c_longlong
_declared = False
GROUP = 64


class _Cache(_c.Structure):
    """``dflash_kv4_cache`` of the C ABI."""
    _fields_ = [("codes", _vp), ("scales", _vp), ("biases", _vp), ("codes_b", _ll), ("codes_h", _ll), ("scales_b", _ll),
                ("scales_h", _ll), ("biases_b", _ll), ("biases_h", _ll)]


class QuantizedKV(NamedTuple):
    """One side of a cache."""
    codes: torch.Tensor
    scales: torch.Tensor
    biases: torch.Tensor


def _ensure_declared():
    global _declared
    if _declared:
        return
    cp, sp = _c.POINTER(_Cache), _c.POINTER(_ll)
    _lib.declare("dflash_kv4_write", _i32, [_vp, sp, _vp, sp, cp, cp, _vp, _vp] + [_i32] * 6 + [_vp])
    _lib.declare("dflash_kv4_read", _i32, [cp, cp, _vp, _vp, _vp] + [_i32] * 7 + [_vp])
    _lib.declare("dflash_kv4_sdpa_workspace_bytes", _c.c_size_t, [_i32] * 7)
    _lib.declare("dflash_kv4_sdpa", _i32, [_vp, sp, cp, cp, _vp, _i32, sp, _vp, _vp] + [_i32] * 7 +
                 [_f32, _i32, _i32, _vp, _c.c_size_t, _vp])
    _declared = True


def _side(cache, name: str):
    """(struct, (B, Hk, capacity, D, dtype)) of one side of a cache; refuses what the kernels cannot address in place."""
    codes, scales, biases = cache
    if codes.ndim != 4 or codes.dtype not in (torch.int32, torch.uint32):
        raise ValueError(f"{name} codes must be int32 [B, Hk, capacity, D/8], got {codes.dtype} {tuple(codes.shape)}")
    B, Hk, cap, words = codes.shape
    D = words * 8
    if D not in (128, 256):
        raise ValueError(f"{name}: D={D} is not supported (need 128 or 256)")
    for what, t in (("scales", scales), ("biases", biases)):
        if tuple(t.shape) != (B, Hk, cap, D // GROUP):
            raise ValueError(f"{name} {what} must be [B, Hk, capacity, D/{GROUP}] = {(B, Hk, cap, D // GROUP)}, got {tuple(t.shape)}")
    if scales.dtype not in (torch.bfloat16, torch.float16) or biases.dtype != scales.dtype:
        raise ValueError(f"{name} scales and biases must share bfloat16 or float16")
    for t in (codes, scales, biases):
        if t.stride(3) != 1 or t.stride(2) != t.shape[3]:
            raise ValueError(f"{name}: the positions of a cache must be contiguous")
    s = _Cache(codes.data_ptr(), scales.data_ptr(), biases.data_ptr(), codes.stride(0), codes.stride(1), scales.stride(0),
               scales.stride(1), biases.stride(0), biases.stride(1))
    return s, (B, Hk, cap, D, scales.dtype)


def _sides(k_cache, v_cache):
    k, kd = _side(k_cache, "key cache")
    v, vd = _side(v_cache, "value cache")
    if kd != vd:
        raise ValueError(f"the key cache {kd} and the value cache {vd} differ")
    return k, v, kd


def _rows(t: torch.Tensor):
    """(tensor, strides of its first three dimensions) with contiguous 16-byte aligned rows; anything else is copied."""
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in range(3)):
        t = t.contiguous()
    # the stride of a dimension of one element is never used
    return t, (_ll * 3)(*[t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)])


def _per_sequence(t, B: int, name: str):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [B] = {(B,)}")
    return t


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
    the cache's type, code = round((x - bias) / scale) in 0..15.  A group that holds a NaN or infinity reads back as NaN.  Rows
    outside the capacity are not stored and set the device error word (``dflash_device_error``, code 61).
    """
    _ensure_declared()
    dev = _lib.require_cuda(keys, values, *k_cache, *v_cache, offsets, counts)
    k, v, (B, Hk, cap, D, dt) = _sides(k_cache, v_cache)
    if keys.ndim != 4 or tuple(keys.shape) != tuple(values.shape) or tuple(keys.shape[:2]) != (B, Hk) or keys.shape[3] != D:
        raise ValueError(f"keys and values must be [B, Hk, T, D] = {(B, Hk, 'T', D)}, got {tuple(keys.shape)} and {tuple(values.shape)}")
    if keys.dtype != dt or values.dtype != dt:
        raise ValueError(f"keys and values must have the cache's dtype {dt}")
    _per_sequence(offsets, B, "offsets")
    if counts is not None:
        _per_sequence(counts, B, "counts")
    keys, ks = _rows(keys)
    values, vs = _rows(values)
    with torch.cuda.device(dev):
        st = _lib.lib().dflash_kv4_write(keys.data_ptr(), ks, values.data_ptr(), vs, _c.byref(k), _c.byref(v), offsets.data_ptr(),
                                         _lib.ptr(counts), B, Hk, keys.shape[2], D, cap, _lib.dtype_code(dt), _lib.stream_ptr(dev))
    _lib.check(st, "dflash_kv4_write")


def quantized_kv_read(k_cache, v_cache, start: Union[int, torch.Tensor], length: int):
    """Dense keys and values ``[B, Hk, length, D]`` of positions ``start .. start + length - 1`` in the cache's type.  ``start``
    is an int, or an int32 tensor ``[B]`` on the device; positions outside the capacity read as zero."""
    _ensure_declared()
    starts = start if isinstance(start, torch.Tensor) else None
    dev = _lib.require_cuda(*k_cache, *v_cache, starts)
    k, v, (B, Hk, cap, D, dt) = _sides(k_cache, v_cache)
    length = int(length)
    if length < 0:
        raise ValueError(f"length={length} is negative")
    first = 0
    if starts is not None:
        _per_sequence(starts, B, "start")
    else:
        first = int(start)
        if not -2 ** 31 <= first < 2 ** 31:
            raise ValueError(f"start={first} does not fit 32 bits")
    out = [torch.empty(B, Hk, length, D, dtype=dt, device=dev) for _ in range(2)]
    with torch.cuda.device(dev):
        st = _lib.lib().dflash_kv4_read(_c.byref(k), _c.byref(v), out[0].data_ptr(), out[1].data_ptr(), _lib.ptr(starts), first, B, Hk,
                                        length, D, cap, _lib.dtype_code(dt), _lib.stream_ptr(dev))
    _lib.check(st, "dflash_kv4_read")
    return out[0], out[1]


def quantized_kv_sdpa(queries, k_cache, v_cache, scale: float, lengths: Union[int, torch.Tensor],
                      mask: Optional[torch.Tensor] = None, *, max_length: Optional[int] = None, num_splits: int = 0):
    """Softmax attention of ``queries`` ``[B, Hq, T, D]``, T >= 1 (a token, a verify block, a chunk of a prompt), over the cache.

    ``lengths``: positions every sequence holds, the T queries' own among them - an int, or an int32 tensor ``[B]`` read on
    the device.  Row ``t`` of sequence ``b`` sees position ``n`` iff ``n <= lengths[b] - T + t`` (and ``n < lengths[b]``).
    ``max_length`` (default: the int, or the capacity) bounds the lengths: positions from it on are not read.  ``mask`` is a bool
    (False hides) or additive (the queries' dtype or float32; -inf hides) tensor that broadcasts to ``[B, Hq, T, max_length]``;
    it is read in place.  Returns ``[B, Hq, T, D]``; a row that sees nothing is zero.  Hidden keys and values never reach a row,
    whatever they hold; a visible value with a non-finite scale or bias makes its row NaN.  ``num_splits`` fixes the number of
    key ranges (0: from the SM count).
    """
    _ensure_declared()
    on_device = isinstance(lengths, torch.Tensor)
    dev = _lib.require_cuda(queries, *k_cache, *v_cache, lengths if on_device else None, mask)
    k, v, (B, Hk, cap, D, dt) = _sides(k_cache, v_cache)
    if queries.ndim != 4 or queries.shape[0] != B or queries.shape[3] != D or queries.shape[1] < 1 or queries.shape[1] % Hk:
        raise ValueError(f"queries must be [B, Hq, T, D] = {(B, f'n*{Hk}', 'T', D)}, got {tuple(queries.shape)}")
    if queries.dtype != dt:
        raise ValueError(f"queries must have the cache's dtype {dt}")
    Hq, T = queries.shape[1], queries.shape[2]
    if on_device:
        _per_sequence(lengths, B, "lengths")
        n_max = cap if max_length is None else int(max_length)
    else:
        n_max = int(lengths)
        if max_length is not None and int(max_length) != n_max:
            raise ValueError("max_length goes with lengths on the device")
    if not 0 <= n_max <= cap:
        raise ValueError(f"length {n_max} outside 0..{cap}")
    kind, ms = 0, (_ll * 4)()
    if mask is not None:
        if mask.dtype == torch.bool:
            kind = 1
        elif mask.dtype == dt:
            kind = 2
        elif mask.dtype == torch.float32:
            kind = 3
        else:
            raise ValueError(f"mask must be bool, {dt} or float32, got {mask.dtype}")
        mask = mask.expand(B, Hq, T, n_max)
        ms = (_ll * 4)(*mask.stride())
    queries, qs = _rows(queries)
    out = torch.empty(B, Hq, T, D, dtype=dt, device=dev)
    if out.numel() == 0:
        return out
    if n_max == 0:
        return out.zero_()
    lib = _lib.lib()
    with torch.cuda.device(dev):
        need = lib.dflash_kv4_sdpa_workspace_bytes(B, Hq, Hk, T, D, n_max, num_splits)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        st = lib.dflash_kv4_sdpa(queries.data_ptr(), qs, _c.byref(k), _c.byref(v), _lib.ptr(mask), kind, ms, out.data_ptr(),
                                 lengths.data_ptr() if on_device else 0, B, Hq, Hk, T, D, cap, n_max, float(scale),
                                 _lib.dtype_code(dt), num_splits, _lib.ptr(ws), need, _lib.stream_ptr(dev))
    _lib.check(st, "dflash_kv4_sdpa")
    return out


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

    def read(self, start: Union[int, torch.Tensor], length: int):
        return quantized_kv_read(self.keys, self.values, start, length)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (*self.keys, *self.values))
