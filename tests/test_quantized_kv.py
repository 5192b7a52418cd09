"""The 4-bit KV cache without a GPU: the quantisation's definition, and what the entry points refuse."""
import ctypes

import pytest
import torch

from dflash_mlx_b200 import _lib, quantized_kv as qkv
from oracle import quantized_kv as ref
from oracle import qmm as oq


def test_codes_are_the_packed_weights_layout():
    x = torch.randn(2, 3, 5, 128).to(torch.bfloat16)
    codes, scales, biases = ref.quantise(x)
    want = oq.dequantize(codes.reshape(-1, 16), scales.reshape(-1, 2), biases.reshape(-1, 2), 64).reshape(x.shape)
    assert torch.equal(ref.values(codes, scales, biases, torch.float32), want.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantisation_error_is_half_a_step(dtype):
    x = (3 * torch.randn(64, 256) + 1).to(dtype)
    codes, scales, biases = ref.quantise(x)
    got = ref.values(codes, scales, biases)
    # half a step, and the top code is off by what rounding the scale moves it: 15 * scale * eps / 2
    step = scales.double().repeat_interleave(64, -1)
    assert bool(((got - x.double()).abs() <= step * (0.5 + 15 * torch.finfo(dtype).eps / 2 + 1e-5)).all())


def test_refuses_cpu_tensors():
    k, v = qkv.allocate(1, 2, 64, 128, device="cpu")
    x = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        qkv.quantized_kv_write(x, x, k, v, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        qkv.quantized_kv_read(k, v, 0, 4)
    with pytest.raises(ValueError, match="CUDA"):
        qkv.quantized_kv_sdpa(x, k, v, 1.0, 4)


def test_refuses_bad_caches():
    k, v = qkv.allocate(1, 2, 64, 128, device="cpu")
    check = lambda one, other=v: _lib.native().check_cache(*one, *other)  # noqa: E731
    check(k)
    with pytest.raises(ValueError, match="D=64"):
        check((k.codes[..., :8], k.scales, k.biases))
    with pytest.raises(ValueError, match="int32"):
        check((k.codes.long(), k.scales, k.biases))
    with pytest.raises(ValueError, match="scales must be"):
        check((k.codes, k.scales[..., :1], k.biases))
    with pytest.raises(ValueError, match="share"):
        check((k.codes, k.scales, k.biases.half()))
    with pytest.raises(ValueError, match="share"):
        check((k.codes, k.scales.float(), k.biases.float()))
    with pytest.raises(ValueError, match="contiguous"):
        check((k.codes[:, :, ::2], k.scales[:, :, ::2], k.biases[:, :, ::2]))
    with pytest.raises(ValueError, match="differ"):
        check(k, qkv.allocate(1, 2, 32, 128, device="cpu")[1])
    with pytest.raises(ValueError, match="D=96"):
        qkv.allocate(1, 1, 8, 96, device="cpu")
    with pytest.raises(ValueError, match="dtype"):
        qkv.allocate(1, 1, 8, 128, dtype=torch.float32, device="cpu")


_ll, _vp, _i32 = ctypes.c_longlong, ctypes.c_void_p, ctypes.c_int


class _Cache(ctypes.Structure):
    """``dflash_kv4_cache`` of the C ABI."""
    _fields_ = [("codes", _vp), ("scales", _vp), ("biases", _vp), ("codes_b", _ll), ("codes_h", _ll), ("scales_b", _ll),
                ("scales_h", _ll), ("biases_b", _ll), ("biases_h", _ll)]


def _declare():
    cp, sp = ctypes.POINTER(_Cache), ctypes.POINTER(_ll)
    _lib.declare("dflash_kv4_write", _i32, [_vp, sp, _vp, sp, cp, cp, _vp, _vp] + [_i32] * 6 + [_vp])
    _lib.declare("dflash_kv4_read", _i32, [cp, cp, _vp, _vp, _vp] + [_i32] * 7 + [_vp])
    _lib.declare("dflash_kv4_sdpa_workspace_bytes", ctypes.c_size_t, [_i32] * 7)
    _lib.declare("dflash_kv4_sdpa", _i32, [_vp, sp, cp, cp, _vp, _i32, sp, _vp, _vp] + [_i32] * 7 +
                 [ctypes.c_float, _i32, _i32, _vp, ctypes.c_size_t, _vp])


def _cache_struct(base=0x1000, **kw):
    s = _Cache(base, base, base, 1024, 512, 128, 64, 128, 64)
    for name, value in kw.items():
        setattr(s, name, value)
    return s


def _write(lib, k, v, B=1, Hk=2, T=1, D=128, cap=32, dtype=0, keys=0x1000, strides=(256, 128, 128), offsets=0x1000):
    st = (ctypes.c_longlong * 3)(*strides)
    return lib.dflash_kv4_write(keys, st, keys, st, ctypes.byref(k), ctypes.byref(v), offsets, None, B, Hk, T, D, cap, dtype, None)


def test_c_entries_refuse_before_any_launch():
    _declare()
    lib = _lib.lib()
    ok = _cache_struct()
    assert _write(lib, ok, ok, T=0) == 0 and _write(lib, ok, ok, B=0) == 0      # nothing to do
    assert _write(lib, ok, ok, D=64) == -2
    assert _write(lib, ok, ok, Hk=0) == -2
    assert _write(lib, ok, ok, T=-1) == -2
    assert _write(lib, ok, ok, cap=0) == -2
    assert _write(lib, ok, ok, dtype=2) == -1
    assert _write(lib, ok, ok, keys=0) == -1
    assert _write(lib, ok, ok, offsets=0) == -1
    assert _write(lib, ok, ok, keys=0x1008) == -3
    assert _write(lib, ok, ok, strides=(256, 128, 132)) == -3
    assert _write(lib, _cache_struct(codes=0), ok) == -1
    assert _write(lib, _cache_struct(codes=0x1004), ok) == -3
    assert _write(lib, ok, _cache_struct(scales=0x1002)) == -3
    assert _write(lib, ok, _cache_struct(codes_h=514)) == -3
    st3, st4 = (ctypes.c_longlong * 3)(256, 128, 128), (ctypes.c_longlong * 4)()

    def sdpa(B=1, Hq=2, Hk=2, T=1, D=128, cap=32, n=32, dtype=0, mask=None, kind=0, q=0x1000, ws=None, ws_bytes=0, splits=0):
        return lib.dflash_kv4_sdpa(q, st3, ctypes.byref(ok), ctypes.byref(ok), mask, kind, st4, 0x1000, None, B, Hq, Hk, T, D, cap, n,
                                   1.0, dtype, splits, ws, ws_bytes, None)
    assert sdpa(Hq=3) == -2 and b"query heads" in lib.dflash_last_error_string()
    assert sdpa(n=33) == -2 and sdpa(n=-1) == -2
    assert sdpa(D=192) == -2
    assert sdpa(dtype=2) == -1
    assert sdpa(mask=0x1000) == -1 and sdpa(kind=1) == -1 and sdpa(mask=0x1000, kind=4) == -1
    assert sdpa(q=0) == -1 and sdpa(q=0x1002) == -3
    assert sdpa(B=70000) == -2
    assert sdpa(T=0) == 0
    assert sdpa(cap=4096, n=4096, splits=4) == -4          # no workspace
    need = lib.dflash_kv4_sdpa_workspace_bytes(1, 2, 2, 1, 128, 4096, 4)
    assert need > 0 and sdpa(cap=4096, n=4096, splits=4, ws=0x1000, ws_bytes=need - 1) == -4
    assert sdpa(cap=4096, n=4096, splits=4, ws=0x1008, ws_bytes=need) == -3
    assert lib.dflash_kv4_sdpa_workspace_bytes(1, 3, 2, 1, 128, 4096, 4) == 0
    assert lib.dflash_kv4_read(ctypes.byref(ok), ctypes.byref(ok), 0x1000, 0x1008, None, 0, 1, 2, 4, 128, 32, 0, None) == -3
    assert lib.dflash_kv4_read(ctypes.byref(ok), None, 0x1000, 0x1000, None, 0, 1, 2, 4, 128, 32, 0, None) == -1
    assert lib.dflash_kv4_read(ctypes.byref(ok), ctypes.byref(ok), None, None, None, 0, 1, 2, 4, 128, 32, 0, None) == -1
    assert lib.dflash_kv4_read(ctypes.byref(ok), ctypes.byref(ok), 0x1000, 0x1000, None, 0, 1, 2, 0, 128, 32, 0, None) == 0


def test_c_attention_refuses_splits_and_masks_it_cannot_address():
    _declare()
    lib = _lib.lib()
    ok = _cache_struct()
    st3, st4 = (ctypes.c_longlong * 3)(256, 128, 128), (ctypes.c_longlong * 4)()

    def sdpa(mask=None, kind=0, splits=0):
        return lib.dflash_kv4_sdpa(0x1000, st3, ctypes.byref(ok), ctypes.byref(ok), mask, kind, st4, 0x1000, None, 1, 2, 2, 1, 128, 1 << 20, 1 << 20,
                                   1.0, 0, splits, None, 0, None)
    assert sdpa(splits=-1) == -1 and sdpa(splits=1025) == -1 and b"num_splits" in lib.dflash_last_error_string()
    assert sdpa(splits=1024) == -4                         # the workspace is what it lacks
    for bad in (-1, 1025):
        assert lib.dflash_kv4_sdpa_workspace_bytes(1, 2, 2, 1, 128, 1 << 20, bad) == 0
    assert sdpa(mask=0x1001, kind=2) == -3 and sdpa(mask=0x1002, kind=3) == -3
    assert sdpa(mask=0x1001, kind=1, splits=4) == -4 and sdpa(mask=0x1002, kind=2, splits=4) == -4
