"""The 4-bit KV cache's arguments at unusual places in memory: what is copied, what is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import _lib, quantized_kv as qkv  # noqa: E402
from oracle import quantized_kv as ref  # noqa: E402
from tests.test_quantized_kv_gpu import ints, make_cache, no_device_error, states  # noqa: E402, F401

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("off", [1, 3, 4, 8])
def test_contiguous_rows_off_their_boundary(off, dtype):
    """Contiguous tensors that start between two 16-byte boundaries are copied like any others that the kernels cannot read."""
    B, Hk, T, D, n = 2, 2, 5, 128, 40
    k_cache, v_cache = make_cache(B, Hk, n, D, dtype)
    flat = states((off + B * Hk * T * D,), dtype, 1)
    x = flat[off:].view(B, Hk, T, D)
    assert x.is_contiguous()
    qkv.quantized_kv_write(x, x, k_cache, v_cache, ints(3, 7))
    want = ref.quantise(x)
    for c in (k_cache, v_cache):
        for got, part in zip(c, want):
            assert torch.equal(got[0, :, 3:8], part[0]) and torch.equal(got[1, :, 7:12], part[1])
    assert torch.equal(qkv.quantized_kv_sdpa(x, k_cache, v_cache, 0.1, n), qkv.quantized_kv_sdpa(x.clone(), k_cache, v_cache, 0.1, n))


def test_rows_that_did_not_fit_are_reported():
    cache = qkv.QuantizedKVCache(2, 1, 20, 128)
    x = states((2, 1, 8, 128), torch.bfloat16, 1)
    cache.update(x, x)
    cache.check_device_error("prompt")
    cache.commit(ints(8, 15))
    before = [p.clone() for p in cache.values]
    cache.update(x, x)
    with pytest.raises(_lib.DFlashError, match="second block.*61.*capacity"):
        cache.check_device_error("second block")
    cache.check_device_error("after")
    for got, old, part in zip(cache.values, before, ref.quantise(x)):
        assert torch.equal(got[0, :, 8:16], part[0]) and torch.equal(got[1, :, 15:], part[1, :, :5]) and torch.equal(got[1, :, :15], old[1, :, :15])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value_as_a_group_s_maximum_and_minimum(dtype):
    """Scales, biases and codes to the last bit, whatever a group's range is."""
    x = torch.arange(-(1 << 15), 1 << 15, device=DEV, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.isfinite()]
    rows = torch.zeros(1, 1, len(x), 128, dtype=dtype, device=DEV)
    rows[0, 0, :, 7] = x                                  # from zero to x, or from x to zero
    rows[0, 0, :, 64:] = x.flip(0)[:, None] * torch.linspace(-1, 1, 64, device=DEV).to(dtype)
    rows[0, 0, :, 64] = x.roll(977)
    rows = rows.nan_to_num(0, 0, 0)
    k_cache, v_cache = qkv.allocate(1, 1, len(x), 128, dtype=dtype)
    qkv.quantized_kv_write(rows, rows, k_cache, v_cache, ints(0))
    for c in (k_cache, v_cache):
        for got, want in zip(c, ref.quantise(rows)):
            assert torch.equal(got, want)
