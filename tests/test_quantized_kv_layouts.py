"""Which caches may be written, and how a write that was not carried out is reported."""
import pytest
import torch

from dflash_mlx_b200 import _lib, quantized_kv as qkv


def written(*arrays):
    return _lib.native().check_cache(*arrays, True)


def test_caches_that_would_be_written_twice():
    B, Hk, cap, D = 2, 3, 32, 128
    k, v = qkv.allocate(B, Hk, cap, D, device="cpu")
    written(*k, *v)
    whole = [torch.zeros(2, B, Hk, cap, n, dtype=dt) for n, dt in ((D // 8, torch.int32), (D // 64, torch.bfloat16), (D // 64, torch.bfloat16))]
    written(*[p[0] for p in whole], *[p[1] for p in whole])                      # both sides in one allocation
    mixed = [torch.zeros(B, 2, Hk, cap, p.shape[-1], dtype=p.dtype) for p in whole]
    written(*[p[:, 0] for p in mixed], *[p[:, 1] for p in mixed])                # side by side in every sequence
    turned = [torch.zeros(Hk, B, cap, p.shape[-1], dtype=p.dtype).transpose(0, 1) for p in whole]
    written(*turned, *v)
    written(*[p[:, 1:, 8:24] for p in k], *[p[:, 1:, 8:24] for p in v])          # a slice
    one = [p[:1].expand(1, Hk, cap, -1) for p in k]
    written(*one, *[p[:1] for p in v])
    # the same sequence, head or side twice, and blocks that overlap
    for bad in ([p[:1].expand(B, -1, -1, -1) for p in k], [p[:, :1].expand(-1, Hk, -1, -1) for p in k],
                [p.as_strided(p.shape, (Hk * cap * p.shape[-1], cap // 2 * p.shape[-1], p.shape[-1], 1)) for p in k],
                [p.as_strided(p.shape, (cap * p.shape[-1], cap * p.shape[-1], p.shape[-1], 1)) for p in k],
                [k[0], k[1], v[2].as_strided(v[2].shape, (4 * cap, 2 * cap, 2, 1))]):
        with pytest.raises(ValueError, match="repeat or overlap"):
            written(*bad, *v)
        _lib.native().check_cache(*bad, *v)                                       # to be read they are fine
    for bad in ((*k, *k), (k[0], k[1], k[1], *v), (*k, v[0], k[1], v[2])):
        with pytest.raises(ValueError, match="one another"):
            written(*bad)


@pytest.mark.parametrize("code,text", [(61 | (5 << 8), "capacity"), (62 | (3 << 8), "wait"), (31, "refused")])
def test_a_device_error_is_raised(code, text, monkeypatch):
    class Library:
        def dflash_device_error(self, device):
            assert device == 3
            return words.pop()

    words = [0, code]
    monkeypatch.setattr(_lib, "lib", Library)
    with pytest.raises(_lib.DFlashError, match=f"step 7: device error word {code & 0xFF} .detail {code >> 8}.*{text}"):
        qkv.check_device_error("cuda:3", "step 7")
    qkv.check_device_error("cuda:3", "step 8")            # nothing since
