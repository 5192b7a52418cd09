"""Token log-probabilities without a GPU: what the entry points refuse."""
import ctypes

import pytest
import torch

from dflash_mlx_b200 import _lib, logprobs


def test_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        logprobs.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int32))


def test_c_entry_refuses_before_any_launch():
    vp, i32 = ctypes.c_void_p, ctypes.c_int
    _lib.declare("dflash_token_logprobs", i32, [vp, ctypes.c_longlong, vp, vp, ctypes.c_float] + [vp] * 4 + [i32] * 4 + [vp])
    lib = _lib.lib()

    def call(x=0x1000, ld=100, tokens=0x1000, t=1.0, lp=0x1000, tops=0x1000, ids=0x1000, R=1, V=100, k=4, dtype=0):
        return lib.dflash_token_logprobs(x, ld, tokens, None, t, lp, None, tops, ids, R, V, k, dtype, None)
    assert call(R=0) == 0
    assert call(R=-1) == -2 and call(V=0) == -2 and call(ld=99) == -2
    assert call(k=33) == -2 and call(k=-1) == -2 and call(V=3, ld=3, k=4) == -2
    for t in (0.0, -1.0, float("inf"), float("nan")):
        assert call(t=t) == -1
    assert call(x=0) == -1 and call(tokens=0) == -1 and call(lp=0) == -1 and call(tops=0) == -1 and call(ids=0) == -1
    assert call(x=0x1001) == -3 and call(x=0x1002, dtype=2) == -3
    assert call(dtype=7) == -1
