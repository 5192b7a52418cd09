"""Which of the two attention kernels sizes take, and over how many key ranges."""
import ctypes

from dflash_mlx_b200 import _lib

i32 = ctypes.c_int


def plan(B, Hq, Hk, T, max_length, num_splits=0):
    """(whether the tcgen05 kernel runs, key ranges)"""
    _lib.declare("dflash_kv4_sdpa_plan", i32, [i32] * 6 + [ctypes.POINTER(i32), i32])
    out = (i32 * 2)()
    assert _lib.lib().dflash_kv4_sdpa_plan(B, Hq, Hk, T, max_length, num_splits, out, 2) == 2
    return bool(out[0]), out[1]


def test_few_rows_never_and_many_rows_over_much_always():
    for n in (1, 100, 131072):
        assert not plan(4, 16, 1, 1, n)[0] and not plan(64, 32, 2, 1, n)[0]
        assert plan(1, 8, 1, 2048, n)[0]
    assert not plan(1, 24, 4, 16, 512)[0] and plan(1, 24, 4, 16, 8192)[0]
    # once a length sends them there, every longer one does
    for Hq, Hk, T in ((1, 1, 17), (12, 2, 4), (24, 4, 16), (8, 8, 40)):
        took = [plan(1, Hq, Hk, T, n)[0] for n in range(1, 30000, 97)]
        assert took[-1] and took == sorted(took)


def test_ranges_hold_at_least_128_keys():
    for n in (1, 127, 128, 129, 5000, 131072):
        for Hq, Hk, T in ((1, 1, 1), (8, 1, 1), (24, 4, 16), (24, 4, 500)):
            most = (n + 127) // 128
            assert 1 <= plan(1, Hq, Hk, T, n)[1] <= most
            for s in (1, 2, 1024):
                assert plan(1, Hq, Hk, T, n, s)[1] == min(s, most)


def test_refusals():
    plan(1, 1, 1, 1, 1)
    out = (i32 * 2)()
    for args in ((0, 1, 1, 1, 1, 0), (1, 3, 2, 1, 1, 0), (1, 1, 1, 0, 1, 0), (1, 1, 1, 1, 0, 0), (1, 1, 1, 1, 1, 1025), (1, 1, 1, 1, 1, -1),
                 (1, 2, 1, 600000, 1, 0)):
        assert _lib.lib().dflash_kv4_sdpa_plan(*args, out, 2) == -2, args
    assert _lib.lib().dflash_kv4_sdpa_plan(1, 1, 1, 1, 1, 0, out, 1) == -1
    assert _lib.lib().dflash_kv4_sdpa_plan(1, 1, 1, 1, 1, 0, None, 2) == -1
