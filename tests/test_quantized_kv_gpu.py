"""The 4-bit KV cache on the GPU against the 64-bit oracle."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import _lib, logprobs, quantized_kv as qkv  # noqa: E402
from oracle import logprobs as ref_logprobs, quantized_kv as ref  # noqa: E402

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def states(shape, dtype, seed, spread=1.0):
    return (spread * torch.randn(shape, generator=gen(seed), device=DEV) + 0.3).to(dtype)


def make_cache(B, Hk, cap, D, dtype, seed=0, spread=1.0):
    return tuple(qkv.QuantizedKV(*ref.quantise(states((B, Hk, cap, D), dtype, seed + i, spread))) for i in range(2))


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# A row's error against its norm.  Rounding the output: eps / 2 (2^-8, 2^-11).  Rounding p * scale to fp16 multiplies every term
# p (code - 8) scale by 1 + 2^-11 at most; against the sum of the terms themselves that is at most 8 / rms(code - 8) = 1.75 times
# 2^-11, twice allowed for rows whose terms cancel more than usual: 2^-9.  Scores are fp32 sums: 2^-24 of 256 terms of up to 8
# times the score's own scale, 5e-4 with room.
TOL = {torch.bfloat16: 2.0 ** -8 + 2.0 ** -9 + 5e-4, torch.float16: 2.0 ** -11 + 2.0 ** -9 + 5e-4}


@pytest.fixture(autouse=True)
def no_device_error():
    """A bounded wait that ran out is a failure even where the values are right."""
    yield
    assert _lib.lib().dflash_device_error(0) == 0


def check_rows(got, want, dtype):
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    err = (got.double() - want).nan_to_num(0).norm(dim=-1)
    norm = want.nan_to_num(0).norm(dim=-1)
    # subnormal outputs aside, a zero row has to be zero
    bad = err > TOL[dtype] * norm + 1e-7 * (norm > 0)
    assert not bool(bad.any()), (float((err / norm.clamp_min(1e-30)).max()), bad.nonzero()[:5].tolist())


# ---- write and read ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Hk,D,T,cap", [(1, 1, 128, 1, 1), (1, 4, 256, 1, 64), (3, 2, 128, 16, 40), (2, 3, 256, 7, 33), (2, 2, 128, 613, 700),
                                          (1, 4, 256, 701, 701)])
def test_write_then_read(B, Hk, D, T, cap, dtype):
    k_cache, v_cache = make_cache(B, Hk, cap, D, dtype, seed=10)
    k, v = states((B, Hk, T, D), dtype, 20, 3.0), states((B, Hk, T, D), dtype, 21)
    k[0, 0, 0, :64] = 1.5                                  # a group without a range
    v[0, 0, T - 1, 64:] = 0
    at = [(5 * b) % (cap - T + 1) for b in range(B)]
    want = []
    for x, c in ((k, k_cache), (v, v_cache)):
        w = [p.clone() for p in c]
        for part, new in zip(w, ref.quantise(x)):
            for b in range(B):
                part[b, :, at[b]:at[b] + T] = new[b]
        want.append(w)
    qkv.quantized_kv_write(k, v, k_cache, v_cache, ints(*at))
    for c, w in zip((k_cache, v_cache), want):
        for got, p in zip(c, w):
            assert torch.equal(got, p)                    # to the last bit, and every other row as it was
    for c, x in zip(want, qkv.quantized_kv_read(k_cache, v_cache, 0, cap)):
        assert torch.equal(x, ref.values(*c, torch.float32).to(dtype))
    got = qkv.quantized_kv_read(k_cache, v_cache, ints(*at), T)
    for c, x in zip(want, got):
        for b in range(B):
            assert torch.equal(x[b], ref.values(*[p[b, :, at[b]:at[b] + T] for p in c], torch.float32).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_write_extremes(dtype):
    k_cache, v_cache = make_cache(1, 1, 16, 128, dtype)
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = states((1, 1, 8, 128), dtype, 3)
    x[0, 0, 0, 0], x[0, 0, 0, 1] = big, -big              # the range overflows fp32 unless each side is divided first
    x[0, 0, 1] = 0
    x[0, 0, 2, :64] = torch.where(torch.arange(64, device=DEV) % 2 == 0, tiny, -tiny).to(dtype)
    x[0, 0, 3, 70] = math.inf
    x[0, 0, 4, 3] = math.nan
    x[0, 0, 5, 64:] = -big
    x[0, 0, 6, 5], x[0, 0, 6, 6] = -math.inf, math.inf
    qkv.quantized_kv_write(x, x, k_cache, v_cache, ints(2))
    for c in (k_cache, v_cache):
        for got, want in zip(c, ref.quantise(x)):
            assert torch.equal(got[:, :, 2:10].nan_to_num(77.0) if got.is_floating_point() else got[:, :, 2:10],
                               want.nan_to_num(77.0) if want.is_floating_point() else want)
    back = qkv.quantized_kv_read(k_cache, v_cache, 2, 8)[0]
    assert bool(back[0, 0, 3, 64:].isnan().all()) and bool(back[0, 0, 3, :64].isfinite().all())
    assert bool(back[0, 0, 4, :64].isnan().all()) and bool(back[0, 0, 4, 64:].isfinite().all())
    assert torch.equal(back[0, 0, 1], torch.zeros_like(back[0, 0, 1]))


def test_write_padded_batch_and_capacity():
    dtype = torch.bfloat16
    k_cache, v_cache = make_cache(4, 2, 20, 128, dtype)
    before = [p.clone() for p in (*k_cache, *v_cache)]
    k, v = states((4, 2, 8, 128), dtype, 5), states((4, 2, 8, 128), dtype, 6)
    k[1, :, 3:] = math.nan                                # padding is not even looked at
    _lib.lib().dflash_device_error(0)
    qkv.quantized_kv_write(k, v, k_cache, v_cache, ints(0, 12, 17, 3), counts=ints(0, 3, 3, 99))
    assert _lib.lib().dflash_device_error(0) == 0
    for i, (x, part) in enumerate([(k, 0), (k, 1), (k, 2), (v, 0), (v, 1), (v, 2)]):
        want = before[i]
        new = ref.quantise(x)[part]
        want[1, :, 12:15], want[2, :, 17:20], want[3, :, 3:11] = new[1, :, :3], new[2, :, :3], new[3, :, :8]
        assert torch.equal((*k_cache, *v_cache)[i], want)
    # positions outside the cache are dropped and reported
    qkv.quantized_kv_write(k, v, k_cache, v_cache, ints(18, -3, 2 ** 31 - 4, 0), counts=ints(8, 2, 8, 0))
    code = _lib.lib().dflash_device_error(0)
    assert code & 0xFF == 61
    for i, (x, part) in enumerate([(k, 0), (k, 1), (k, 2), (v, 0), (v, 1), (v, 2)]):
        before[i][0, :, 18:20] = ref.quantise(x)[part][0, :, :2]
        assert torch.equal((*k_cache, *v_cache)[i], before[i])


def test_read_outside_is_zero_and_long_starts():
    k_cache, v_cache = make_cache(2, 1, 10, 128, torch.float16)
    k, v = qkv.quantized_kv_read(k_cache, v_cache, ints(-2, 8), 5)
    full = ref.values(*k_cache, torch.float32).half()
    assert torch.equal(k[0, :, 2:], full[0, :, :3]) and not bool(k[0, :, :2].any())
    assert torch.equal(k[1, :, :2], full[1, :, 8:]) and not bool(k[1, :, 2:].any()) and not bool(v[1, :, 2:].any())
    assert qkv.quantized_kv_read(k_cache, v_cache, 3, 0)[0].shape == (2, 1, 0, 128)
    assert not bool(qkv.quantized_kv_read(k_cache, v_cache, 2 ** 31 - 1, 3)[0].any())


def test_write_strided_and_sliced():
    """Keys as a transposed view of a projection, and a cache that is a slice of a larger one."""
    B, Hk, T, D, dtype = 2, 2, 5, 128, torch.bfloat16
    proj = states((B, T, 2 * Hk * D + 8), dtype, 8)
    k = proj[..., :Hk * D].view(B, T, Hk, D).transpose(1, 2)
    v = proj[..., Hk * D:2 * Hk * D].view(B, T, Hk, D).transpose(1, 2)
    odd = proj[..., 1:1 + Hk * D].view(B, T, Hk, D).transpose(1, 2)       # rows that are not 16-byte aligned: copied
    whole = make_cache(3, 4, 40, D, dtype)
    k_cache, v_cache = (qkv.QuantizedKV(*[p[1:, 2:, 4:36] for p in c]) for c in whole)
    before = [p.clone() for c in whole for p in c]
    qkv.quantized_kv_write(k, v, k_cache, v_cache, ints(0, 27))
    for x, c in ((k, k_cache), (v, v_cache)):
        for got, want in zip(c, ref.quantise(x.contiguous())):
            assert torch.equal(got[0, :, :5], want[0]) and torch.equal(got[1, :, 27:32], want[1])
    for c, old in zip([p for c in whole for p in c], before):
        assert torch.equal(c[0], old[0]) and torch.equal(c[:, :2], old[:, :2]) and torch.equal(c[1, 2:, 9:], old[1, 2:, 9:])
    qkv.quantized_kv_write(odd, v, k_cache, v_cache, ints(3, 3))
    assert torch.equal(k_cache.codes[:, :, 3:8], ref.quantise(odd.contiguous())[0])
    back = qkv.quantized_kv_read(k_cache, v_cache, 3, 5)[0]
    assert torch.equal(back, ref.values(*ref.quantise(odd.contiguous()), torch.float32).to(dtype))


# ---- attention --------------------------------------------------------------------------------------------------------
def run_sdpa(B, Hq, Hk, D, T, lengths, dtype, *, mask=None, cap=None, max_length=None, seed=0, num_splits=0, spread=1.0):
    cap = cap or max(1, max(lengths)) + 3
    k_cache, v_cache = make_cache(B, Hk, cap, D, dtype, seed, spread)
    q = states((B, Hq, T, D), dtype, seed + 5)
    scale = D ** -0.5 / spread
    got = qkv.quantized_kv_sdpa(q, k_cache, v_cache, scale, ints(*lengths), mask, max_length=max_length, num_splits=num_splits)
    check_rows(got, ref.sdpa(q, k_cache, v_cache, scale, lengths, mask, max_length), dtype)
    return q, k_cache, v_cache, scale, got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("Hq,Hk,T", [(1, 1, 1), (6, 1, 1), (8, 2, 2), (9, 1, 1), (16, 2, 1), (12, 3, 4), (6, 1, 16), (4, 4, 5), (24, 1, 3)])
def test_attention_shapes(Hq, Hk, T, D, dtype):
    run_sdpa(2, Hq, Hk, D, T, [T + 130, T], dtype)


@pytest.mark.parametrize("T", [1, 16])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300, 1025])
def test_attention_lengths(n, T):
    # lengths below T leave the first rows without a key
    run_sdpa(1, 4, 2, 128, T, [n], torch.bfloat16, seed=n)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_ragged_and_empty(dtype):
    q, k, v, scale, got = run_sdpa(5, 4, 2, 128, 4, [0, 3, 513, 200, 4], dtype, cap=513)
    assert not bool(got[0].any()) and not bool(got[1, :, 0].any())
    # negative lengths see nothing, lengths beyond max_length are cut off but keep their causal order
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(-7, 3, 515, 200, 4), max_length=512)
    check_rows(got, ref.sdpa(q, k, v, scale, [-7, 3, 515, 200, 4], max_length=512), dtype)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
def test_attention_splits(splits):
    run_sdpa(2, 6, 2, 256, 3, [900, 17], torch.bfloat16, num_splits=splits)


@pytest.mark.parametrize("T", [65, 130, 257])
def test_attention_prompt_chunks(T):
    run_sdpa(1, 3, 1, 128, T, [T], torch.bfloat16, seed=T)
    run_sdpa(2, 2, 1, 256, T, [T + 77, T - 1], torch.float16, seed=T)


def test_attention_host_length_and_no_keys():
    q, k, v, scale, got = run_sdpa(2, 4, 2, 128, 3, [50, 50], torch.bfloat16)
    assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, 50), got)
    assert not bool(qkv.quantized_kv_sdpa(q, k, v, scale, 0).any())
    assert qkv.quantized_kv_sdpa(q[:, :, :0], k, v, scale, 50).shape == (2, 4, 0, 128)
    for bad in (dict(lengths=54), dict(lengths=-1), dict(lengths=50, max_length=51), dict(lengths=ints(1)),
                dict(lengths=ints(1, 2).long()), dict(lengths=ints(5, 5), max_length=99)):
        with pytest.raises(ValueError):
            qkv.quantized_kv_sdpa(q, k, v, scale, **bad)
    for bad in (math.nan, math.inf, 1e39):
        with pytest.raises(ValueError, match="scale"):
            qkv.quantized_kv_sdpa(q, k, v, bad, 50)
    for bad in (q[:, :3], q.half(), q[..., :64], q[:1]):
        with pytest.raises(ValueError):
            qkv.quantized_kv_sdpa(bad, k, v, scale, 50)
    with pytest.raises(ValueError):
        qkv.quantized_kv_sdpa(q, k, v, scale, 50, torch.zeros(1, 1, 1, 50, device=DEV, dtype=torch.float64))
    with pytest.raises(RuntimeError):
        qkv.quantized_kv_sdpa(q, k, v, scale, 50, torch.ones(1, 1, 1, 49, device=DEV, dtype=torch.bool))


@pytest.mark.parametrize("T", [1, 4, 40])
@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("shape", ["full", "keys", "heads", "rows"])
def test_attention_masks(shape, kind, T):
    B, Hq, Hk, D, n, dtype = 2, 4, 2, 128, 150, torch.bfloat16
    dims = {"full": (B, Hq, T, n), "keys": (B, 1, 1, n), "heads": (1, Hq, 1, n), "rows": (T, n)}[shape]
    keep = torch.rand(dims, generator=gen(3), device=DEV) < 0.6
    if shape == "full":
        keep[0, 1, 0] = False                             # a row with nothing left
    mask = keep
    if kind != "bool":
        mask = torch.where(keep, torch.randn(dims, generator=gen(4), device=DEV), torch.full(dims, -math.inf, device=DEV))
        mask = mask.to(dtype if kind == "type" else torch.float32)
    _, _, _, _, got = run_sdpa(B, Hq, Hk, D, T, [n, n - 20], dtype, mask=mask, cap=n, max_length=n)
    if shape == "full":
        assert not bool(got[0, 1, 0].any())


@pytest.mark.parametrize("T", [5, 40])
@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
def test_attention_mask_alignment(kind, T):
    """A mask's place in memory changes nothing, nor does what lies around it."""
    B, Hq, Hk, D, n, dtype = 2, 5, 1, 128, 203, torch.bfloat16
    k, v = make_cache(B, Hk, n, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.rand(B, Hq, T, n, generator=gen(3), device=DEV) < 0.7
    mask, around = keep, True
    if kind != "bool":
        mask = torch.where(keep, torch.randn(keep.shape, generator=gen(4), device=DEV), -math.inf).to(dtype if kind == "type" else torch.float32)
        around = math.nan
    want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), mask)
    check_rows(want, ref.sdpa(q, k, v, scale, [n, n - 70], mask), dtype)
    for off in [*range(17), 31]:
        wide = torch.full((B, Hq, T, off + n + off % 3), around, dtype=mask.dtype, device=DEV)
        wide[..., off:off + n] = mask
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), wide[..., off:off + n]), want), off
    for turned in (mask.transpose(-1, -2).contiguous().transpose(-1, -2), mask.repeat_interleave(2, -1)[..., ::2]):
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), turned), want)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_attention_queries_that_are_not_finite(odd, kind, T):
    """They make their own row NaN, unless its mask leaves nothing: then it is zero like any other."""
    B, Hq, Hk, D, n, dtype = 1, 4, 1, 128, 100, torch.bfloat16
    k, v = make_cache(B, Hk, n, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.ones(B, Hq, T, n, dtype=torch.bool, device=DEV)
    keep[0, 1, 1] = False
    keep[0, 2, 2, 40:] = False
    mask = keep if kind == "bool" else torch.where(keep, 0.5, -math.inf).to(dtype if kind == "type" else torch.float32)
    want = qkv.quantized_kv_sdpa(q, k, v, scale, n, mask)
    q[0, 1, 1, 5] = q[0, 2, 2, 77] = odd
    got = qkv.quantized_kv_sdpa(q, k, v, scale, n, mask)
    assert not bool(want[0, 1, 1].any()) and not bool(got[0, 1, 1].any())
    assert bool(got[0, 2, 2].isnan().all())
    got[0, 2, 2] = want[0, 2, 2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("T", [1, 17])
@pytest.mark.parametrize("splits", [9, 600, 1024])
def test_attention_as_many_splits_as_there_may_be(splits, T):
    run_sdpa(1, 1, 1, 128, T, [140001], torch.bfloat16, cap=140100, max_length=140001, num_splits=splits)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [2009, 2048 + 64, 2048 + 65, 9001])
@pytest.mark.parametrize("T", [4, 10, 21])
def test_attention_few_of_128_rows_over_many_tiles(T, n, D):
    """Rows that fill only some warps of a block, over ranges that end inside either half of their last 128 keys: nothing may run
    ahead of the last ones.  The same bits every time, and right."""
    B, Hq, Hk, dtype = 1, 12, 2, torch.bfloat16
    _, _, _, _, got = args = run_sdpa(B, Hq, Hk, D, T, [n], dtype, cap=n, max_length=n, num_splits=1)
    q, k, v, scale = args[:4]
    for _ in range(30):
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, n, num_splits=1), got)


@pytest.mark.parametrize("T", [2, 40])
def test_attention_lowest_finite_mask(T):
    """The type's lowest value is a number: a row that has nothing else is the mean of what it may see."""
    n, dtype = 70, torch.bfloat16
    mask = torch.full((1, 1, T, n), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    mask[0, 0, 1, 20] = 0
    q, k, v, scale, got = run_sdpa(1, 2, 1, 128, T, [n], dtype, mask=mask, cap=n, max_length=n)
    mean = ref.values(*v)[0, 0, :n - T + 1].mean(0)
    # scores vanish next to the lowest value in fp32 and in the oracle's 64 bits alike
    assert float((got[0, 0, 0].double() - mean).norm() / mean.norm()) < TOL[dtype]
    assert float((got[0, 0, 1].double() - ref.values(*v)[0, 0, 20]).norm()) < TOL[dtype] * float(ref.values(*v)[0, 0, 20].norm())


@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_nan_in_hidden_places(T):
    """What a row does not see never reaches it: behind the length, behind the row, under the mask."""
    B, Hq, Hk, D, n, dtype = 2, 4, 1, 256, 90, torch.bfloat16
    k, v = make_cache(B, Hk, 128, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.ones(B, 1, 1, 128, dtype=torch.bool, device=DEV)
    keep[:, :, :, [4, 33]] = False
    want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), keep)
    for bad in (math.nan, math.inf, -math.inf):
        for c in (k, v):
            for part in (c.scales, c.biases):
                part[:, :, [4, 33], 1] = bad
                part[0, :, n:] = bad
                part[1, :, n - 11:] = bad
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), keep), want)
    if T > 1:                                             # the last key is seen by the last row alone
        v.biases[0, 0, n - 1, 2] = math.nan
        got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), keep)
        assert bool(got[0, :, T - 1].isnan().all()) and torch.equal(got[0, :, :T - 1], want[0, :, :T - 1]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("spread", [1e-6, 1e-3, 300.0, 1e5, 1e30])
def test_attention_value_ranges(spread, T):
    """bf16 reaches far beyond fp16: scales of any size, mixed within a sequence."""
    B, Hq, Hk, D, n, dtype = 1, 4, 1, 128, 200, torch.bfloat16
    k, _ = make_cache(B, Hk, n, D, dtype, 1)
    x = states((B, Hk, n, D), torch.float32, 2) * spread
    x[:, :, 100:150] *= 1e-4
    v = qkv.QuantizedKV(*ref.quantise(x.to(dtype)))
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.ones(1, Hq, 1, n, dtype=torch.bool, device=DEV)
    keep[:, 0, :, :100] = False                           # head 0 sees the small values alone
    keep[:, 0, :, 150:] = False
    got = qkv.quantized_kv_sdpa(q, k, v, scale, n, keep)
    check_rows(got, ref.sdpa(q, k, v, scale, [n], keep), dtype)


def test_attention_negative_scales_and_large_scores():
    """Other quantisers store negative scales; large scores make the running maximum move often."""
    B, Hq, Hk, D, n, dtype = 1, 2, 1, 128, 400, torch.bfloat16
    k, v = make_cache(B, Hk, n, D, dtype, 4)
    for c in (k, v):
        c.biases.copy_((c.biases.float() + 15 * c.scales.float()).to(dtype))
        c.scales.neg_()
    for T in (1, 40):
        q = states((B, Hq, T, D), dtype, 9, 4.0)
        got = qkv.quantized_kv_sdpa(q, k, v, 1.0, n)
        check_rows(got, ref.sdpa(q, k, v, 1.0, [n]), dtype)


@pytest.mark.parametrize("T", [1, 40])
def test_attention_query_strides(T):
    B, Hq, Hk, D, n, dtype = 2, 4, 2, 128, 100, torch.bfloat16
    k, v = make_cache(B, Hk, n, D, dtype)
    flat = states((B, T, Hq * D + 8), dtype, 3)
    q = flat[..., :Hq * D].view(B, T, Hq, D).transpose(1, 2)
    want = qkv.quantized_kv_sdpa(q.contiguous(), k, v, 0.1, n)
    assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, 0.1, n), want)
    odd = flat[..., 3:3 + Hq * D].view(B, T, Hq, D).transpose(1, 2)
    assert torch.equal(qkv.quantized_kv_sdpa(odd, k, v, 0.1, n), qkv.quantized_kv_sdpa(odd.contiguous(), k, v, 0.1, n))
    one = flat[:1, :1, :D].view(1, 1, 1, D).expand(B, Hq, T, D)
    assert torch.equal(qkv.quantized_kv_sdpa(one, k, v, 0.1, n), qkv.quantized_kv_sdpa(one.contiguous(), k, v, 0.1, n))


def test_attention_cache_slices():
    whole = make_cache(3, 4, 80, 128, torch.bfloat16)
    k, v = (qkv.QuantizedKV(*[p[1:, 1:3, 8:72] for p in c]) for c in whole)
    dense = [qkv.QuantizedKV(*[p.contiguous() for p in c]) for c in (k, v)]
    for T in (1, 40):
        q = states((2, 4, T, 128), torch.bfloat16, 3)
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, 0.1, 61), qkv.quantized_kv_sdpa(q, *dense, 0.1, 61))


def test_results_do_not_change_from_call_to_call():
    k, v = make_cache(2, 2, 700, 256, torch.bfloat16)
    for T in (1, 7, 40):
        q = states((2, 12, T, 256), torch.bfloat16, 3)
        first = qkv.quantized_kv_sdpa(q, k, v, 0.06, ints(700, 333))
        for _ in range(5):
            assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, 0.06, ints(700, 333)), first)


@pytest.mark.parametrize("seed", range(24))
def test_attention_random_shapes(seed):
    """Heads, rows, lengths, masks and types drawn at random, both kernels and their edges."""
    import random
    r = random.Random(seed)
    dtype, D = r.choice(TYPES), r.choice([128, 256])
    Hk, g = r.choice([1, 2, 3]), r.choice([1, 2, 5, 6, 8])
    T = r.choice([1, 2, 3, r.randint(4, 16), r.randint(17, 60)])
    B = r.randint(1, 3)
    cap = r.randint(max(T, 2), 700)
    n_max = r.randint(1, cap)
    lengths = [r.choice([0, T, n_max, r.randint(0, n_max), cap + 5]) for _ in range(B)]
    mask = None
    if r.random() < 0.5:
        dims = r.choice([(B, 1, 1, n_max), (1, g * Hk, T, n_max), (n_max,), (B, 1, T, 1)])
        keep = torch.rand(dims, generator=gen(seed), device=DEV) < 0.7
        mask = r.choice([keep, torch.where(keep, torch.randn(dims, generator=gen(seed), device=DEV), -math.inf).to(r.choice([dtype, torch.float32]))])
    run_sdpa(B, g * Hk, Hk, D, T, lengths, dtype, mask=mask, cap=cap, max_length=n_max, seed=seed, num_splits=r.choice([0, 0, 1, 3]))


@pytest.mark.parametrize("T", [2, 40])
def test_attention_scales_and_nan_queries(T):
    """Zero and negative scales; a NaN or infinite query stays in its own row."""
    k, v = make_cache(1, 2, 300, 128, torch.bfloat16)
    q = states((1, 4, T, 128), torch.bfloat16, 3)
    for scale in (0.0, -0.1, 1e-30):
        check_rows(qkv.quantized_kv_sdpa(q, k, v, scale, 300), ref.sdpa(q, k, v, scale, [300]), torch.bfloat16)
    want = qkv.quantized_kv_sdpa(q, k, v, 0.1, 300)
    for bad in (math.nan, math.inf):
        p = q.clone()
        p[0, 1, 1, 5] = bad
        got = qkv.quantized_kv_sdpa(p, k, v, 0.1, 300)
        assert bool(got[0, 1, 1].isnan().all())
        got[0, 1, 1] = want[0, 1, 1]
        assert torch.equal(got, want)
    tiny = q * 1e-30                                       # queries below fp16's range
    check_rows(qkv.quantized_kv_sdpa(tiny, k, v, 1e29, 300), ref.sdpa(tiny, k, v, 1e29, [300]), torch.bfloat16)
    big = q * 1e30
    check_rows(qkv.quantized_kv_sdpa(big, k, v, 1e-31, 300), ref.sdpa(big, k, v, 1e-31, [300]), torch.bfloat16)


def test_extreme_lengths_and_shared_caches():
    k, v = make_cache(1, 2, 64, 128, torch.bfloat16)
    for T in (2, 40):
        q = states((3, 4, T, 128), torch.bfloat16, 3)
        shared = [qkv.QuantizedKV(*[p.expand(3, -1, -1, -1) for p in c]) for c in (k, v)]     # one prefix, three readers
        lengths = [-2 ** 31, 2 ** 31 - 1, 50]
        got = qkv.quantized_kv_sdpa(q, *shared, 0.1, ints(*lengths))
        assert not bool(got[0].any())
        check_rows(got, ref.sdpa(q, *shared, 0.1, lengths), torch.bfloat16)
        x = states((3, 2, T, 128), torch.bfloat16, 4)
        with pytest.raises(ValueError, match="repeat"):
            qkv.quantized_kv_write(x, x, *shared, ints(0, 0, 0))


def test_long_cache_offsets_pass_32_bits():
    """2^31 words of codes in one array: positions far into it are addressed in 64 bits."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 30 GB")
    B, Hk, D, cap, dtype = 2, 1, 256, 2 ** 25 + 64, torch.bfloat16      # B * cap * 32 words = 2^31 + 4096 words
    k, v = qkv.allocate(B, Hk, cap, D, dtype=dtype, device=DEV)
    x = states((B, Hk, 96, D), dtype, 3)
    at = cap - 96
    qkv.quantized_kv_write(x, x, k, v, ints(at, at))
    want = ref.values(*ref.quantise(x), torch.float32).to(dtype)
    assert torch.equal(qkv.quantized_kv_read(k, v, at, 96)[1], want)
    q = states((B, 2, 1, D), dtype, 4)
    keep = torch.zeros(1, 1, 1, cap, dtype=torch.bool, device=DEV)
    keep[..., at:] = True
    got = qkv.quantized_kv_sdpa(q, k, v, 0.06, cap, keep)
    small = [qkv.QuantizedKV(*[p[:, :, at:].contiguous() for p in c]) for c in (k, v)]
    check_rows(got, ref.sdpa(q, *small, 0.06, [96, 96]), dtype)


def test_streams_graphs_and_two_calls_at_once():
    """Captured once and replayed at other positions; graphs and streams side by side share nothing."""
    B, Hq, Hk, D, T, dtype = 2, 12, 2, 128, 4, torch.bfloat16
    cache = qkv.QuantizedKVCache(B, Hk, 600, D, dtype=dtype)
    cache.keys, cache.values = make_cache(B, Hk, 600, D, dtype)
    k, v, q = (states((B, h, T, D), dtype, s) for h, s in ((Hk, 1), (Hk, 2), (Hq, 3)))
    outs = []

    def step():
        cache.update(k, v)
        outs.append(cache.attend(q, 0.09))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append((g, outs[-1]))
    for at in (5, 333, 590):
        cache.offsets.fill_(at)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        want = ref.sdpa(q, cache.keys, cache.values, 0.09, [at + T] * B)
        for g, out in graphs:
            check_rows(out, want, dtype)
        for x, c in ((k, cache.keys), (v, cache.values)):
            assert torch.equal(c.codes[:, :, at:at + T], ref.quantise(x)[0])


def test_cache_runs_prompt_verify_rollback_and_tokens():
    """A prompt in chunks, a verify block of which a part is accepted, then single tokens: against dense attention over what
    the cache stands for."""
    B, Hq, Hk, D, dtype = 2, 6, 2, 128, torch.bfloat16
    cache = qkv.QuantizedKVCache(B, Hk, 256, D, dtype=dtype)
    assert cache.nbytes == 2 * B * Hk * 256 * (D // 2 + 4 * D // 64)
    kept = [torch.zeros(B, 0, dtype=torch.long)]
    dense_k, dense_v = [torch.zeros(B, Hk, 256, D, dtype=dtype, device=DEV) for _ in range(2)]
    at = torch.zeros(B, dtype=torch.int32, device=DEV)
    for i, (T, accepted) in enumerate([(90, 90), (37, 37), (16, ints(5, 16)), (16, ints(1, 1)), (1, 1), (1, 1)]):
        q, k, v = states((B, Hq, T, D), dtype, 3 * i), states((B, Hk, T, D), dtype, 3 * i + 1), states((B, Hk, T, D), dtype, 3 * i + 2)
        cache.update(k, v)
        for b in range(B):
            o = int(at[b])
            dense_k[b, :, o:o + T], dense_v[b, :, o:o + T] = k[b], v[b]
        got = cache.attend(q, D ** -0.5)
        check_rows(got, ref.sdpa(q, ref.quantise(dense_k), ref.quantise(dense_v), D ** -0.5, (at + T).tolist()), dtype)
        cache.commit(accepted)
        at += accepted
        assert torch.equal(cache.offsets, at)
    n = int(at.min())
    assert torch.equal(cache.read(0, n)[0], ref.values(*ref.quantise(dense_k[:, :, :n]), torch.float32).to(dtype))
    assert kept


# ---- many rows over long caches (few rows and short caches take the other kernel) ----------------------------------------
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["none", "bool", "type", "f32"])
@pytest.mark.parametrize("shape", ["full", "keys", "heads", "rows"])
def test_long_attention_masks(shape, kind, D):
    """Every kind of mask at every alignment of its rows, rows and whole tiles with nothing left among them."""
    B, Hq, Hk, T, n, dtype = 2, 4, 2, 40, 1311, torch.float16 if shape == "heads" else torch.bfloat16
    dims = {"full": (B, Hq, T, n), "keys": (B, 1, 1, n), "heads": (1, Hq, 1, n), "rows": (T, n)}[shape]
    keep = torch.rand(dims, generator=gen(3), device=DEV) < 0.6
    keep[..., 200:420] = False
    if shape == "full":
        keep[0, 1, 0] = False
        keep[1, 3, :30] = False
    mask = keep if kind == "bool" else None
    if kind in ("type", "f32"):
        mask = torch.where(keep, torch.randn(dims, generator=gen(4), device=DEV), torch.full(dims, -math.inf, device=DEV))
        mask = mask.to(dtype if kind == "type" else torch.float32)
    for lengths in ([n, n - 20], [n - 700, n]):
        _, _, _, _, got = run_sdpa(B, Hq, Hk, D, T, lengths, dtype, mask=mask, cap=n, max_length=n)
        if shape == "full" and mask is not None:
            assert not bool(got[0, 1, 0].any()) and not bool(got[1, 3, :30].any())


@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
def test_long_attention_mask_alignment(kind):
    B, Hq, Hk, D, n, T, dtype = 2, 5, 1, 128, 1203, 40, torch.bfloat16
    k, v = make_cache(B, Hk, n, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.rand(B, Hq, T, n, generator=gen(3), device=DEV) < 0.7
    mask, around = keep, True
    if kind != "bool":
        mask = torch.where(keep, torch.randn(keep.shape, generator=gen(4), device=DEV), -math.inf).to(dtype if kind == "type" else torch.float32)
        around = math.nan
    want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), mask)
    check_rows(want, ref.sdpa(q, k, v, scale, [n, n - 70], mask), dtype)
    for off in [*range(17), 31]:
        wide = torch.full((B, Hq, T, off + n + off % 3), around, dtype=mask.dtype, device=DEV)
        wide[..., off:off + n] = mask
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), wide[..., off:off + n]), want), off
    for turned in (mask.transpose(-1, -2).contiguous().transpose(-1, -2), mask.repeat_interleave(2, -1)[..., ::2]):
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 70), turned), want)


@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_long_attention_values_that_are_not_finite(odd, kind):
    """Behind the length, behind the row, under the mask they reach nothing; a query's own row they do."""
    B, Hq, Hk, D, n, T, dtype = 2, 4, 1, 256, 1290, 40, torch.bfloat16
    k, v = make_cache(B, Hk, n + 30, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.ones(B, Hq, T, n + 30, dtype=torch.bool, device=DEV)
    keep[:, :, :, [4, 33, 1000]] = False
    keep[0, 1, 1] = False
    mask = keep if kind == "bool" else torch.where(keep, 0.5, -math.inf).to(dtype if kind == "type" else torch.float32)
    want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), mask)
    check_rows(want, ref.sdpa(q, k, v, scale, [n, n - 11], mask), dtype)
    for c in (k, v):
        for part in (c.scales, c.biases):
            part[:, :, [4, 33, 1000], 1] = odd
            part[0, :, n:] = odd
            part[1, :, n - 11:] = odd
    assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), mask), want)
    q[0, 1, 1, 5] = q[0, 2, 2, 77] = odd
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), mask)
    assert not bool(got[0, 1, 1].any()) and bool(got[0, 2, 2].isnan().all())
    got[0, 2, 2] = want[0, 2, 2]
    assert torch.equal(got, want)
    v.biases[0, 0, n - 1, 2] = math.nan                   # seen by the last row alone
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, n - 11), mask)
    assert bool(got[0, :, T - 1].isnan().all()) and torch.equal(got[1], want[1]) and torch.equal(got[0, :, :2].isnan(), torch.zeros_like(got[0, :, :2]).bool())


@pytest.mark.parametrize("spread", [1e-6, 1e-3, 300.0, 1e5, 1e30])
def test_long_attention_value_ranges(spread):
    B, Hq, Hk, D, n, T, dtype = 1, 8, 1, 128, 1500, 40, torch.bfloat16
    k, _ = make_cache(B, Hk, n, D, dtype, 1)
    x = states((B, Hk, n, D), torch.float32, 2) * spread
    x[:, :, 100:150] *= 1e-4
    x[:, :, 1200:1300] *= 1e-3
    v = qkv.QuantizedKV(*ref.quantise(x.to(dtype)))
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    keep = torch.ones(1, Hq, 1, n, dtype=torch.bool, device=DEV)
    keep[:, 0, :, :100] = False                           # head 0 sees the small values alone
    keep[:, 0, :, 150:1200] = False
    keep[:, 0, :, 1300:] = False
    got = qkv.quantized_kv_sdpa(q, k, v, scale, n, keep)
    check_rows(got, ref.sdpa(q, k, v, scale, [n], keep), dtype)


@pytest.mark.parametrize("falling", [True, False])
def test_long_attention_biases_by_distance_and_lowest_values(falling):
    """Biases that grow or fall along the keys move the running maximum with every tile; the lowest finite value hides nothing."""
    B, Hq, Hk, D, n, T, dtype = 1, 8, 1, 128, 1400, 40, torch.bfloat16
    far = torch.arange(n, device=DEV).float()
    slopes = torch.pow(2.0, -torch.arange(Hq, device=DEV) / 2.0)[None, :, None, None]
    mask = (slopes * (far - n if falling else -far)).to(dtype).expand(B, Hq, T, n).contiguous()
    mask[:, 3] = torch.finfo(dtype).min
    _, _, v, _, got = run_sdpa(B, Hq, Hk, D, T, [n], dtype, mask=mask, cap=n, max_length=n)
    mean = ref.values(*v)[0, 0, :n - T + 1].mean(0)
    # P is rounded to fp16 (2^-11), and a mean of 1400 values with both signs is some 30 times smaller than they are
    assert float((got[0, 3, 0].double() - mean).norm()) < TOL[dtype] * float(mean.norm()) + 2.0 ** -11 * float(ref.values(*v)[0, 0].std())


def test_long_attention_negative_scales_and_strides():
    B, Hq, Hk, D, n, T, dtype = 2, 4, 1, 128, 1300, 40, torch.bfloat16
    whole = make_cache(3, 4, n + 20, D, dtype, 4)
    for c in whole:
        c.biases.copy_((c.biases.float() + 15 * c.scales.float()).to(dtype))
        c.scales.neg_()
    k, v = (qkv.QuantizedKV(*[p[1:, 2:3, 8:8 + n] for p in c]) for c in whole)
    dense = [qkv.QuantizedKV(*[p.contiguous() for p in c]) for c in (k, v)]
    flat = states((B, T, Hq * D + 8), dtype, 3, 4.0)
    for start in (0, 3):
        q = flat[..., start:start + Hq * D].view(B, T, Hq, D).transpose(1, 2)
        for scale in (0.3, -0.3, 0.0):
            got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n, 7))
            check_rows(got, ref.sdpa(q, *dense, scale, [n, 7]), dtype)
            assert torch.equal(got, qkv.quantized_kv_sdpa(q.contiguous(), *dense, scale, ints(n, 7)))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("n", [12009, 12032 + 64, 12032 + 65])
@pytest.mark.parametrize("T", [4, 10, 21])
def test_long_attention_of_few_of_128_rows(T, n, D):
    B, Hq, Hk, dtype = 1, 12, 2, torch.bfloat16
    _, _, _, _, got = args = run_sdpa(B, Hq, Hk, D, T, [n], dtype, cap=n, max_length=n, num_splits=1)
    for _ in range(20):
        assert torch.equal(qkv.quantized_kv_sdpa(*args[:4], n, num_splits=1), got)


def test_verify_cycle_with_token_probabilities():
    """What a server runs per cycle, captured once: the block's keys and values enter the cache, its rows attend, a head makes
    logits, the drafted tokens' log-probabilities decide how many are accepted, and the positions move on, all on the device."""
    B, Hq, Hk, D, T, V, dtype = 2, 8, 2, 128, 16, 3001, torch.bfloat16
    head = states((V, Hq * D), dtype, 1, 0.2)
    cache = qkv.QuantizedKVCache(B, Hk, 400, D, dtype=dtype)
    prompt = [states((B, h, 300, D), dtype, 2 + i) for i, h in enumerate((Hk, Hk))]
    cache.update(*prompt)
    cache.commit(300)
    q, k, v = states((B, Hq, T, D), dtype, 5), states((B, Hk, T, D), dtype, 6), states((B, Hk, T, D), dtype, 7)
    drafted = torch.randint(0, V, (B, T), generator=gen(8), device=DEV)
    threshold = torch.zeros(B, T, device=DEV)

    def cycle():
        cache.update(k, v)
        rows = cache.attend(q, D ** -0.5)
        logits = rows.transpose(1, 2).reshape(B, T, Hq * D) @ head.T
        lp = logprobs.token_logprobs(logits, drafted, top_k=4)
        accepted = (lp.logprobs >= threshold).to(torch.int32).cumprod(1).sum(1, dtype=torch.int32)
        cache.commit(accepted)
        return rows, logits, lp, accepted

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        cycle()                                           # a threshold of probability 1 accepts nothing
    torch.cuda.current_stream().wait_stream(side)
    assert cache.offsets.tolist() == [300, 300]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, logits, lp, accepted = cycle()
    dense = [torch.cat([p, torch.zeros(B, Hk, 100, D, dtype=dtype, device=DEV)], 2) for p in prompt]
    at = [300, 300]
    for step, counts in enumerate([(16, 3), (0, 16), (5, 1)]):
        q.copy_(states(q.shape, dtype, 20 + step)); k.copy_(states(k.shape, dtype, 30 + step)); v.copy_(states(v.shape, dtype, 40 + step))
        for b in range(B):
            threshold[b] = -math.inf
            threshold[b, counts[b]:] = 1.0
            for d, x in zip(dense, (k, v)):
                d[b, :, at[b]:at[b] + T] = x[b]
        graph.replay()
        check_rows(rows, ref.sdpa(q, ref.quantise(dense[0]), ref.quantise(dense[1]), D ** -0.5, [o + T for o in at]), dtype)
        want = ref_logprobs.token_logprobs(logits.flatten(0, 1), drafted.flatten().cpu(), 4)
        # fp32 sums of 3001 terms: 5e-6 of the sum and 2^-23 of values up to some tens
        assert float((lp.logprobs.flatten().cpu().double() - want[0]).abs().max()) < 2e-5
        assert torch.equal(lp.top_ids.flatten(0, 1).cpu().long(), want[3])
        assert accepted.tolist() == list(counts)
        at = [o + c for o, c in zip(at, counts)]
        assert cache.offsets.tolist() == at


def test_refusals_leave_everything_alone():
    k_cache, v_cache = make_cache(2, 2, 32, 128, torch.bfloat16)
    x = states((2, 2, 4, 128), torch.bfloat16, 1)
    for args, kw in (((x.half(), x.half()), {}), ((x, x[:, :1]), {}), ((x[..., :64], x[..., :64]), {}), ((x, x), {"offsets": ints(0)}),
                     ((x, x), {"offsets": ints(0, 0).long()}), ((x, x), {"counts": ints(1)}), ((x[:1], x[:1]), {})):
        kw = {"offsets": ints(0, 0), **kw}
        with pytest.raises(ValueError):
            qkv.quantized_kv_write(*args, k_cache, v_cache, **kw)
    with pytest.raises(ValueError):
        qkv.quantized_kv_read(k_cache, v_cache, 0, -1)
    with pytest.raises(ValueError):
        qkv.quantized_kv_read(k_cache, v_cache, 2 ** 31, 1)
    qkv.quantized_kv_write(x[:, :, :0], x[:, :, :0], k_cache, v_cache, ints(0, 0))
    assert torch.equal(k_cache.codes, make_cache(2, 2, 32, 128, torch.bfloat16)[0].codes)
