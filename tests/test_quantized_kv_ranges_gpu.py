"""The 4-bit KV cache's attention where keys and values differ in size as far as their type allows, in both kernels."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import quantized_kv as qkv  # noqa: E402
from oracle import quantized_kv as ref  # noqa: E402
from tests.test_quantized_kv_gpu import TOL, check_rows, gen, ints, make_cache, no_device_error, states  # noqa: E402, F401
from tests.test_quantized_kv_plan import plan  # noqa: E402

DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16
# T, keys, capacity: up to 8 and up to 16 rows of 4 heads, and many rows under a bound on the lengths that sends them to the tcgen05
# kernel
KERNELS = {"eight": (2, 190, 220), "sixteen": (3, 190, 220), "many": (40, 1290, 13000)}


def test_each_kernel_is_reached():
    for which, (T, _, cap) in KERNELS.items():
        assert plan(1, 4, 1, T, cap)[0] == plan(2, 4, 1, T, cap)[0] == (which == "many")


def part_of(k, v, name):
    return getattr(k if name[0] == "k" else v, "scales" if name[2:] == "scales" else "biases")


# ---- what a row does not see changes no bit of it --------------------------------------------------------------------------
@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("name", ["k scales", "k biases", "v scales", "v biases"])
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 256)])
def test_large_finite_values_in_hidden_places(dtype, D, name, kind, which):
    T, n, cap = KERNELS[which]
    B, Hq, Hk = 2, 4, 1
    k, v = make_cache(B, Hk, cap, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    hidden = [4, 33, n - 100, n - 60, n - 2]
    keep = torch.ones(1, 1, 1, cap, dtype=torch.bool, device=DEV)
    keep[..., hidden] = False
    mask = keep if kind == "bool" else torch.where(keep, 0.5, -math.inf).to(dtype if kind == "type" else torch.float32)
    lengths = ints(n, n - 11)
    want = qkv.quantized_kv_sdpa(q, k, v, scale, lengths, mask)
    check_rows(want, ref.sdpa(q, k, v, scale, [n, n - 11], mask), dtype)
    part = part_of(k, v, name)
    for big in (torch.finfo(dtype).max, -torch.finfo(dtype).max, 1e4, 1e30 if dtype == BF16 else 300.0):
        part[:, :, hidden, 1] = big
        part[0, :, n:] = big
        part[1, :, n - 11:] = big
        assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, lengths, mask), want), big


@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("name", ["k scales", "k biases", "v scales", "v biases"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("masked", [False, True])
def test_keys_that_some_rows_see(masked, dtype, name, which):
    """The last keys are seen by the last rows alone, others by some heads alone: the rest of the rows keep their bits."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, D = 1, 4, 1, 128
    k, v = make_cache(B, Hk, cap, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    mask = None
    if masked:
        mask = torch.ones(1, Hq, 1, cap, dtype=torch.bool, device=DEV)
        mask[:, :2, :, 20:n:7] = False
    want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), mask)
    part = part_of(k, v, name)
    part[0, 0, n - 1] = torch.finfo(dtype).max
    if masked:
        part[0, 0, 20:n - 1:7] = torch.finfo(dtype).max
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), mask)
    heads = slice(0, 2) if masked else slice(0, Hq)
    assert torch.equal(got[:, heads, :T - 1], want[:, heads, :T - 1])


# ---- keys and values of any size, seen by some rows and hidden from others ----------------------------------------------------
@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("octaves", [9, 14, 20, 40, 100])
def test_sizes_that_differ_within_a_block(octaves, kind, side, which):
    """Every third key or value is larger by `octaves`; head 0 sees the small ones alone, head 1 the large ones, head 2 all."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, D, dtype = 1, 4, 1, 128, BF16
    k, v = make_cache(B, Hk, cap, D, dtype)
    x = states((B, Hk, cap, D), torch.float32, 3)
    large = torch.arange(cap, device=DEV) % 3 == 1
    # values from 2^(-octaves/2) to 2^(octaves/2); keys up to 2^octaves, whose scores leave one key with all of the weight
    x = x * torch.where(large, 2.0 ** (octaves / 2), 2.0 ** (-octaves / 2) if side == "v" else 1.0)[:, None]
    side_of = qkv.QuantizedKV(*ref.quantise(x.to(dtype)))
    if side == "k":
        k = side_of
    else:
        v = side_of
    keep = torch.ones(1, Hq, 1, cap, dtype=torch.bool, device=DEV)
    keep[:, 0] = ~large
    keep[:, 1] = large
    mask = keep if kind == "bool" else torch.where(keep, 0.5, -math.inf).to(dtype if kind == "type" else torch.float32)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), mask)
    want = ref.sdpa(q, k, v, scale, [n], mask)
    if side == "v":
        check_rows(got, want, dtype)
        return
    # head 0's scores are of ordinary size; the others' winners may be too near to one another for fp32 scores of that size
    check_rows(got[:, :1], want[:, :1], dtype)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("splits", [0, 1])
def test_small_values_first_then_large_ones_and_back(splits, D, which):
    """A row's values of a size of their own in every stretch of its keys, from the type's smallest to its largest."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, dtype = 1, 4, 1, BF16
    k, _ = make_cache(B, Hk, cap, D, dtype)
    q, scale = states((B, Hq, T, D), dtype, 9), D ** -0.5
    stretch = n // 6
    for order in ((-120, -40, 0, 3, 40, 110), (110, 40, 3, 0, -40, -120), (0, 90, -90, 0, 60, -60)):
        octave = torch.tensor([order[min(i // stretch, 5)] for i in range(cap)], device=DEV)
        x = states((B, Hk, cap, D), torch.float64, 3) * torch.pow(2.0, octave.double())[:, None]
        v = qkv.QuantizedKV(*ref.quantise(x.to(dtype)))
        keep = torch.ones(1, Hq, 1, cap, dtype=torch.bool, device=DEV)
        for h in range(3):                                # a head sees two of the stretches
            keep[:, h] = ((torch.arange(cap, device=DEV) // stretch) % 3 == h)
        got, want = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), keep, num_splits=splits), ref.sdpa(q, k, v, scale, [n], keep)
        check_rows(got, want, dtype)
        # however small the row is: half a step of bf16's subnormals in each channel aside
        assert bool(((got.double() - want).norm(dim=-1) <= TOL[dtype] * want.norm(dim=-1) + D ** 0.5 * 2.0 ** -134).all())


@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("dtype,most", [(BF16, 2.0 ** 104), (BF16, 2.0 ** 126), (F16, 60000.0)])
@pytest.mark.parametrize("splits", [0, 1, 12])
def test_values_that_span_their_type(splits, dtype, most, which):
    """Groups from far below to far above zero, as the write makes them; 60000 (1 + TOL) is still an fp16 number, and a mean of values of
    2^126 an fp32 one, although their sum is none."""
    T, n, cap = KERNELS[which]
    k, _ = make_cache(1, 1, cap, 128, dtype)
    x = states((1, 1, cap, 128), dtype, 3)
    x[..., 5], x[..., 6] = most, -most
    v = qkv.QuantizedKV(*ref.quantise(x))
    q, scale = states((1, 4, T, 128), dtype, 9), 128 ** -0.5
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), num_splits=splits)
    check_rows(got, ref.sdpa(q, k, v, scale, [n]), dtype)


# ---- scores of any size -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("kind", ["none", "bool", "f32"])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 1e7, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(sign, size, kind, which):
    """Keys that are one number each, exact in every step, so that scores of `size` still tell their order: a row is the mean of the
    values of its best keys."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, D, dtype = 1, 4, 1, 128, BF16
    _, v = make_cache(B, Hk, cap, D, dtype)
    level = torch.randint(0, 8, (cap,), generator=gen(7), device=DEV).to(dtype)     # the best is seen often, by all rows
    level[:10] = 11                                       # not a power of two: products of it are rounded
    k = qkv.QuantizedKV(torch.zeros(B, Hk, cap, D // 8, dtype=torch.int32, device=DEV), torch.zeros(B, Hk, cap, D // 64, dtype=dtype, device=DEV),
                        (sign * level)[None, None, :, None].expand(B, Hk, cap, D // 64).contiguous())
    q = torch.full((B, Hq, T, D), sign * 1.0, dtype=dtype, device=DEV)
    scale = size / (11 * D)                               # a level apart: size / 11, so that a lower one has no weight
    mask = None if kind == "none" else torch.ones(1, Hq, 1, cap, dtype=torch.bool, device=DEV)
    if kind != "none":
        mask[:, 1, :, :5] = False
    if kind == "f32":
        mask = torch.where(mask, 0.0, -math.inf)
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(n), mask)
    check_rows(got, ref.sdpa(q, k, v, scale, [n], mask), dtype)


@pytest.mark.parametrize("which", KERNELS)
def test_large_scores_under_many_ranges(which):
    """Ranges of keys that differ in their best score by little next to its size keep their weights."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, D, dtype = 1, 4, 1, 128, BF16
    _, v = make_cache(B, Hk, cap, D, dtype)
    level = torch.randint(0, 2, (cap,), generator=gen(7), device=DEV).float() * 0.5 + 64
    k = qkv.QuantizedKV(torch.zeros(B, Hk, cap, D // 8, dtype=torch.int32, device=DEV), torch.zeros(B, Hk, cap, D // 64, dtype=dtype, device=DEV),
                        level.to(dtype)[None, None, :, None].expand(B, Hk, cap, D // 64).contiguous())
    q = torch.ones(B, Hq, T, D, dtype=dtype, device=DEV)
    # scores 2^17 and 2^17 + 2^10: the difference decides; then scores 2^17 (1 + 2^-7 ..) with a difference of 2, where fp32 is exact
    for splits in (1, 2, 5, 9):
        got = qkv.quantized_kv_sdpa(q, k, v, 16.0, ints(n), num_splits=splits)
        check_rows(got, ref.sdpa(q, k, v, 16.0, [n]), dtype)


@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("kind", ["none", "bool", "type", "f32"])
@pytest.mark.parametrize("seed", range(8))
def test_random_sizes(seed, kind, which):
    """Every key and value at a size of its own, the weights spread over all of them: scores of the same size through the queries' other
    channels, so that small and large values meet in every row."""
    T, n, cap = KERNELS[which]
    B, Hq, Hk, D, dtype = 2, 4, 1, [128, 256][seed % 2], [BF16, F16][seed // 2 % 2]
    far = 30 if dtype == BF16 else 5
    k, v = ([states((B, Hk, cap, D), torch.float32, 10 * seed + i) for i in range(2)])
    size = torch.pow(2.0, (2 * torch.rand(2, B, Hk, cap, 1, generator=gen(seed), device=DEV) - 1) * far)
    # The queries do not look at these channels.  The tcgen05 kernel keeps a key's elements to 2^-39 of its largest one (2^-25 of a
    # unit that puts that one at 2^14): next to 2^20 times larger channels, elements of 2^-6 of their own largest to 2^-39 2^26 = 2^-13.
    # (fp32 products see more only where the queries are 2^-15 times smaller in the large channels, as here.)
    k[..., 64:] *= torch.pow(size[0], 2 / 3)
    v = v * torch.where(torch.rand(B, Hk, cap, 1, generator=gen(seed + 50), device=DEV) < 0.3, size[1], torch.ones_like(size[1]))
    k, v = (qkv.QuantizedKV(*ref.quantise(x.to(dtype))) for x in (k, v))
    q = states((B, Hq, T, D), dtype, 9)
    q[..., 64:] = 0
    keep = torch.rand(B, Hq, 1, cap, generator=gen(seed + 100), device=DEV) < 0.5
    mask = None if kind == "none" else keep if kind == "bool" else torch.where(keep, 0.5, -math.inf).to(dtype if kind == "type" else torch.float32)
    lengths = [n, n - 33]
    got = qkv.quantized_kv_sdpa(q, k, v, 0.125, ints(*lengths), mask, num_splits=[0, 1, 3][seed % 3])
    check_rows(got, ref.sdpa(q, k, v, 0.125, lengths, mask), dtype)


@pytest.mark.parametrize("which", KERNELS)
@pytest.mark.parametrize("octaves", [4, 10, 14, 17, 20])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -8, 2.0 ** -3, 2.0, 2.0 ** 6])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_small_weights_behind_a_large_one(dtype, size, octaves, which):
    """Keys with most of the weight and a value of zero, 63 others behind each 2^-octaves as likely whose values agree: the row is what
    they say.  A rounding of their weights that goes one way does not average out."""
    T, _, _ = KERNELS[which]
    n, D, Hq = 40000, 128, 4
    # Probabilities p take 2^-25 in fp16 at the least: of p 2^6 in the tcgen05 kernel, in the other one of p times the value's scale,
    # itself times 2^8 between 2^-7 and 2^3 and brought beyond 2^10 elsewhere.  Cases where that is more than 2^-9 are left out.
    scaled = 1.3 * size / 15 * 2 ** 8
    if 2.0 ** -25 > 2.0 ** -9 * 2.0 ** (-octaves - 0.45) * (2 ** 6 if which == "many" else scaled if 2 <= scaled < 2 ** 11 else 2 ** 10):
        pytest.skip("below what the kernel's probabilities resolve")
    k, v = qkv.allocate(1, 1, n, D, dtype=dtype)
    large = torch.arange(n, device=DEV) % 64 == 0
    v.codes[:, :, ~large] = 0x2E5D4C7B                    # eight different codes, the same for all keys
    v.scales[:, :, ~large] = size / 15 * 1.3
    v.biases[:, :, ~large] = -size / 3
    # not a power of two apart, and the last bit of fp16's eleven differs from key to key
    far = octaves * math.log(2) + 0.3 + 0.001 * torch.arange(n, device=DEV).remainder(7)
    mask = torch.where(large, 0.0, -far)[None, None, None]
    q = states((1, Hq, T, D), dtype, 9)
    got = qkv.quantized_kv_sdpa(q, k, v, 0.1, ints(n + T), mask, max_length=n).double()
    want = ref.sdpa(q, k, v, 0.1, [n + T], mask)
    # TOL has 2^-9 for the probabilities; half a step of fp16's subnormal outputs on top
    assert bool(((got - want).norm(dim=-1) <= TOL[dtype] * want.norm(dim=-1) + D ** 0.5 * (2.0 ** -25 if dtype == F16 else 0)).all())
