"""The tcgen05 attention kernel over every kind of shape, mask, range and length: each case asserts that it is the one that runs.
It takes more than 16 rows per KV head over long caches; a large bound on the lengths sends short sequences there too."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import quantized_kv as qkv  # noqa: E402
from oracle import quantized_kv as ref  # noqa: E402
from tests.test_quantized_kv_gpu import TOL, TYPES, check_rows, gen, ints, make_cache, no_device_error, states  # noqa: E402, F401
from tests.test_quantized_kv_plan import plan  # noqa: E402

DEV = "cuda"


def bound(B, Hq, Hk, T, at_least=1):
    """The smallest multiple of 100 from `at_least` on that sends these sizes to the tcgen05 kernel, plus an odd rest."""
    n = max(1, -(-at_least // 100)) * 100
    while not plan(B, Hq, Hk, T, n)[0]:
        n += 100
    return n + 13


def run(B, Hq, Hk, D, T, lengths, dtype, *, mask=None, seed=0, num_splits=0, spread=1.0, max_length=None):
    n_max = max_length or bound(B, Hq, Hk, T, max(lengths))
    assert plan(B, Hq, Hk, T, n_max, num_splits)[0]
    k, v = make_cache(B, Hk, n_max + 5, D, dtype, seed, spread)
    q = states((B, Hq, T, D), dtype, seed + 5)
    scale = D ** -0.5 / spread
    got = qkv.quantized_kv_sdpa(q, k, v, scale, ints(*lengths), mask, max_length=n_max, num_splits=num_splits)
    check_rows(got, ref.sdpa(q, k, v, scale, lengths, mask, n_max), dtype)
    return q, k, v, scale, n_max, got


@pytest.mark.parametrize("seed", range(40))
def test_random_shapes(seed):
    r = random.Random(seed)
    dtype, D = r.choice(TYPES), r.choice([128, 256])
    Hk, g = r.choice([1, 2, 3]), r.choice([1, 2, 5, 6, 8])
    T = r.choice([-(-17 // g), r.randint(-(-17 // g), 20 + 17 // g), r.randint(17, 60), r.randint(61, 140)])
    B = max(1, min(r.randint(1, 3), 1200 // (g * Hk * T)))
    n_max = bound(B, g * Hk, Hk, T) + r.randint(0, 300)
    lengths = [r.choice([0, 1, T - 1, T, T + 1, r.randint(0, 400), r.randint(0, 1500), n_max, n_max + 5]) for _ in range(B)]
    mask = None
    if r.random() < 0.6:
        dims = r.choice([(B, 1, 1, n_max), (1, g * Hk, T, n_max), (n_max,), (B, 1, T, 1), (T, n_max)])
        keep = torch.rand(dims, generator=gen(seed), device=DEV) < 0.7
        mask = r.choice([keep, torch.where(keep, torch.randn(dims, generator=gen(seed), device=DEV), -math.inf).to(r.choice([dtype, torch.float32]))])
    run(B, g * Hk, Hk, D, T, lengths, dtype, mask=mask, seed=seed, num_splits=r.choice([0, 0, 1, 3, 50]), max_length=n_max)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 300, 385, 1025])
@pytest.mark.parametrize("T", [9, 40])
def test_lengths(T, n):
    """Lengths below T leave the first rows without a key; ranges that end at every place of a pair of tiles."""
    run(1, 4, 2, 128, T, [n], torch.bfloat16, seed=n, num_splits=1)
    run(2, 4, 1, 128, T, [n, 77], torch.float16, seed=n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,Hq,Hk,D", [(65, 3, 1, 128), (130, 2, 1, 256), (257, 3, 1, 128), (257, 6, 2, 256), (500, 1, 1, 128), (501, 2, 1, 256)])
def test_prompt_chunks(T, Hq, Hk, D, dtype):
    """Chunks of several tiles of 128 rows: alone in the cache, behind a prefix, longer than what is there, empty."""
    for n in (T, T + 777, T - 1, 3):
        run(1, Hq, Hk, D, T, [n], dtype, seed=T)


@pytest.mark.parametrize("kind", ["bool", "type", "f32"])
@pytest.mark.parametrize("shape", ["full", "keys", "heads", "rows"])
def test_masks_of_prompt_chunks(shape, kind):
    B, Hq, Hk, D, T, dtype = 1, 3, 1, 128, 150, torch.bfloat16
    n_max = bound(B, Hq, Hk, T, 700)
    dims = {"full": (B, Hq, T, n_max), "keys": (B, 1, 1, n_max), "heads": (1, Hq, 1, n_max), "rows": (T, n_max)}[shape]
    keep = torch.rand(dims, generator=gen(3), device=DEV) < 0.6
    keep[..., 200:420] = False
    if shape == "full":
        keep[0, 1, 0] = keep[0, 2, 100:] = False
    mask = keep
    if kind != "bool":
        mask = torch.where(keep, torch.randn(dims, generator=gen(4), device=DEV), -math.inf).to(dtype if kind == "type" else torch.float32)
    for n in (700, 150, 333):
        *_, got = run(B, Hq, Hk, D, T, [n], dtype, mask=mask, max_length=n_max)
        if shape == "full":
            assert not bool(got[0, 1, 0].any()) and not bool(got[0, 2, 100:].any())


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 8, 9, 64, 1024])
def test_ranges(splits):
    """Ranges of all kinds of lengths, most of them empty for the shorter sequence; few are joined by one kernel, many by another."""
    run(2, 6, 2, 256, 9, [1900, 17], torch.bfloat16, num_splits=splits)


@pytest.mark.parametrize("kind", ["none", "bool", "f32"])
def test_queries_at_the_ends_of_their_range(kind):
    B, Hq, Hk, D, T, n, dtype = 1, 4, 2, 128, 40, 300, torch.bfloat16
    n_max = bound(B, Hq, Hk, T)
    k, v = make_cache(B, Hk, n_max, D, dtype)
    q = states((B, Hq, T, D), dtype, 3)
    mask = None if kind == "none" else torch.ones(1, Hq, 1, n_max, dtype=torch.bool, device=DEV)
    if kind != "none":
        mask[:, 1, :, 5:200] = False
    if kind == "f32":
        mask = torch.where(mask, 0.25, -math.inf)

    def attend(x, scale):
        return qkv.quantized_kv_sdpa(x, k, v, scale, ints(n), mask, max_length=n_max)

    for scale in (0.0, -0.1, 1e-30):
        check_rows(attend(q, scale), ref.sdpa(q, k, v, scale, [n], mask, n_max), dtype)
    for size in (1e-30, 1e-20, 1e20, 1e30):               # beyond fp16's range on either side
        x, scale = q * size, 0.1 / size
        check_rows(attend(x, scale), ref.sdpa(x, k, v, scale, [n], mask, n_max), dtype)
    mixed = q * torch.pow(10.0, -torch.arange(T, device=DEV).double())[:, None].to(dtype)   # every row at a size of its own
    check_rows(attend(mixed, 0.1), ref.sdpa(mixed, k, v, 0.1, [n], mask, n_max), dtype)
    want = attend(q, 0.1)
    for bad in (math.nan, math.inf):
        x = q.clone()
        x[0, 1, 1, 5] = bad
        got = attend(x, 0.1)
        assert bool(got[0, 1, 1].isnan().all())
        got[0, 1, 1] = want[0, 1, 1]
        assert torch.equal(got, want)


def test_extreme_lengths_and_shared_caches():
    B, Hq, Hk, D, T, dtype = 3, 4, 2, 128, 40, torch.bfloat16
    n_max = bound(B, Hq, Hk, T)
    k, v = make_cache(1, Hk, n_max, D, dtype)
    q = states((B, Hq, T, D), dtype, 3)
    shared = [qkv.QuantizedKV(*[p.expand(B, -1, -1, -1) for p in c]) for c in (k, v)]
    lengths = [-2 ** 31, 2 ** 31 - 1, 50]
    got = qkv.quantized_kv_sdpa(q, *shared, 0.1, ints(*lengths))
    assert not bool(got[0].any())
    check_rows(got, ref.sdpa(q, *shared, 0.1, lengths), dtype)


@pytest.mark.parametrize("D", [128, 256])
def test_slices_and_strides(D):
    B, Hq, Hk, T, dtype = 2, 4, 2, 40, torch.bfloat16
    n_max = bound(B, Hq, Hk, T)
    whole = make_cache(3, 4, n_max + 20, D, dtype)
    k, v = (qkv.QuantizedKV(*[p[1:, 1:3, 8:8 + n_max] for p in c]) for c in whole)
    dense = [qkv.QuantizedKV(*[p.contiguous() for p in c]) for c in (k, v)]
    flat = states((B, T, Hq * D + 8), dtype, 3)
    for start in (0, 3):
        q = flat[..., start:start + Hq * D].view(B, T, Hq, D).transpose(1, 2)
        for n in (61, 500):
            got = qkv.quantized_kv_sdpa(q, k, v, 0.1, ints(n, n // 2))
            assert torch.equal(got, qkv.quantized_kv_sdpa(q.contiguous(), *dense, 0.1, ints(n, n // 2)))
            check_rows(got, ref.sdpa(q, *dense, 0.1, [n, n // 2]), dtype)


def test_lowest_finite_mask():
    B, Hq, Hk, D, T, n, dtype = 1, 2, 1, 128, 40, 70, torch.bfloat16
    n_max = bound(B, Hq, Hk, T)
    mask = torch.full((1, 1, T, n_max), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    mask[0, 0, 1, 20] = 0
    _, _, v, _, _, got = run(B, Hq, Hk, D, T, [n], dtype, mask=mask, max_length=n_max)
    mean = ref.values(*v)[0, 0, :n - T + 1].mean(0)
    assert float((got[0, 0, 0].double() - mean).norm() / mean.norm()) < TOL[dtype]


def test_prompt_verify_rollback_through_the_cache_class():
    """The class bounds the lengths by its capacity; chunks and verify blocks of a large one take the tcgen05 kernel."""
    B, Hq, Hk, D, dtype = 2, 6, 2, 128, torch.bfloat16
    cap = bound(B, Hq, Hk, 16)
    cache = qkv.QuantizedKVCache(B, Hk, cap, D, dtype=dtype)
    dense = [torch.zeros(B, Hk, 512, D, dtype=dtype, device=DEV) for _ in range(2)]
    at = torch.zeros(B, dtype=torch.int32, device=DEV)
    for i, (T, accepted) in enumerate([(90, 90), (137, 137), (16, ints(5, 16)), (16, ints(1, 0)), (16, ints(16, 3)), (1, 1)]):
        assert plan(B, Hq, Hk, T, cap)[0] == (T > 1)
        q, k, v = (states((B, h, T, D), dtype, 3 * i + j) for j, h in enumerate((Hq, Hk, Hk)))
        cache.update(k, v)
        for b in range(B):
            o = int(at[b])
            for d, x in zip(dense, (k, v)):
                d[b, :, o:o + T] = x[b]
        got = cache.attend(q, D ** -0.5)
        check_rows(got, ref.sdpa(q, ref.quantise(dense[0]), ref.quantise(dense[1]), D ** -0.5, (at + T).tolist()), dtype)
        cache.commit(accepted)
        at += accepted
        assert torch.equal(cache.offsets, at)


def test_graphs_and_streams_side_by_side():
    B, Hq, Hk, D, T, dtype = 1, 12, 2, 128, 16, torch.bfloat16
    cap = bound(B, Hq, Hk, T)
    cache = qkv.QuantizedKVCache(B, Hk, cap, D, dtype=dtype)
    cache.keys, cache.values = make_cache(B, Hk, cap, D, dtype)
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
    for at in (5, 1333, cap - T):
        cache.offsets.fill_(at)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            graphs[1][0].replay()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        want = ref.sdpa(q, cache.keys, cache.values, 0.09, [at + T] * B)
        for g, out in graphs:
            check_rows(out, want, dtype)


def test_the_same_bits_every_time():
    for B, Hq, Hk, D, T, n in ((2, 12, 2, 256, 40, 700), (1, 24, 4, 128, 16, 3001), (1, 3, 1, 256, 300, 1300)):
        q, k, v, scale, n_max, first = run(B, Hq, Hk, D, T, [n] * B, torch.bfloat16)
        for _ in range(20):
            assert torch.equal(qkv.quantized_kv_sdpa(q, k, v, scale, ints(*[n] * B), max_length=n_max), first)
