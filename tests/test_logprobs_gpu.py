"""Token log-probabilities on the GPU against the 64-bit oracle."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import logprobs  # noqa: E402
from oracle import logprobs as ref  # noqa: E402

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits(R, V, dtype, seed=0, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(R, V, generator=g, device=DEV)).to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check(x, tokens, top_k=0, temperature=1.0, suppress=None):
    got = logprobs.token_logprobs(x, tokens, top_k=top_k, temperature=temperature, suppress=suppress)
    lp, ent, tops, ids = ref.token_logprobs(x, tokens.cpu(), top_k, temperature, suppress)
    # fp32 sums of terms that carry 2^-22 of exp2 and as much of its argument's rounding (|argument| 2^-24, at most 40 octaves
    # matter): 5e-6 of L and of W at most, next to |value| 2^-24 of the output; the entropy's difference of ln L and W / (L T)
    # is of the size of the largest distance that still counts, 40 octaves * ln 2 = 28
    size = 5e-6
    for a, b, more in ((got.logprobs, lp, 1.0), (got.entropy, ent, 28.0), (got.top_logprobs, tops, 1.0)):
        a = a.cpu().double()
        assert a.shape == b.shape
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        fine = b.isfinite()
        assert bool(((a - b)[fine].abs() <= size * more + 2.0 ** -23 * b[fine].abs()).all()), float((a - b)[fine].abs().max())
    if not bool(x.isnan().any()):
        assert torch.equal(got.top_ids.cpu().long(), ids)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (2, 31, 20), (5, 257, 5), (1, 4097, 32), (7, 20481, 1), (2, 50001, 20), (3, 151936, 20),
                                   (1, 400003, 7)])
def test_shapes(R, V, k, dtype):
    x = logits(R, V, dtype, seed=V)
    check(x, torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV), k)


@pytest.mark.parametrize("R", [16, 40, 333])
def test_rows(R):
    x = logits(R, 5000, torch.bfloat16, seed=R)
    check(x, torch.arange(R, device=DEV) * 7, 10, 0.7)


@pytest.mark.parametrize("temperature", [1e-3, 0.5, 1.7, 50.0])
def test_temperature(temperature):
    check(logits(3, 3001, torch.float32), ints(0, 5, 3000), 8, temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [20, 1500, 70000])
def test_ties_go_to_the_lowest_index(V, dtype):
    k = 20
    x = torch.zeros(4, V, dtype=dtype, device=DEV)
    x[1] = -0.0                                           # one value with the other zero
    x[1, ::2] = 0.0
    x[2, V // 2:] = 1.0
    x[3] = torch.arange(V, device=DEV) // 3 % 2           # two values in turn
    check(x, ints(0, 1, V - 1, 2), k)


@pytest.mark.parametrize("V", [3000, 152000])
def test_sorted_logits(V):
    x = torch.stack([torch.linspace(9, -9, V, device=DEV), torch.linspace(-9, 9, V, device=DEV)])
    check(x, ints(0, V - 1), 32)


@pytest.mark.parametrize("V", [40, 9000, 152000])
def test_suppressed_and_hidden(V):
    x = logits(4, V, torch.bfloat16)
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 3] = 1.0
    suppress = torch.zeros(V, dtype=torch.bool, device=DEV)
    suppress[x[0].topk(5).indices] = True
    suppress[0] = True
    got = check(x, ints(0, 2, 3, 1), 12, suppress=suppress)
    assert float(got.logprobs[0]) == -math.inf and float(got.logprobs[1]) == -math.inf and float(got.entropy[1]) == 0
    assert float(got.logprobs[2]) == 0
    few = torch.ones(V, dtype=torch.bool, device=DEV)     # a grammar that allows three tokens
    few[[1, 7, V - 1]] = False
    check(x, ints(1, 7, 1, V - 1), 12, suppress=few)
    check(x, ints(1, 7, 1, V - 1), 12, suppress=torch.ones(V, dtype=torch.bool, device=DEV))


@pytest.mark.parametrize("seed", range(12))
def test_random_shapes(seed):
    import random
    r = random.Random(seed)
    V = int(2 ** r.uniform(1, 17.3))
    R = r.choice([1, 3, 17, 200 if V < 20000 else 5])
    k = r.randint(0, min(32, V))
    x = logits(R, V, r.choice(TYPES), seed, r.choice([0.1, 2.0, 20.0]))
    suppress = (torch.rand(V, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) < 0.3) if r.random() < 0.5 else None
    tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(seed)).to(DEV)
    check(x, tokens, k, r.choice([1.0, 0.3, 3.0, 400.0]), suppress)


@pytest.mark.parametrize("ascending", [False, True])
def test_rows_that_beat_themselves_again_and_again(ascending):
    """Many rows, one block each, whose later elements keep beating the earlier ones: the list of candidates overflows."""
    x = torch.linspace(-9, 9, 60000, device=DEV).expand(200, -1).contiguous()
    x = x if ascending else x.flip(1).contiguous()
    check(x[:3].repeat(60, 1)[:160], torch.arange(160, device=DEV), 20)


@pytest.mark.parametrize("V", [100, 30000])
def test_nan_infinity_and_lowest(V):
    x = logits(5, V, torch.float32)
    x[0, V - 1] = math.nan
    x[1, 3] = math.inf
    x[2] = torch.finfo(torch.float32).min
    x[3, 5] = torch.finfo(torch.float32).max
    x[4, :50] = torch.finfo(torch.float32).min
    got = check(x, ints(0, 1, 2, 5, 60), 4)
    assert bool((got.top_ids >= 0).all()) and bool((got.top_ids < V).all())


def test_tokens_outside_and_types():
    x = logits(4, 100, torch.float16)
    got = logprobs.token_logprobs(x, ints(-1, 100, -100, 99))
    assert got.logprobs[:3].isnan().all() and bool(got.logprobs[3].isfinite()) and got.top_ids.shape == (4, 0)
    far = torch.tensor([2 ** 32, -2 ** 32 + 5, 99, 7], device=DEV)          # int64 that would wrap into the vocabulary
    got = logprobs.token_logprobs(x, far)
    assert got.logprobs[:2].isnan().all() and bool(got.logprobs[2:].isfinite().all())
    check(x, torch.tensor([1, 2, 3, 4], device=DEV), 3)


def test_layouts():
    x = logits(6, 1003, torch.bfloat16)
    tokens = torch.arange(6, device=DEV)
    want = logprobs.token_logprobs(x, tokens, top_k=5)
    for y in (x.view(2, 3, 1003), torch.nn.functional.pad(x, (3, 2))[:, 3:-2], x.t().contiguous().t()):
        got = logprobs.token_logprobs(y, tokens.view(y.shape[:-1]), top_k=5)
        # odd rows start at every alignment, which moves the shares of the sums: fp32 rounding
        assert torch.equal(got.top_ids.reshape(want.top_ids.shape), want.top_ids)
        for a, b in zip(got[:3], want[:3]):
            assert float((a.reshape(b.shape) - b).abs().max()) < 1e-5
    one = logprobs.token_logprobs(x[2], tokens[2], top_k=5)
    assert one.logprobs.shape == () and torch.equal(one.top_ids, want.top_ids[2])
    assert logprobs.token_logprobs(x[:0], tokens[:0], top_k=2).top_ids.shape == (0, 2)
    same = logprobs.token_logprobs(x[:1].expand(4, -1), tokens[:4], top_k=5)
    assert torch.equal(same.top_ids, want.top_ids[:1].expand(4, -1))


def test_refusals():
    x, t = logits(2, 100, torch.float32), ints(0, 0)
    for bad in (dict(top_k=33), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(suppress=torch.zeros(99, dtype=torch.bool, device=DEV)), dict(suppress=torch.zeros(100, device=DEV))):
        with pytest.raises(ValueError):
            logprobs.token_logprobs(x, t, **bad)
    for logits_bad, tokens_bad in ((x.double(), t), (x, t[:1]), (x, t.float()), (x[:, :0], t), (x[:, :3], t)):
        with pytest.raises(ValueError):
            logprobs.token_logprobs(logits_bad, tokens_bad, top_k=4)


def test_streams_and_graphs():
    x = logits(16, 151936, torch.bfloat16)
    tokens = torch.arange(16, dtype=torch.int32, device=DEV)
    want = logprobs.token_logprobs(x, tokens, top_k=20)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logprobs.token_logprobs(x, tokens, top_k=20)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        got = logprobs.token_logprobs(x, tokens, top_k=20)
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    y = logits(16, 151936, torch.bfloat16, 5)
    x.copy_(y)
    g.replay()
    for a, b in zip(got, logprobs.token_logprobs(y, tokens, top_k=20)):
        assert torch.equal(a, b)
