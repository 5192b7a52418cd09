"""Token log-probabilities of logits and temperatures at the ends of their ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from dflash_mlx_b200 import logprobs  # noqa: E402
from tests.test_logprobs_gpu import TYPES, check, ints, logits  # noqa: E402

DEV = "cuda"
T16 = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 9001])
def test_largest_temperatures(V, dtype):
    """Up to 1e38 a row is nearly uniform over what is not hidden; beyond, log2(e) / temperature leaves the normal numbers: refused."""
    x = logits(4, V, dtype, seed=V)
    x[1, 3] = -math.inf
    suppress = torch.zeros(V, dtype=torch.bool, device=DEV)
    suppress[7] = True
    for temperature in (1e30, 1e38):
        check(x, ints(0, 3, 7, V - 1), 4, temperature, suppress)
    for temperature in (1.1e38, 1.3e38, 2.9e38, 3.2e38, 1e39):
        with pytest.raises(ValueError, match="temperature"):
            logprobs.token_logprobs(x, ints(0, 1, 2, 3), temperature=temperature)


# The products' fp32 sums see differences to the row's maximum only, so the bound of check() holds however large the logits are:
# their own spacing is the input's, not the operator's.
@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("V", [100, 9001, 151936])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 2e-5, 1e-3, 130.0])
def test_large_logits(temperature, V, dtype):
    """One token forced by a large logit, rows far from zero on either side, and rows that span the type."""
    most = torch.finfo(dtype).max
    rows = []
    for big in (1e4, 6e4, 1e6, 9.999e9, 1e12, 1e20, 1e30, most):
        if big > most or big / temperature > 1e38:        # not in the type, or the log-probabilities are no fp32 numbers
            continue
        x = logits(3, V, dtype, seed=V)
        x[0, V // 2] = big                                # the others vanish next to it
        x[1] = -big
        x[1, V // 3:V // 3 + 5] = -big / 2
        x[2] = big                                        # ties at a large value
        x[2, ::3] = big / 2
        rows.append(x)
    x = torch.cat(rows)
    check(x, torch.arange(len(x), device=DEV) * 7 % V, min(5, V), temperature)


@pytest.mark.parametrize("dtype", T16)
@pytest.mark.parametrize("V", [100, 30000])
def test_nan_infinity_and_lowest_in_16_bits(V, dtype):
    x = logits(6, V, dtype)
    x[0, V - 1] = math.nan
    x[1, 3] = math.inf
    x[2] = torch.finfo(dtype).min
    x[3, 5] = torch.finfo(dtype).max
    x[4, :50] = torch.finfo(dtype).min
    x[5] = -math.inf
    got = check(x, ints(0, 1, 2, 5, 60, 9), 4)
    assert bool((got.top_ids >= 0).all()) and bool((got.top_ids < V).all())


@pytest.mark.parametrize("dtype", T16)
def test_large_logits_come_late(dtype):
    """A row whose passes take the usual form until a large logit comes, and the other way round."""
    V = 60000
    for R in (1, 200):                                    # several blocks a row; one
        x = logits(2, V, dtype, seed=R)
        x[0, V - 3] = 6e4
        x[1, 2] = 6e4
        x = x.repeat(R, 1)
        tokens = torch.full((2 * R,), V - 3, dtype=torch.int32, device=DEV)
        for temperature in (1.0, 2e-5):
            check(x[:4], tokens[:4], 5, temperature)
            got, one = (logprobs.token_logprobs(y, tokens[:len(y)], top_k=5, temperature=temperature) for y in (x, x[:2]))
            assert torch.equal(got.top_ids[:2], one.top_ids) and bool(got.logprobs.isfinite().all()) and bool(got.entropy.isfinite().all())
