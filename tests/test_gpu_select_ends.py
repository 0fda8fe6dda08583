"""The choice of experts where scores of different logits are equal in 64 bits, and where a bias is no number: against the
definition of test_gpu_select, ids one by one."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.test_gpu_select import agree, rule_of

pytestmark = pytest.mark.gpu

GROUPS = [(1, 1, 1), (8, 3, 1), (8, 3, 2)]


@pytest.mark.parametrize("experts", [24, 96])
@pytest.mark.parametrize("groups,keep,best", GROUPS)
def test_sigmoids_around_the_largest_exponential(ctx, groups, keep, best, experts):
    """exp(-l) passes 64 bits' range at l = -709.7827: scores are 0 from there on and the least subnormal ones before, so
    logits below it are equal however they lie, and those above are not."""
    rng = np.random.default_rng(17)
    tokens = 60
    border = np.float32(-709.7827)
    logits = (-800 - rng.permutation(experts * tokens).reshape(tokens, experts) % 97).astype(np.float32)
    for t in range(tokens):
        at = rng.permutation(experts)[:experts // 4]
        logits[t, at] = border + rng.integers(-140, 0 if t % 2 else 20, experts // 4) * np.float32(2.0 ** -14)
    for renorm in (0, 1):
        agree(ctx, rule_of(experts, 6, 1, groups, keep, best, renorm), logits, rocm.F32, None)


@pytest.mark.parametrize("experts", [24, 96])
@pytest.mark.parametrize("groups,keep,best", GROUPS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", [15, 22, 23, 24, 25, 26, 27, 28, 29, 31, 32, 33, 60, 126])
def test_softmax_of_logits_whose_steps_are_large(ctx, exponent, sign, groups, keep, best, experts):
    """f32 logits of 2^25 lie 4 apart, of 2^32 512: what 746 less than the largest is has no f32 of its own, and which
    scores are 0 is for 64 bits to say."""
    rng = np.random.default_rng(exponent)
    tokens = 60
    most = np.float32(sign * 2.0 ** exponent * 1.25)
    step = float(np.spacing(abs(most)))
    logits = np.empty((tokens, experts), np.float64)
    for t in range(tokens):
        below = np.rint(rng.uniform(746, 2000, experts) / step) + (2 if step > 300 else 0)
        at = rng.permutation(experts)[:5]
        below[at] = np.rint(rng.uniform(600, 760, 5) / step)
        below[at[0]] = 0
        logits[t] = float(most) - below * step
    logits = logits.astype(np.float32)
    for renorm in (0, 1):
        agree(ctx, rule_of(experts, 6, 0, groups, keep, best, renorm), logits, rocm.F32, None)


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.F16, rocm.BF16])
@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("groups,keep,best", GROUPS)
def test_a_bias_that_is_no_number_counts_where_its_expert_does(ctx, groups, keep, best, sigmoid, dtype):
    """A NaN or infinite bias gives a token NaN shares, but not where the expert's logit masks it."""
    rng = np.random.default_rng(23)
    experts, tokens = 96, 30
    logits = rng.standard_normal((tokens, experts)).astype(np.float32)
    logits[::3, 40] = -np.inf
    logits[1::3, [40, 7, 95]] = -np.inf
    logits[4] = -np.inf
    for special in ((np.nan,), (np.inf,), (np.nan, np.inf, np.nan), (np.inf, -np.inf, np.nan)):
        bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
        bias[[40, 7, 95][:len(special)]] = special
        agree(ctx, rule_of(experts, 6, sigmoid, groups, keep, best), logits, dtype, bias)
