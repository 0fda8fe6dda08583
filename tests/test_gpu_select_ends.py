"""The choice of experts where scores of different logits are equal in 64 bits: against the definition of test_gpu_select,
ids one by one."""
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
