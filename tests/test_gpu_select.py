"""The choice of experts from logits against its definition in 64 bits, and the expert layer on a given choice. Ids are
compared one by one; a share is an f32 rounding (half a step, 2^-24 of it) of a quotient of scores that both sides hold
in 64 bits (some 2^-48 apart)."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty, host
from tests.test_gpu_fp8 import DTYPES, _torch, rows_to
from tests.test_gpu_moe import Layer, forward

pytestmark = pytest.mark.gpu


def rule_of(experts, top, sigmoid=0, groups=1, keep=1, best=1, renorm=1, scale=1.0):
    return rocm.MoeSelection(experts=experts, top_k=top, sigmoid=sigmoid, groups=groups, top_groups=keep,
                             group_best=best, renormalize=renorm, scale=scale)


def definition(rule, logits, bias):
    """(ids, shares) of logits [tokens x experts], one token at a time."""
    ids, shares = [], []
    width = rule.experts // rule.groups
    for row in logits.astype(np.float64):
        with np.errstate(all="ignore"):
            if rule.sigmoid:
                s = 1 / (1 + np.exp(-row))
            else:
                s = np.where(row > -np.inf, np.exp(row - row.max()), 0.0)
                s = s / s.sum() if s.sum() > 0 else np.zeros_like(s)
            c = np.where(row == -np.inf, -np.inf, s if bias is None else s + bias.astype(np.float64))
        if np.isnan(row).any() or np.isnan(c).any() or (row == np.inf).any() or (c == np.inf).any():
            ids.append(list(range(rule.top_k)))
            shares.append([np.nan] * rule.top_k)
            continue
        rank = []
        for g in range(rule.groups):
            best = sorted((v for v in c[g * width:(g + 1) * width] if v > -np.inf), reverse=True)[:rule.group_best]
            rank.append(sum(best) if best else -np.inf)
        kept = sorted(range(rule.groups), key=lambda g: (-rank[g], g))[:rule.top_groups]
        among = [e for e in range(rule.experts) if e // width in kept]
        chosen = sorted(among, key=lambda e: (-c[e], e))[:rule.top_k]
        share = s[chosen]
        if rule.renormalize:
            share = share / share.sum() if share.sum() > 0 else np.zeros_like(share)
        ids.append(chosen)
        shares.append(share * float(rule.scale))
    return np.array(ids, np.int32), np.array(shares, np.float64)


def choose(ctx, rule, logits, dtype, bias):
    import torch
    tokens = logits.shape[0]
    ids, shares = empty((tokens, rule.top_k), torch.int32), empty((tokens, rule.top_k), torch.float32)
    ctx.moe_select(rule, logits, dtype, tokens, bias, ids, shares)
    return host(ctx, ids), host(ctx, shares)


def agree(ctx, rule, logits, dtype, bias):
    ld, l = rows_to(logits, dtype)
    ids, shares = choose(ctx, rule, ld, dtype, None if bias is None else dev(bias))
    want_ids, want = definition(rule, l, bias)
    assert np.array_equal(ids, want_ids)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(shares), nan)
    err = np.abs(shares[~nan].astype(np.float64) - want[~nan])
    assert (err <= (2.0 ** -24 + 2.0 ** -40) * np.abs(want[~nan]) + 2.0 ** -149).all()


# tokens, experts, top, groups, kept groups
CASES = [(1, 1, 1, 1, 1), (1, 64, 8, 1, 1), (3, 8, 2, 4, 2), (7, 20, 3, 1, 1), (16, 24, 6, 3, 2), (33, 65, 5, 5, 3),
         (5, 128, 16, 8, 4), (9, 129, 4, 1, 1), (200, 256, 8, 8, 4), (4, 256, 16, 64, 9), (11, 257, 9, 1, 1),
         (6, 512, 16, 16, 3), (3, 504, 1, 63, 1), (2, 16, 16, 1, 1), (5, 12, 2, 12, 5), (4, 512, 8, 2, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sigmoid,biased,best,renorm,scale", [(0, False, 1, 1, 1.0), (1, True, 2, 1, 2.5),
                                                              (0, True, 2, 0, 1.0), (1, False, 1, 0, 0.5)])
@pytest.mark.parametrize("tokens,experts,top,groups,keep", CASES)
def test_choice_against_64_bits(ctx, dtype, tokens, experts, top, groups, keep, sigmoid, biased, best, renorm, scale):
    rng = np.random.default_rng(tokens + experts + top)
    logits = (1.5 * rng.standard_normal((tokens, experts))).astype(np.float32)
    bias = (0.2 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best, renorm, scale), logits, dtype, bias)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
@pytest.mark.parametrize("experts", [16, 100, 200, 400])
def test_equal_logits_go_to_the_lower_index(ctx, experts, groups, keep, best, sigmoid):
    rng = np.random.default_rng(experts)
    logits = rng.integers(-1, 2, (40, experts)).astype(np.float32)
    logits[0] = 0
    logits[1] = -0.0
    logits[1, ::2] = 0.0
    agree(ctx, rule_of(experts, 4, sigmoid, groups, keep, best), logits, rocm.F32, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
def test_masked_experts_and_values_at_the_ends(ctx, dtype, sigmoid, biased, groups, keep, best):
    rng = np.random.default_rng(5)
    experts, top = 96, 6
    lowest = {rocm.F32: -3.4028235e38, rocm.F16: -65504.0, rocm.BF16: -3.3895314e38}[dtype]
    logits = rng.standard_normal((14, experts)).astype(np.float32)
    logits[0] = -np.inf                      # nothing is left
    logits[1, 1:] = -np.inf                  # one expert is
    logits[2, 5:] = -np.inf                  # fewer than top
    logits[3, ::2] = -np.inf
    logits[4] = lowest                       # a mask of the type's lowest value everywhere
    logits[5, 7:] = lowest
    logits[6, 3] = np.nan
    logits[7, 95] = np.inf
    logits[8, :] = 800.0                     # exponentials past 64 bits' range without the maximum
    logits[9, :] = -800.0
    logits[9, 4] = -799.0
    logits[10, 12:24] = -np.inf              # a whole group of eight masked
    logits[11, 1:12] = -np.inf               # a group of one
    logits[12, 0:12] = np.nan
    logits = np.clip(logits, lowest, None, where=~np.isinf(logits), out=logits)
    bias = (3 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best), logits, dtype, bias)
    if biased:
        bias[10], bias[70] = -np.inf, -3.4028235e38
        agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best), logits, dtype, bias)


def test_scores_closer_than_f32_can_tell(ctx):
    """Biased scores 2^-30 apart in both orders: the larger one leads wherever it stands."""
    rng = np.random.default_rng(2)
    experts, tokens = 64, 50
    logits = np.zeros((tokens, experts), np.float32)
    for t in range(tokens):
        logits[t] = rng.permutation(experts) * np.float32(2.0 ** -28)
    for bias in (None, np.full(experts, 0.25, np.float32)):
        for sigmoid in (0, 1):
            agree(ctx, rule_of(experts, 8, sigmoid), logits, rocm.F32, bias)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("bias", [None, 0.0, 0.25, 1000.0])
@pytest.mark.parametrize("experts,top,groups,keep", [(64, 8, 1, 1), (256, 8, 8, 4), (256, 16, 4, 2), (512, 16, 1, 1),
                                                     (40, 5, 10, 3)])
def test_more_candidates_than_fit(ctx, experts, top, groups, keep, bias, sigmoid):
    """Rows whose scores are all equal, nearly equal, or equal but for a few: the lowest indices, or the few."""
    rng = np.random.default_rng(experts + top)
    logits = np.zeros((12, experts), np.float32)
    logits[1] = rng.permutation(experts) * np.float32(2.0 ** -26)
    logits[2, ::3] = 2.0 ** -24
    logits[3, rng.permutation(experts)[:top + 3]] = 1
    logits[4, experts // 2:] = -1
    logits[5] = 3
    logits[6] = -20 + rng.permutation(experts) * np.float32(2.0 ** -19)
    logits[7:] = rng.integers(-2, 3, (5, experts)) * np.float32(0.5)
    b = None if bias is None else np.full(experts, bias, np.float32)
    for best in (1, 2):
        agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best), logits, rocm.F32, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
def test_scores_that_64_bits_cannot_tell_apart(ctx, dtype, biased, groups, keep, best):
    """A sigmoid's logits where it is 1, or 0, to 64 bits or nearly so; a softmax's far below the largest."""
    rng = np.random.default_rng(11)
    experts, top = 96, 6
    logits = rng.standard_normal((12, experts)).astype(np.float32)
    logits[0] = 40 + rng.permutation(experts)                   # all 1
    logits[1] = rng.uniform(16, 40, experts)
    logits[2, 50:] = rng.uniform(15, 38, experts - 50)
    logits[3] = -rng.uniform(690, 720, experts)                 # the smallest scores, and 0
    logits[4] = -rng.uniform(700, 760, experts)
    logits[4, 20] = 0
    logits[5] = -1000 - rng.permutation(experts)
    logits[6] = -rng.uniform(600, 800, experts)
    logits[6, 90] = 0
    logits[7, 3:] = -2000                                       # a mask by a large number
    logits[8] = rng.uniform(-60, 60, experts)
    logits[9] = np.where(np.arange(experts) % 2, -710.0, -709.5)
    logits[10, ::2] = 16.5
    logits[11, 1:] = -745.5
    bias = (0.01 * rng.standard_normal(experts)).astype(np.float32) if biased else None
    for sigmoid in (0, 1):
        for renorm in (0, 1):
            agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best, renorm), logits, dtype, bias)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts,groups", [(64, 8), (240, 10), (256, 64), (512, 16)])
def test_groups_closer_than_f32_can_tell(ctx, experts, groups, biased, sigmoid):
    """The same values in every group but for 2^-26 here and there: the sums' order is decided far below f32."""
    rng = np.random.default_rng(experts)
    width = experts // groups
    logits = np.zeros((30, experts), np.float32)
    for t in range(30):
        row = np.tile(np.sort(rng.standard_normal(width)).astype(np.float32) * np.float32(0.25), groups)
        at = rng.integers(0, experts, groups)
        row[at] += np.float32(2.0 ** -22) * rng.integers(-2, 3, groups).astype(np.float32)
        logits[t] = row
    bias = np.tile((0.1 * rng.standard_normal(width)).astype(np.float32), groups) if biased else None
    for keep in (1, groups // 2):
        top = min(4, keep * width)
        for best in (1, 2):
            agree(ctx, rule_of(experts, top, sigmoid, groups, keep, best), logits, rocm.F32, bias)


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
@pytest.mark.parametrize("most", [None, 3.0])
def test_logits_so_near_0_that_their_scores_are_equal(ctx, most, groups, keep, best, biased, sigmoid, dtype):
    """exp of any of these is 1, or exp(-most): equal scores, so the lower index."""
    rng = np.random.default_rng(11)
    tokens, experts = 40, 96
    logits = rng.choice(np.array([0, -0.0, 1e-20, -1e-20, 3e-30, -2e-25, 1e-36], np.float32), (tokens, experts))
    logits[::2, ::3] = rng.standard_normal((tokens // 2, experts // 3)) - 2.0
    if most is not None:
        logits[:, 70] = most
    bias = np.zeros(experts, np.float32) if biased else None
    agree(ctx, rule_of(experts, 6, sigmoid, groups, keep, best), logits, dtype, bias)


@pytest.mark.parametrize("sigmoid", [0, 1])
@pytest.mark.parametrize("size", [1e3, 1e6])
@pytest.mark.parametrize("groups", [4, 32])
def test_groups_whose_biases_cancel(ctx, groups, size, sigmoid):
    """A group's two largest are some `size` and -`size`: in f32 each is off by the size's rounding, far more than what the
    sums of scores differ by. In 64 bits the sums are those of two roundings to some 1e-10."""
    rng = np.random.default_rng(groups)
    width = 8
    logits = rng.standard_normal((700, groups * width)).astype(np.float32)
    bias = np.tile(np.array([size, -size] + [-4 * size] * (width - 2), np.float32), groups)
    agree(ctx, rule_of(groups * width, 2, sigmoid, groups, groups // 4, 2), logits, rocm.F32, bias)


def test_many_tokens(ctx):
    rng = np.random.default_rng(3)
    logits = (1.5 * rng.standard_normal((3001, 160))).astype(np.float32)
    bias = (0.1 * rng.standard_normal(160)).astype(np.float32)
    agree(ctx, rule_of(160, 6, 1, 8, 3, 2, 1, 16.0), logits, rocm.F32, bias)


def test_bytes_around_the_outputs_left_alone(ctx):
    import torch
    rng = np.random.default_rng(4)
    tokens, experts, top = 13, 40, 5
    logits = torch.zeros(tokens * experts + 1, dtype=torch.bfloat16, device="cuda")[1:].view(tokens, experts)
    logits.copy_(torch.from_numpy(rng.standard_normal((tokens, experts)).astype(np.float32)))
    ids = torch.full((tokens * top + 8,), 77, dtype=torch.int32, device="cuda")
    shares = torch.full((tokens * top + 8,), 7.0, device="cuda")
    torch.cuda.synchronize()
    rule = rule_of(experts, top, 0, 4, 2)
    ctx.moe_select(rule, logits, rocm.BF16, tokens, None, ids[4:], shares[4:])
    got = host(ctx, ids)
    want, _ = definition(rule, logits.float().cpu().numpy(), None)
    assert np.array_equal(got[4:-4].reshape(tokens, top), want)
    for t, v in ((ids, 77), (shares, 7)):
        assert (t[:4] == v).all() and (t[-4:] == v).all()


def test_refusals(ctx):
    import torch
    logits = torch.zeros(4, 16, device="cuda")
    ids, shares = empty((4, 16), torch.int32), empty((4, 16), torch.float32)

    def refused(code, rule, *args):
        with pytest.raises(rocm.DzError) as e:
            ctx.moe_select(rule, *args)
        assert e.value.code == code, args

    good = dict(experts=16, top=2, groups=4, keep=2)
    for change in (dict(experts=0), dict(experts=513, groups=1, keep=1), dict(top=0), dict(top=17), dict(top=9),
                   dict(groups=0), dict(groups=5), dict(experts=130, groups=65), dict(keep=0), dict(keep=5),
                   dict(best=0), dict(best=3), dict(sigmoid=2), dict(renorm=-1), dict(scale=float("inf")),
                   dict(scale=float("nan"))):
        refused("INVALID_PARAMETERS", rule_of(**{**good, **change}), logits, rocm.F32, 4, None, ids, shares)
    rule = rule_of(**good)
    refused("INVALID_PARAMETERS", rule, logits, 3, 4, None, ids, shares)
    refused("INVALID_REQUEST", rule, None, rocm.F32, 4, None, ids, shares)
    refused("INVALID_REQUEST", rule, logits, rocm.F32, 4, None, None, shares)
    refused("INVALID_REQUEST", rule, logits, rocm.F32, 4, None, ids, None)
    refused("INPUT_TOO_LONG", rule, logits, rocm.F32, (1 << 24) + 1, None, ids, shares)
    ctx.moe_select(rule, None, rocm.F32, 0, None, None, None)


# ---- the expert layer on a choice -------------------------------------------------

LAYERS = [(1, 8, 2, 300, 129), (5, 24, 3, 260, 200), (13, 24, 3, 1000, 70), (16, 128, 8, 130, 300), (40, 6, 4, 384, 100),
          (128, 20, 2, 129, 40), (7, 16, 16, 200, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts,top,hidden,ff", LAYERS)
def test_the_layer_on_its_own_choice_gives_its_own_bits(ctx, tokens, experts, top, hidden, ff, dtype):
    import torch
    rng = np.random.default_rng(tokens + hidden)
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    xd, _ = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    ids, shares = empty((tokens, top), torch.int32), empty((tokens, top), torch.float32)
    layer.moe.route(xd, dtype, tokens, ids, shares)
    y = empty((tokens, hidden), _torch(dtype))
    layer.moe.forward_selected(xd, dtype, tokens, ids, shares, y)
    ctx.sync()
    assert torch.equal(y, forward(ctx, layer, xd, dtype, tokens, hidden))
    # the router's logits, and the plain rule on them
    logits = empty((tokens, experts), torch.float32)
    layer.moe.logits(xd, dtype, tokens, logits)
    got_ids, got = choose(ctx, rule_of(experts, top), logits, rocm.F32, None)
    assert np.array_equal(got_ids, host(ctx, ids))
    assert np.allclose(got, host(ctx, shares), rtol=16 * 2.0 ** -24, atol=0)
    layer.moe.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 6, 20, 128])
def test_a_choice_by_another_rule_against_64_bits(ctx, tokens, dtype):
    """Norm-free: logits, the sigmoid rule with bias and groups, the experts; the layer's shares are the rule's."""
    import torch
    rng = np.random.default_rng(tokens)
    experts, top, hidden, ff = 12, 3, 200, 90
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    xd, x = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    rule = rule_of(experts, top, 1, 4, 2, 2, 1, 2.5)
    logits = empty((tokens, experts), torch.float32)
    layer.moe.logits(xd, dtype, tokens, logits)
    ids, shares = empty((tokens, top), torch.int32), empty((tokens, top), torch.float32)
    ctx.moe_select(rule, logits, rocm.F32, tokens, dev(bias), ids, shares)
    y = empty((tokens, hidden), _torch(dtype))
    layer.moe.forward_selected(xd, dtype, tokens, ids, shares, y)
    ctx.sync()
    picked, share = host(ctx, ids), host(ctx, shares).astype(np.float64)
    want_ids, want_shares = definition(rule, host(ctx, logits), bias)
    assert np.array_equal(picked, want_ids)
    layer.route = lambda _: (picked, share, np.zeros_like(share))
    want, tol = layer(x.astype(np.float64), dtype)
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err / tol).max()
    layer.moe.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [2, 9, 30, 128])
def test_choices_that_no_layer_has_give_nan_and_touch_no_other_token(ctx, tokens, dtype):
    import torch
    rng = np.random.default_rng(tokens)
    experts, top, hidden, ff = 10, 4, 300, 130
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    xd, x = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    picked = np.stack([rng.permutation(experts)[:top] for _ in range(tokens)]).astype(np.int32)
    share = rng.random((tokens, top)).astype(np.float32)
    right = empty((tokens, hidden), _torch(dtype))
    layer.moe.forward_selected(xd, dtype, tokens, dev(picked), dev(share), right)
    ctx.sync()
    layer.route = lambda _: (picked, share.astype(np.float64), np.zeros(share.shape))
    want, tol = layer(x.astype(np.float64), dtype)
    assert (np.abs(right.double().cpu().numpy() - want) <= tol).all()
    wrong = picked.copy()
    bad = {0: (top - 1, experts), tokens // 2: (0, -1), tokens - 1: (top - 1, wrong[tokens - 1, 0])}
    for t, (i, e) in bad.items():
        wrong[t, i] = e
    for extreme in (-(1 << 31), (1 << 31) - 1, None):
        if extreme is not None:
            wrong[0, top - 1] = extreme
        else:
            wrong[:] = picked
            wrong[0] = wrong[0, 0]
            bad = {0: 0}
        y = empty((tokens, hidden), _torch(dtype))
        layer.moe.forward_selected(xd, dtype, tokens, dev(wrong), dev(share), y)
        ctx.sync()
        rows = list(bad)
        assert torch.isnan(y[rows]).all()
        others = [t for t in range(tokens) if t not in bad]
        err = np.abs(y.double().cpu().numpy() - want)
        assert (err <= tol)[others].all()
    layer.moe.free()


def test_every_token_the_same_experts(ctx):
    import torch
    rng = np.random.default_rng(1)
    tokens, experts, top, hidden, ff = 128, 9, 3, 200, 70
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    xd, x = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), rocm.F32)
    picked = np.tile(np.array([8, 0, 4], np.int32), (tokens, 1))
    share = rng.random((tokens, top)).astype(np.float32)
    y = empty((tokens, hidden), torch.float32)
    layer.moe.forward_selected(xd, rocm.F32, tokens, dev(picked), dev(share), y)
    ctx.sync()
    layer.route = lambda _: (picked, share.astype(np.float64), np.zeros(share.shape))
    want, tol = layer(x.astype(np.float64), rocm.F32)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    layer.moe.free()


def test_selected_refusals(ctx):
    import torch
    layer = Layer(ctx, np.random.default_rng(0), 4, 2, 64, 32, 1)
    x, y = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 64, device="cuda")
    ids, shares = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, device="cuda")
    torch.cuda.synchronize()
    calls = [("INVALID_REQUEST", (None, rocm.F32, 2, ids, shares, y)), ("INVALID_REQUEST", (x, rocm.F32, 2, None, shares, y)),
             ("INVALID_REQUEST", (x, rocm.F32, 2, ids, None, y)), ("INVALID_REQUEST", (x, rocm.F32, 2, ids, shares, None)),
             ("INVALID_PARAMETERS", (x, 4, 2, ids, shares, y)), ("INPUT_TOO_LONG", (x, rocm.F32, 129, ids, shares, y))]
    for code, args in calls:
        with pytest.raises(rocm.DzError) as e:
            layer.moe.forward_selected(*args)
        assert e.value.code == code
    with pytest.raises(rocm.DzError):
        layer.moe.logits(x, rocm.F32, 2, None)
    layer.moe.forward_selected(None, rocm.F32, 0, None, None, None)
    layer.moe.logits(None, rocm.F32, 0, None)
    layer.moe.free()


@pytest.mark.parametrize("tokens", [3, 40])
def test_a_decoder_layer_s_entry_captured_and_replayed(ctx, tokens):
    """Norm with the residual, logits, the choice, the experts in one recording: every replay gives the eager bits."""
    import torch
    rng = np.random.default_rng(31)
    experts, top, hidden, ff = 16, 4, 520, 130
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    rule = rule_of(experts, top, 1, 4, 2, 2)
    bias, w = dev((0.1 * rng.standard_normal(experts)).astype(np.float32)), dev(np.ones(hidden, np.float32))
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        bf = torch.bfloat16
        x, r, h, normed, out, eager = (empty((tokens, hidden), bf) for _ in range(6))
        q, s = empty((tokens, 640), torch.uint8), empty((5, tokens), torch.float32)
        logits = empty((tokens, experts), torch.float32)
        ids, shares = empty((tokens, top), torch.int32), empty((tokens, top), torch.float32)

        def fill():
            for t in (x, r):
                t.copy_(torch.from_numpy(rng.standard_normal((tokens, hidden)).astype(np.float32)))
            torch.cuda.synchronize()

        def run(y):
            ctx.add_rmsnorm_fp8(x, r, rocm.BF16, tokens, hidden, w, 1e-6, h, q, s, y=normed, zero_centered=False)
            layer.moe.logits(normed, rocm.BF16, tokens, logits)
            ctx.moe_select(rule, logits, rocm.F32, tokens, bias, ids, shares)
            layer.moe.forward_selected(normed, rocm.BF16, tokens, ids, shares, y)

        fill()
        run(out)
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with rocm.capture(graph, stream):
            run(out)
            capture = ctx.capture_id()
        for i in range(4):
            fill()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            run(eager)
            ctx.sync()
            assert out.abs().max() > 0 and torch.equal(out, eager), i
        del graph
        ctx.capture_release(capture)
    finally:
        ctx.set_stream(None)
    layer.moe.free()
