"""The mixture-of-experts layer over many 128-blocks of both widths, so that every LDS stage is filled, read and
filled again, in each of its kernels' forms; routers of each type; and values up to the ends of f32. Tolerances as in
test_gpu_moe."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import DTYPES, VALUES, _torch, f64, make_weight, rows_to, spread
from tests.test_gpu_moe import Layer, forward

pytestmark = pytest.mark.gpu

# tokens, experts, top, hidden, ff, and experts that most tokens go to. Above 16 tokens: 16 rows at a time up to 12
# rows an expert on average, else 32; more rows of one expert than that read its weight again.
WIDE = [(20, 6, 2, 1300, 1190, ()), (40, 8, 2, 1300, 1190, (5, 2)), (40, 3, 2, 1157, 1300, ()),
        (70, 2, 2, 1300, 1157, ()), (128, 5, 1, 1290, 1100, (3,))]
# up to 16 tokens: workgroups over several tiles of ff with uneven shares of hidden; batches of a long ff
FEW = [(16, 32, 4, 1300, 600, ()), (1, 2, 1, 100, 40000, ()), (15, 1, 1, 130, 5000, ()), (7, 2, 1, 260, 9000, ()),
       (2, 3, 2, 2100, 2200, ())]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts,top,hidden,ff,favoured", WIDE + FEW)
def test_many_blocks_against_64_bits(ctx, tokens, experts, top, hidden, ff, favoured, dtype):
    import torch
    rng = np.random.default_rng(tokens + experts + hidden)
    router = (rng.standard_normal((experts, hidden)) / np.sqrt(hidden)).astype(np.float32)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    for i, e in enumerate(favoured):
        router[e, 0] = 6 - i
    if favoured:
        x[:, 0] = 1 + np.abs(x[:, 0])
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1, router=router)
    xd, xf = rows_to(x, dtype)
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    want, tol = layer(xf.astype(np.float64), dtype)
    if favoured:
        ids = layer.route(xf.astype(np.float64))[0]
        assert max(np.bincount(ids.ravel())) > 32
    err = np.abs(f64(y) - want)
    assert (err <= tol).all(), (err / tol).max()
    assert torch.equal(y, forward(ctx, layer, xd, dtype, tokens, hidden))
    layer.moe.free()


@pytest.mark.parametrize("router_dtype", [rocm.F16, rocm.BF16])
def test_a_16_bit_router_is_the_f32_one_of_its_values(ctx, router_dtype):
    import torch
    rng = np.random.default_rng(router_dtype)
    tokens, experts, top, hidden, ff = 9, 21, 4, 203, 90
    parts = {}
    for name, (n, k) in dict(gate=(ff, hidden), up=(ff, hidden), down=(hidden, ff)).items():
        made = [make_weight(rng, n, k) for _ in range(experts)]
        parts[name] = dev(np.stack([c for c, _ in made])), dev(np.stack([s for _, s in made]) / np.float32(np.sqrt(k)))
    rd, rf = rows_to((rng.standard_normal((experts, hidden)) / np.sqrt(hidden)).astype(np.float32), router_dtype)
    room = torch.zeros(experts * hidden + 1, dtype=rd.dtype, device="cuda")
    room[1:] = rd.flatten()  # at an odd address
    torch.cuda.synchronize()
    cfg = rocm.MoeConfig(experts=experts, top_k=top, hidden=hidden, ff=ff, renormalize=1)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    xd = dev(x)
    outs = []
    for router, dtype in ((dev(rf), rocm.F32), (room[1:], router_dtype)):
        moe = ctx.moe(cfg, router, dtype, parts["gate"], parts["up"], parts["down"])
        ids, shares = empty((tokens, top), torch.int32), empty((tokens, top), torch.float32)
        y = empty((tokens, hidden), torch.float32)
        moe.route(xd, rocm.F32, tokens, ids, shares)
        moe.forward(xd, rocm.F32, tokens, y)
        ctx.sync()
        outs.append((ids, shares, y))
        moe.free()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    logits = x.astype(np.float64) @ rf.astype(np.float64).T
    assert np.array_equal(outs[0][0].cpu().numpy(), np.argsort(-logits, axis=1, kind="stable")[:, :top])
    bad = room.clone()
    bad[-1] = float("inf")
    torch.cuda.synchronize()
    with pytest.raises(rocm.DzError) as e:
        ctx.moe(cfg, bad[1:], router_dtype, parts["gate"], parts["up"], parts["down"])
    assert e.value.code == "INVALID_CHECKPOINT"


class Scaled(Layer):
    """A layer of equal logits whose block scales are around `scales` of its projections."""

    def __init__(self, ctx, rng, experts, top, hidden, ff, **scales):
        self.shape = experts, top, hidden, ff, 1
        self.router = np.zeros((experts, hidden), np.float32)
        held, self.wide = {}, {}
        for name, (n, k) in dict(gate=(ff, hidden), up=(ff, hidden), down=(hidden, ff)).items():
            made = [make_weight(rng, n, k) for _ in range(experts)]
            codes = np.stack([c for c, _ in made])
            s = (np.stack([s for _, s in made]).astype(np.float64) * (scales[name] / 0.006)).astype(np.float32)
            assert (s > 2.0 ** -126).all() and np.isfinite(s).all()
            self.wide[name] = [VALUES[c] * spread(b, *c.shape) for c, b in zip(codes, s)]
            held[name] = dev(codes), dev(s)
        cfg = rocm.MoeConfig(experts=experts, top_k=top, hidden=hidden, ff=ff, renormalize=1)
        self.moe = ctx.moe(cfg, dev(self.router), rocm.F32, held["gate"], held["up"], held["down"])


LARGEST = {rocm.F32: 5.9e33, rocm.F16: 65504.0, rocm.BF16: 5.9e33}  # 128 * 448 of them stay in f32


@pytest.mark.parametrize("tokens", [3, 20])
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_up_to_the_documented_range(ctx, dtype, tokens):
    """Rows of the largest values that a layer takes, every one of them compared."""
    rng = np.random.default_rng(60 + dtype)
    hidden, ff = 300, 140
    x = rng.choice([-1.0, 1.0], (tokens, hidden)).astype(np.float32) * np.float32(LARGEST[dtype])
    x[1] *= rng.random(hidden).astype(np.float32)
    xd, xf = rows_to(x, dtype)
    assert np.isfinite(xf).all() and np.abs(xf).max() > 0.99 * LARGEST[dtype]
    scale = 1 / (LARGEST[dtype] * 100 * np.sqrt(hidden))
    layer = Scaled(ctx, rng, 4, 2, hidden, ff, gate=scale, up=scale, down=1e-3)
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    want, tol = layer(xf.astype(np.float64), dtype)
    assert 1e-3 < np.abs(want).max() < 6e4
    assert (np.abs(f64(y) - want) <= tol).all()
    layer.moe.free()


@pytest.mark.parametrize("tokens", [3, 20])
@pytest.mark.parametrize("dtype", DTYPES)
def test_h_up_to_the_documented_range(ctx, dtype, tokens):
    """silu(gate) up of 1e33 comes out as the definition has it."""
    rng = np.random.default_rng(70 + dtype)
    hidden, ff = 140, 300
    xd, xf = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    layer = Scaled(ctx, rng, 4, 2, hidden, ff, gate=1e13, up=1e13, down=1e-35)
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    with np.errstate(over="ignore"):
        want, tol = layer(xf.astype(np.float64), dtype)
        e = layer.route(xf.astype(np.float64))[0][0, 0]
        a, b = layer.wide["gate"][e] @ xf[0].astype(np.float64), layer.wide["up"][e] @ xf[0].astype(np.float64)
        assert 1e31 < np.abs(a / (1 + np.exp(-a)) * b).max() < 5.9e33
    assert 1e-3 < np.abs(want).max() < 6e4
    assert (np.abs(f64(y) - want) <= tol).all()
    layer.moe.free()


@pytest.mark.parametrize("tokens", [3, 20])
@pytest.mark.parametrize("dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("exponent", [-109, -126, -132])
def test_activations_down_to_the_documented_steps(ctx, exponent, dtype, tokens):
    """x, then h, of 2^exponent to 2^(exponent + 1): off by half a step of 2^-133 more than other activations."""
    rng = np.random.default_rng(90 + dtype)
    hidden, ff, size = 300, 140, 2.0 ** exponent
    x = rng.choice([-1.0, 1.0], (tokens, hidden)) * (1 + rng.random((tokens, hidden)))
    xd, xf = rows_to((x * size).astype(np.float32), dtype)
    scale = 1 / (size * 100 * np.sqrt(hidden))
    layer = Scaled(ctx, rng, 4, 2, hidden, ff, gate=scale, up=scale, down=1e-3)
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    rows = xf.astype(np.float64)
    want, tol = layer(rows, dtype)
    assert 1e-3 < np.abs(want).max() < 6e4
    assert (np.abs(f64(y) - want) <= tol + stepped(layer, rows, dtype, 2.0 ** -134)[0]).all()
    layer.moe.free()

    xd, xf = rows_to(x.astype(np.float32), dtype)
    scale = np.sqrt(size) / (100 * np.sqrt(hidden))
    layer = Scaled(ctx, rng, 4, 2, hidden, ff, gate=scale, up=scale, down=1e-3 / size)
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    rows = xf.astype(np.float64)
    want, tol = layer(rows, dtype)
    assert 1e-3 < np.abs(want).max() < 6e4
    assert (np.abs(f64(y) - want) <= tol + stepped(layer, rows, dtype, 2.0 ** -134)[1]).all()
    layer.moe.free()


def stepped(layer, x, dtype, off):
    """What y may move by where each value of x, or of h, is `off`: silu(a') b' - silu(a) b is at most
    1.1 |a' - a| |b'| + |a| |b' - b|, since silu's slope is below 1.1; and 1% for the roundings of what moved."""
    ids, c, _ = layer.route(x)
    of_x, of_h = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(x.shape[0]):
        for e, share in zip(ids[t], c[t]):
            g, u, d = (layer.wide[p][e] for p in ("gate", "up", "down"))
            a, b, da, db = g @ x[t], u @ x[t], np.abs(g).sum(1) * off, np.abs(u).sum(1) * off
            of_x[t] += share * (np.abs(d) @ (1.1 * da * (np.abs(b) + db) + np.abs(a) * db))
            of_h[t] += share * np.abs(d).sum(1) * off
    return 1.01 * of_x, 1.01 * of_h


@pytest.mark.parametrize("tokens", [3, 20])
@pytest.mark.parametrize("dtype", [rocm.F32, rocm.BF16])
def test_a_token_past_f32_s_range_touches_no_other(ctx, dtype, tokens):
    """silu(gate) up of 1e54 is no f32: that token's outputs are not finite, the others keep their bits."""
    import torch
    rng = np.random.default_rng(80 + dtype)
    hidden = 200
    layer = Layer(ctx, rng, 4, 2, hidden, 130, 1, router=np.zeros((4, hidden), np.float32))
    xd, _ = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    clean = forward(ctx, layer, xd, dtype, tokens, hidden)
    xd[1] *= 1e27
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    keep = [t for t in range(tokens) if t != 1]
    assert not torch.isfinite(y[1]).any()
    assert torch.equal(y[keep], clean[keep])
    layer.moe.free()
