"""The mixture-of-experts layer on e4m3 weights, against its definition in 64 bits.

Tolerances, with u = 2^-24 and sums of n terms off by at most n u of their magnitudes (any order): a logit is
off by dl = hidden u sum|x r|, a share by the relative 2 max(dl) + 8 u (expf and the quotients: a few ulps);
gate and up by (hidden + 2 blocks) u sum|x w|; h = silu(gate) up carries 1.1 |up| dgate + |silu| dup, a few ulps
(16 u |h|), and its own rounding to 16 bits (2^-16, f16 and bf16) or 24 (f32); y the down product of that, its own
sums and the shares' error, then the output's rounding, eps / 2 or half the smallest subnormal."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import EPS, LEAST, VALUES, _torch, f64, make_weight, rows_to, spread

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


class Layer:
    def __init__(self, ctx, rng, experts, top, hidden, ff, norm, router=None):
        self.shape = experts, top, hidden, ff, norm
        self.router = (rng.standard_normal((experts, hidden)) / np.sqrt(hidden)).astype(np.float32) \
            if router is None else router
        parts = {}
        for name, (n, k) in dict(gate=(ff, hidden), up=(ff, hidden), down=(hidden, ff)).items():
            made = [make_weight(rng, n, k) for _ in range(experts)]
            codes, scales = np.stack([c for c, _ in made]), np.stack([s for _, s in made])
            scales = (scales / (1.0 * np.sqrt(k))).astype(np.float32)
            parts[name] = codes, scales
        self.wide = {name: [VALUES[c] * spread(s, *c.shape) for c, s in zip(*p)] for name, p in parts.items()}
        cfg = rocm.MoeConfig(experts=experts, top_k=top, hidden=hidden, ff=ff, renormalize=norm)
        held = {name: (dev(c), dev(s)) for name, (c, s) in parts.items()}
        self.moe = ctx.moe(cfg, dev(self.router), rocm.F32, held["gate"], held["up"], held["down"])

    def route(self, x):
        """(ids, shares, their relative error) of rows x (64 bits)."""
        experts, top, hidden, ff, norm = self.shape
        r = self.router.astype(np.float64)
        logits = x @ r.T
        off = hidden * U * (np.abs(x) @ np.abs(r).T)
        ids = np.argsort(-logits, axis=1, kind="stable")[:, :top]
        p = np.exp(logits - logits.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        c = np.take_along_axis(p, ids, 1)
        if norm:
            c /= c.sum(1, keepdims=True)
        return ids, c, (2 * off.max(1, keepdims=True) + 8 * U) * np.ones_like(c)

    def __call__(self, x, dtype):
        """(y, tolerance) of rows x (64 bits) for outputs of `dtype`."""
        experts, top, hidden, ff, norm = self.shape
        ids, c, dc = self.route(x)
        y, off = np.zeros(x.shape), np.zeros(x.shape)
        kept = 2.0 ** -24 if dtype == rocm.F32 else 2.0 ** -16
        for t in range(x.shape[0]):
            for e, share, dshare in zip(ids[t], c[t], dc[t]):
                g, u, d = (self.wide[p][e] for p in ("gate", "up", "down"))
                a, b = g @ x[t], u @ x[t]
                n = (hidden + 2 * (-(-hidden // 128))) * U
                da, db = n * (np.abs(g) @ np.abs(x[t])), n * (np.abs(u) @ np.abs(x[t]))
                silu = a / (1 + np.exp(-a))
                h = silu * b
                dh = 1.1 * np.abs(b) * da + np.abs(silu) * db + (16 * U + kept) * np.abs(h)
                n = (ff + 2 * (-(-ff // 128)) + 2 * top + 16) * U
                y[t] += share * (d @ h)
                off[t] += share * (np.abs(d) @ (dh + (n + dshare) * np.abs(h)))
        return y, off * (1 + EPS[dtype]) + EPS[dtype] * np.abs(y) + LEAST[dtype]


def forward(ctx, layer, xd, dtype, tokens, hidden):
    import torch
    y = torch.full((tokens, hidden), float("nan"), dtype=_torch(dtype), device="cuda")
    torch.cuda.synchronize()
    layer.moe.forward(xd, dtype, tokens, y)
    ctx.sync()
    return y


# tokens, experts, top, hidden, ff, renormalize
CASES = [(1, 1, 1, 1, 1, 1), (1, 8, 2, 128, 128, 1), (1, 64, 8, 520, 200, 0), (2, 5, 5, 130, 17, 1),
         (7, 20, 3, 1000, 70, 0), (16, 4, 2, 256, 300, 1), (17, 3, 1, 200, 129, 0), (33, 6, 4, 384, 100, 1),
         (64, 16, 2, 260, 144, 1), (65, 2, 2, 129, 40, 0), (128, 9, 3, 300, 96, 1), (3, 130, 16, 64, 48, 1),
         (5, 512, 4, 72, 16, 0), (16, 128, 8, 130, 2100, 1), (15, 40, 1, 300, 200, 0), (8, 2, 2, 1100, 257, 1),
         (100, 300, 2, 140, 33, 0), (19, 30, 1, 257, 513, 1)]


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.F16, rocm.BF16])
@pytest.mark.parametrize("tokens,experts,top,hidden,ff,norm", CASES)
def test_layer_against_64_bits(ctx, tokens, experts, top, hidden, ff, norm, dtype):
    import torch
    rng = np.random.default_rng(tokens + experts + hidden)
    layer = Layer(ctx, rng, experts, top, hidden, ff, norm)
    xd, xf = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
    x = xf.astype(np.float64)
    ids, shares = empty((tokens, top), torch.int32), empty((tokens, top), torch.float32)
    layer.moe.route(xd, dtype, tokens, ids, shares)
    ctx.sync()
    want_ids, want, rel = layer.route(x)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(f64(shares) - want) <= rel * want).all()
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    want, tol = layer(x, dtype)
    err = np.abs(f64(y) - want)
    assert (err <= tol).all(), (err / tol).max()
    assert torch.equal(y, forward(ctx, layer, xd, dtype, tokens, hidden))
    layer.moe.free()


def test_equal_logits_go_to_the_lower_index(ctx):
    import torch
    rng = np.random.default_rng(1)
    for experts, top in ((6, 3), (70, 5), (300, 16)):
        hidden = 40
        router = (rng.integers(-2, 3, (experts, hidden)) / 4).astype(np.float32)
        router[experts // 2:] = router[: experts - experts // 2]  # each logit at least twice
        router[1] = router[0]
        layer = Layer(ctx, rng, experts, top, hidden, 16, 1, router=router)
        x = rng.integers(-1, 2, (9, hidden)).astype(np.float32)  # logits exact in f32
        x[4] = 0  # all equal
        ids, shares = empty((9, top), torch.int32), empty((9, top), torch.float32)
        layer.moe.route(dev(x), rocm.F32, 9, ids, shares)
        ctx.sync()
        assert np.array_equal(ids.cpu().numpy(), layer.route(x.astype(np.float64))[0])
        layer.moe.free()


@pytest.mark.parametrize("tokens", [16, 40, 128])
def test_every_token_to_the_same_experts(ctx, tokens):
    """One expert's list is as long as the call, the others' empty."""
    rng = np.random.default_rng(tokens)
    hidden, router = 96, np.zeros((7, 96), np.float32)
    router[5, 0], router[2, 0] = 3, 2
    layer = Layer(ctx, rng, 7, 2, hidden, 64, 1, router=router)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    x[:, 0] = 1 + np.abs(x[:, 0])
    y = forward(ctx, layer, dev(x), rocm.F32, tokens, hidden)
    want, tol = layer(x.astype(np.float64), rocm.F32)
    assert set(layer.route(x.astype(np.float64))[0].ravel()) == {2, 5}
    assert (np.abs(f64(y) - want) <= tol).all()
    layer.moe.free()


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.F16, rocm.BF16])
def test_a_token_that_is_not_finite_touches_no_other(ctx, dtype):
    import torch
    rng = np.random.default_rng(9)
    tokens, hidden = 21, 200
    layer = Layer(ctx, rng, 6, 2, hidden, 130, 0)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    xd, _ = rows_to(x, dtype)
    xd_bad = xd.clone()
    bad = [0, 7, 20]
    for t, v in zip(bad, (float("nan"), float("inf"), -float("inf"))):
        xd_bad[t, 11 * t % hidden] = v
    clean = x.copy()
    clean[bad] = 0  # any finite rows in their place
    for t in bad:
        xd[t] = 0
    torch.cuda.synchronize()
    y = forward(ctx, layer, xd_bad, dtype, tokens, hidden)
    keep = [t for t in range(tokens) if t not in bad]
    want, tol = layer(xd.double().cpu().numpy(), dtype)
    assert torch.isnan(y[bad]).all()
    assert (np.abs(f64(y[keep]) - want[keep]) <= tol[keep]).all()
    # the call after it is clean
    y = forward(ctx, layer, xd, dtype, tokens, hidden)
    assert (np.abs(f64(y) - want) <= tol).all()
    layer.moe.free()


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.F16, rocm.BF16])
def test_rows_at_odd_addresses_and_bytes_around_the_output_left_alone(ctx, dtype):
    import torch
    rng = np.random.default_rng(15)
    hidden = 131
    layer = Layer(ctx, rng, 6, 2, hidden, 77, 1)
    for tokens in (1, 5, 13, 40):
        xd, xf = rows_to(rng.standard_normal((tokens, hidden)).astype(np.float32), dtype)
        room = torch.zeros(tokens * hidden + 1, dtype=xd.dtype, device="cuda")
        room[1:] = xd.flatten()
        out = torch.full((tokens * hidden + 9,), 7.0, dtype=xd.dtype, device="cuda")
        torch.cuda.synchronize()
        layer.moe.forward(room[1:], dtype, tokens, out[3:])
        ctx.sync()
        want, tol = layer(xf.astype(np.float64), dtype)
        assert (np.abs(f64(out[3:3 + tokens * hidden].view(tokens, hidden)) - want) <= tol).all()
        assert (out[:3] == 7).all() and (out[3 + tokens * hidden:] == 7).all()
    layer.moe.free()


def test_large_values_keep_their_range(ctx):
    """x near bf16's and f32's ends: the terms of an activation do not overflow."""
    rng = np.random.default_rng(13)
    layer = Layer(ctx, rng, 4, 2, 130, 64, 1, router=np.zeros((4, 130), np.float32))
    x = np.full((3, 130), 0.0, np.float32)
    x[0, 3], x[1, 5], x[2, 129] = 1e30, 3e4, 1e-30
    y = forward(ctx, layer, dev(x), rocm.F32, 3, 130)
    want, tol = layer(x.astype(np.float64), rocm.F32)
    fine = np.abs(want) < 3e38
    assert (np.abs(f64(y) - want)[fine] <= tol[fine]).all()
    layer.moe.free()


def test_refusals(ctx):
    import torch
    rng = np.random.default_rng(2)
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    f = torch.ones(1 << 16, device="cuda")
    torch.cuda.synchronize()

    def make(router=f, router_dtype=rocm.F32, gate=(t, f), up=(t, f), down=(t, f), **kw):
        cfg = dict(experts=4, top_k=2, hidden=32, ff=16, renormalize=1)
        cfg.update(kw)
        return ctx.moe(rocm.MoeConfig(**cfg), router, router_dtype, gate, up, down)

    def refused(code, call, *args, **kw):
        with pytest.raises(rocm.DzError) as e:
            call(*args, **kw)
        assert e.value.code == code, e.value

    for kw in (dict(experts=0), dict(experts=513), dict(top_k=0), dict(top_k=5), dict(hidden=0), dict(ff=0),
               dict(hidden=65537), dict(ff=-1), dict(renormalize=2), dict(experts=64, top_k=17), dict(router_dtype=5)):
        refused("INVALID_PARAMETERS", make, **kw)
    for kw in (dict(router=None), dict(gate=(None, f)), dict(up=(t, None)), dict(down=(None, None))):
        refused("INVALID_REQUEST", make, **kw)
    nan, neg, inf = t.clone(), f.clone(), f.clone()
    nan[4 * 16 * 32 - 1], neg[3], inf[4 * 32 - 1] = 0x7F, -1.0, float("inf")
    torch.cuda.synchronize()
    for kw in (dict(gate=(nan, f)), dict(up=(nan, f)), dict(down=(nan, f)), dict(gate=(t, neg)), dict(up=(t, neg)),
               dict(down=(t, neg)), dict(router=inf)):
        refused("INVALID_CHECKPOINT", make, **kw)
    moe = make()
    refused("INPUT_TOO_LONG", moe.forward, f, rocm.F32, rocm.MOE_MAX_TOKENS + 1, f)
    refused("INVALID_PARAMETERS", moe.forward, f, 4, 1, f)
    refused("INVALID_REQUEST", moe.forward, None, rocm.F32, 1, f)
    refused("INVALID_REQUEST", moe.forward, f, rocm.F32, 1, None)
    refused("INVALID_REQUEST", moe.route, f, rocm.F32, 1, None, f)
    refused("INVALID_REQUEST", moe.route, f, rocm.F32, 1, t, None)
    moe.forward(None, rocm.F32, 0, None)
    moe.route(None, rocm.F32, 0, None, None)
    moe.free()


def test_captured_layer_replayed(ctx):
    """A layer recorded into a graph, replayed over new inputs between eager calls of another size."""
    import torch
    rng = np.random.default_rng(31)
    hidden = 264
    layer = Layer(ctx, rng, 12, 3, hidden, 96, 1)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        for dtype, tokens in ((rocm.BF16, 1), (rocm.F32, 20), (rocm.F16, 70)):
            x = torch.zeros(tokens, hidden, dtype=_torch(dtype), device="cuda")
            y, eager = torch.empty_like(x), torch.empty_like(x)
            torch.cuda.synchronize()
            layer.moe.forward(x, dtype, tokens, y)
            ctx.sync()
            graph = torch.cuda.CUDAGraph()
            with rocm.capture(graph, stream):
                layer.moe.forward(x, dtype, tokens, y)
                capture = ctx.capture_id()
            for i in range(4):
                x.copy_(torch.from_numpy(rng.standard_normal((tokens, hidden)).astype(np.float32)))
                torch.cuda.synchronize()
                with torch.cuda.stream(stream):
                    graph.replay()
                torch.cuda.synchronize()
                layer.moe.forward(x, dtype, tokens, eager)
                ctx.sync()
                assert torch.equal(y, eager), (dtype, i)
                want, tol = layer(x.double().cpu().numpy(), dtype)
                assert (np.abs(f64(y) - want) <= tol).all()
            del graph
            ctx.capture_release(capture)
    finally:
        ctx.set_stream(None)
    layer.moe.free()


def test_a_decoder_block_of_8_bit_weights(ctx):
    """The operators as a served block runs them: a norm, one quantization that two projections share, the
    output projection, the residual, and the expert layer on the next norm; recorded and replayed."""
    import torch
    rng = np.random.default_rng(41)
    d, width, tokens = 256, 384, 5
    layer = Layer(ctx, rng, 8, 2, d, 128, 1)
    made = {name: make_weight(rng, n, k) for name, (n, k) in dict(a=(width, d), b=(width, d), o=(d, width)).items()}
    for name in made:
        made[name] = made[name][0], (made[name][1] * 0.05).astype(np.float32)
    w = {name: ctx.fp8_weight(dev(c), dev(s), *c.shape) for name, (c, s) in made.items()}
    ones = dev(np.ones(d, np.float32))
    f32 = dict(dtype=torch.float32, device="cuda")
    x, normed, moe_out = (torch.zeros(tokens, d, **f32) for _ in range(3))
    a, b = torch.zeros(tokens, width, **f32), torch.zeros(tokens, width, **f32)
    out = torch.zeros(tokens, d, **f32)
    q, s = torch.zeros(tokens, d, dtype=torch.uint8, device="cuda"), torch.zeros(d // 128, tokens, **f32)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)

    def block():
        ctx.rmsnorm(x, normed, tokens, d, ones, 1e-6, zero_centered=False)
        ctx.fp8_quantize(normed, rocm.F32, tokens, d, q, s)
        ctx.fp8_linear_q8(w["a"], q, s, tokens, a, rocm.F32)
        ctx.fp8_linear_q8(w["b"], q, s, tokens, b, rocm.F32)
        ctx.silu_mul(a, b, tokens * width)
        ctx.fp8_linear(w["o"], a, rocm.F32, tokens, out, rocm.F32)
        ctx.add(out, x, rocm.F32, tokens * d)
        ctx.rmsnorm(out, normed, tokens, d, ones, 1e-6, zero_centered=False)
        layer.moe.forward(normed, rocm.F32, tokens, moe_out)
        ctx.add(out, moe_out, rocm.F32, tokens * d)

    def plain(v):
        def fp8(rows, name):
            from tests.test_gpu_fp8 import quantize
            codes, scales = made[name]
            qq, ss = quantize(rows.astype(np.float32))
            r = VALUES[qq].reshape(tokens, -1, 128) * ss.T.astype(np.float64)[:, :, None]
            return r.reshape(tokens, -1) @ (VALUES[codes] * spread(scales, *codes.shape)).T

        def norm(rows):
            return rows / np.sqrt((rows ** 2).mean(1, keepdims=True) + 1e-6)
        n = norm(v)
        g, u = fp8(n, "a"), fp8(n, "b")
        o = fp8(g / (1 + np.exp(-g)) * u, "o") + v
        return o + layer(norm(o), rocm.F32)[0]

    try:
        torch.cuda.synchronize()
        block()
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with rocm.capture(graph, stream):
            block()
            capture = ctx.capture_id()
        for i in range(3):
            v = rng.standard_normal((tokens, d)).astype(np.float32)
            x.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            got = f64(out)
            block()
            ctx.sync()
            assert np.array_equal(got, f64(out))
            # an ulp before a quantization may move a code by a step, 2^-3 of its value, for a few of them
            want = plain(v.astype(np.float64))
            assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)
        del graph
        ctx.capture_release(capture)
    finally:
        ctx.set_stream(None)
    for h in w.values():
        h.free()
    layer.moe.free()
