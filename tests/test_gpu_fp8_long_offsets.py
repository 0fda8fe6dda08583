"""Weights, activations, outputs and expert layers of more than 2^32 bytes or 2^31 values: the far ends of each against
64 bits, with the tolerances of test_gpu_fp8 and test_gpu_moe."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev
from tests.test_gpu_fp8 import VALUES, _torch, check, f64, product, quantize
from tests.test_gpu_moe import Layer, forward

pytestmark = pytest.mark.gpu

MANY = (1 << 22) + 96  # rows of 1024 bytes: past 2^32 bytes


def random_codes(seed, *shape):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 127, shape, generator=g, device="cuda", dtype=torch.uint8)
    return codes.bitwise_or_(torch.randint(0, 2, shape, generator=g, device="cuda", dtype=torch.uint8).mul_(128))


def random_scales(rng, *shape):
    return (rng.random(shape) * 0.01 + 1e-3).astype(np.float32)


def ends(rng, count, size, tail):
    """`count` places below `size`, its first and last ones among them."""
    return np.unique(np.concatenate([[0], rng.integers(0, size, count), np.arange(size - tail, size)]))


def column_part(q, s, codes, scales, cols, k):
    """product() for some columns: each with its own block's scales."""
    y, mags = [], []
    for block in np.unique(cols // 128):
        mine = cols[cols // 128 == block]
        a, b = product(q, s, codes[mine].cpu().numpy(), scales[block:block + 1], len(mine), k)
        y.append(a), mags.append(b)
    return np.concatenate(y, 1), np.concatenate(mags, 1)


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("m", [1, 3, 40])
def test_a_weight_past_32_bits(ctx, m, y_dtype):
    import torch
    rng = np.random.default_rng(m)
    n, k = MANY, 1024
    codes, scales = random_codes(m, n, k), random_scales(rng, -(-n // 128), k // 128)
    x = (0.1 * rng.standard_normal((m, k))).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda")
    sd, xd = dev(scales), dev(x)
    w = ctx.fp8_weight(codes, sd, n, k)
    ctx.fp8_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    cols = ends(rng, 60, n, 200)
    want, mags = column_part(*quantize(x), codes, scales, cols, k)
    check(f64(y[:, torch.from_numpy(cols).cuda()]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()
    del codes, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.BF16])
def test_activations_past_32_bits(ctx, y_dtype):
    import torch
    rng = np.random.default_rng(5)
    m, n, k = MANY, 33, 1024
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.1)
    codes, scales = random_codes(6, n, k), random_scales(rng, 1, k // 128)
    y = torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda")
    sd = dev(scales)
    w = ctx.fp8_weight(codes, sd, n, k)
    ctx.fp8_linear(w, x, rocm.BF16, m, y, y_dtype)
    ctx.sync()
    rows = torch.from_numpy(ends(rng, 300, m, 300)).cuda()
    want, mags = product(*quantize(x[rows].float().cpu().numpy()), codes.cpu().numpy(), scales, n, k)
    check(f64(y[rows]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()
    del x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.F16])
def test_outputs_past_32_bits(ctx, y_dtype):
    import torch
    rng = np.random.default_rng(7)
    m, n, k = 70001, 31001, 130
    codes, scales = random_codes(8, n, k), random_scales(rng, -(-n // 128), 2)
    x = (0.1 * rng.standard_normal((m, k))).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda")
    sd, xd = dev(scales), dev(x)
    w = ctx.fp8_weight(codes, sd, n, k)
    ctx.fp8_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    rows = ends(rng, 20, m, 20)
    want, mags = product(*quantize(x[rows]), codes.cpu().numpy(), scales, n, k)
    check(f64(y[torch.from_numpy(rows).cuda()]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("tokens", [2, 18])
def test_an_expert_layer_past_32_bits(ctx, tokens):
    """Each projection has more than 2^32 bytes of codes; the tokens go to the last experts."""
    import torch
    rng = np.random.default_rng(9)
    experts, top, d = 258, 2, 4096
    layer = Layer.__new__(Layer)
    layer.shape = experts, top, d, d, 1
    layer.router = np.zeros((experts, d), np.float32)
    layer.router[-1, 0], layer.router[-2, 0] = 2, 1
    layer.wide, held = {}, {}
    for i, name in enumerate(("gate", "up", "down")):
        codes, scales = random_codes(20 + i, experts, d, d), random_scales(rng, experts, d // 128, d // 128) / np.float32(64)
        held[name] = codes, dev(scales)
        layer.wide[name] = {e: VALUES[codes[e].cpu().numpy()] *
                            scales[e].astype(np.float64).repeat(128, 0).repeat(128, 1) for e in range(experts - 2, experts)}
    cfg = rocm.MoeConfig(experts=experts, top_k=top, hidden=d, ff=d, renormalize=1)
    layer.moe = ctx.moe(cfg, dev(layer.router), rocm.F32, held["gate"], held["up"], held["down"])
    x = rng.standard_normal((tokens, d)).astype(np.float32)
    x[:, 0] = 1 + np.abs(x[:, 0])
    few = [0, tokens - 1]
    y = forward(ctx, layer, dev(x), rocm.F32, tokens, d)
    want, tol = layer(x[few].astype(np.float64), rocm.F32)
    assert set(layer.route(x.astype(np.float64))[0].ravel()) == {experts - 2, experts - 1}
    assert (np.abs(f64(y[few]) - want) <= tol).all()
    layer.moe.free()
    del held
    torch.cuda.empty_cache()
