"""The largest sizes that the 8-bit floating point entry points take, against 64 bits, with the tolerances of
test_gpu_fp8 and test_gpu_moe."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import VALUES, _torch, check, f64, make_weight, product, quantize, spread
from tests.test_gpu_moe import Layer, forward

pytestmark = pytest.mark.gpu

WIDEST, LONGEST = 1 << 20, 1 << 24


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.F16])
@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_the_widest_rows(ctx, m, y_dtype):
    rng = np.random.default_rng(m)
    n, k = 20, WIDEST
    codes, scales = make_weight(rng, n, k)
    x = (0.01 * rng.standard_normal((m, k))).astype(np.float32)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    xd, y = dev(x), empty((m, n), _torch(y_dtype))
    ctx.fp8_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    few = sorted({0, m // 2, m - 1})
    want, mags = product(*quantize(x[few]), codes, scales, n, k)
    assert np.abs(want).max() < 6e4
    check(f64(y[few]), want, mags, k, y_dtype)
    assert np.isfinite(f64(y)).all()
    w.free()


@pytest.mark.parametrize("m", [1, 2, 40])
def test_the_most_rows_of_a_weight(ctx, m):
    import torch
    rng = np.random.default_rng(m)
    n, k = LONGEST, 5
    codes, scales = make_weight(rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    y = empty((m, n), torch.float32)
    ctx.fp8_linear(w, dev(x), rocm.F32, m, y, rocm.F32)
    ctx.sync()
    few = sorted({0, m - 1})
    want, mags = product(*quantize(x[few]), codes, scales, n, k)
    check(f64(y[few]), want, mags, k, rocm.F32)
    assert torch.isfinite(y).all()
    d = empty((n, k), torch.float32)
    ctx.fp8_dequant(w, d)
    ctx.sync()
    assert torch.equal(d, torch.from_numpy((VALUES[codes].astype(np.float32) * spread(scales, n, k).astype(np.float32))).cuda())
    w.free()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.BF16])
def test_the_most_rows_of_activations(ctx, y_dtype):
    rng = np.random.default_rng(3)
    m, n, k = LONGEST, 2, 3
    codes, scales = make_weight(rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    y = empty((m, n), _torch(y_dtype))
    ctx.fp8_linear(w, dev(x), rocm.F32, m, y, y_dtype)
    ctx.sync()
    part = np.unique(np.concatenate([np.arange(4096), rng.integers(0, m, 1 << 16), np.arange(m - 4096, m)]))
    import torch
    want, mags = product(*quantize(x[part]), codes, scales, n, k)
    check(f64(y[torch.from_numpy(part).cuda()]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()


@pytest.mark.parametrize("dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("tokens,experts,top,hidden,ff", [(128, 16, 16, 64, 65536), (128, 16, 16, 65536, 48),
                                                          (1, 16, 16, 65536, 48), (3, 4, 2, 50, 65536),
                                                          (128, 512, 16, 40, 24)])
def test_the_widest_expert_layers(ctx, tokens, experts, top, hidden, ff, dtype):
    import torch
    rng = np.random.default_rng(tokens + hidden)
    layer = Layer(ctx, rng, experts, top, hidden, ff, 1)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden)).astype(np.float32)).cuda().to(_torch(dtype))
    few = sorted({0, tokens // 2 + 1, tokens - 1} & set(range(tokens)))
    y = forward(ctx, layer, x, dtype, tokens, hidden)
    want, tol = layer(x[few].double().cpu().numpy(), dtype)
    assert (np.abs(f64(y[few]) - want) <= tol).all()
    assert torch.isfinite(y).all()
    layer.moe.free()
