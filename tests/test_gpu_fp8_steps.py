"""The products' tile kernels over many steps along k, so that every LDS stage is filled, read and filled again, on
grids of several ragged tiles that leave k whole; and one row by either entry point. Tolerances as in test_gpu_fp8.

k is cut only where all runs of it fit one round of the chip, `resident` tiles a compute unit: grids of more than half
a round stay whole, which each shape here asserts for the tiles that it is meant for."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import DTYPES, _torch, check, f64, make_weight, product, quantize, rows_to, to_codes

pytestmark = pytest.mark.gpu

# tile: rows, columns, workgroups a compute unit, 128-blocks of a step, stages
TILES = {"32x32k4": (32, 32, 1, 4, 4), "64x32k4": (64, 32, 1, 4, 3), "64x64k4": (64, 64, 1, 4, 2),
         "64x64": (64, 64, 2, 1, 4), "64x64k2": (64, 64, 2, 2, 2), "128x128": (128, 128, 1, 2, 2),
         "256x128": (256, 128, 1, 1, 3), "256x256": (256, 256, 1, 1, 2)}
SMALL, LARGE = (1101, 1090, 4200), (2901, 2701, 2300)


def shape_of(ctx, tile):
    bm, bn, resident, step, stages = TILES[tile]
    m, n, k = LARGE if bm >= 128 else SMALL
    tiles = -(-m // bm) * -(-n // bn)
    assert 2 * tiles > resident * ctx.info()["compute_units"]  # k is not cut
    assert -(-(-(-k // 128)) // step) >= 2 * stages            # every stage is filled twice at least
    return m, n, k


@pytest.fixture(scope="module")
def made():
    """Codes, scales, and the product in 64 bits, by shape and kind, made once."""
    kept = {}

    def get(shape, integer):
        if (shape, integer) not in kept:
            m, n, k = shape
            rng = np.random.default_rng(m + n + k + integer)
            codes, scales = make_weight(rng, n, k, integer)
            if integer:
                g = -(-k // 128)
                q = np.zeros((m, g * 128), np.uint8)
                q[:, :k] = to_codes(rng.integers(-16, 17, (m, k)).astype(np.float64))
                s = (rng.random((g, m)) + 0.5).astype(np.float32)
            else:
                q, s = quantize((0.1 * rng.standard_normal((m, k))).astype(np.float32))
            kept[shape, integer] = q, s, codes, scales, *product(q, s, codes, scales, n, k)
        return kept[shape, integer]

    yield get
    kept.clear()


@pytest.mark.parametrize("integer", [False, True])
@pytest.mark.parametrize("y_dtype", DTYPES)
@pytest.mark.parametrize("tile", TILES)
def test_many_steps_on_many_tiles(ctx, made, tile, y_dtype, integer):
    import torch
    m, n, k = shape = shape_of(ctx, tile)
    q, s, codes, scales, want, mags = made(shape, integer)
    assert np.abs(want).max() < 6e4
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    y, again = (torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda") for _ in range(2))
    qd, sd = dev(q), dev(s)
    ctx.select_variant("fp8", tile)
    try:
        ctx.fp8_linear_q8(w, qd, sd, m, y, y_dtype)
        ctx.fp8_linear_q8(w, qd, sd, m, again, y_dtype)
        ctx.sync()
    finally:
        ctx.select_variant("fp8", "auto")
    check(f64(y), want, mags, k, y_dtype, exact_dots=integer)
    assert torch.equal(y, again)
    w.free()


@pytest.mark.parametrize("y_dtype", DTYPES)
@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 40, 9000), (1, 1000, 520), (1, 17, 4097), (1, 17000, 300),
                                   (3, 300, 1000), (20, 77, 5000), (70, 131, 2600), (300, 512, 256)])
def test_both_entry_points_give_the_same_bits(ctx, m, n, k, x_dtype, y_dtype):
    """One row has a kernel that quantizes by itself; the others share theirs."""
    import torch
    rng = np.random.default_rng(m + n + k)
    codes, scales = make_weight(rng, n, k)
    xd, _ = rows_to((0.1 * rng.standard_normal((m, k))).astype(np.float32), x_dtype)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    g = -(-k // 128)
    q, s = empty((m, g * 128), torch.uint8), empty((g, m), torch.float32)
    one, two = empty((m, n), _torch(y_dtype)), empty((m, n), _torch(y_dtype))
    ctx.fp8_linear(w, xd, x_dtype, m, one, y_dtype)
    ctx.fp8_quantize(xd, x_dtype, m, k, q, s)
    ctx.fp8_linear_q8(w, q, s, m, two, y_dtype)
    ctx.sync()
    assert torch.isfinite(one).all() and torch.equal(one, two)
    w.free()
