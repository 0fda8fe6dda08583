"""Zeros of either sign keep it: e4m3(-0 / scale) is 0x80 whatever the block's scale."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import bits_equal, empty, host
from tests.test_gpu_fp8 import DTYPES, quantize, rows_to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_negative_zeros_in_blocks_of_every_scale(ctx, dtype):
    import torch
    rng = np.random.default_rng(dtype + 5)
    m, k = 40, 300
    x = rng.standard_normal((m, k)).astype(np.float32)
    if dtype != rocm.F16:
        x[8:16] *= np.float32(2.0 ** 90)   # large scales
        x[16:24] *= np.float32(2.0 ** -90)  # a scale below 2^-60
    x[24:30] *= np.float32(2.0 ** -12)
    x[rng.random((m, k)) < 0.3] = -0.0
    x[rng.random((m, k)) < 0.2] = 0.0
    x[30:32] = -0.0                         # nothing but zeros: the scale's floor
    x[32, ::2], x[32, 1::2] = 0.0, -0.0
    xd, xf = rows_to(x, dtype)
    assert (np.signbit(xf) & (xf == 0)).sum() > 1000
    q, s = empty((m, 384), torch.uint8), empty((3, m), torch.float32)
    ctx.fp8_quantize(xd, dtype, m, k, q, s)
    wq, ws = quantize(xf)
    assert bits_equal(host(ctx, s), ws)
    assert bits_equal(host(ctx, q), wq)


def test_the_weight_quantizer_gives_the_same_zeros(ctx):
    """-0 of a weight comes back as -0."""
    import torch
    w = np.ones((4, 130), np.float32)
    w[1:3, ::3] = -0.0
    wd, _ = rows_to(w, rocm.F32)
    h = ctx.fp8_weight_quantize(wd, rocm.F32, 4, 130)
    y = empty((4, 130), torch.float32)
    ctx.fp8_dequant(h, y)
    assert np.array_equal(np.signbit(host(ctx, y)), np.signbit(w))
    h.free()
