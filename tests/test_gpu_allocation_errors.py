"""An allocation that the card refuses is that call's error alone: the runtime keeps the last error of a thread until
it is read, and the next call's launches must not find it."""
import ctypes

import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import check, f64, make_weight, product, quantize

pytestmark = pytest.mark.gpu

M, N, K = 20, 70, 200


@pytest.fixture
def fresh():
    c = rocm.Context(0)
    yield c
    c.close()


def refused(call, *args):
    with pytest.raises(rocm.DzError) as e:
        call(*args)
    assert e.value.code == "RESOURCE_LIMIT", e.value


def small_product(ctx, rng):
    import torch
    codes, scales = make_weight(rng, N, K)
    x = rng.standard_normal((M, K)).astype(np.float32)
    w = ctx.fp8_weight(dev(codes), dev(scales), N, K)
    y = empty((M, N), torch.float32)
    ctx.fp8_linear(w, dev(x), rocm.F32, M, y, rocm.F32)
    ctx.sync()
    want, mags = product(*quantize(x), codes, scales, N, K)
    check(f64(y), want, mags, K, rocm.F32)
    w.free()


def test_a_weight_that_does_not_fit(fresh):
    """2^24 x 2^20 codes are 16 TiB: refused before anything is read."""
    rng = np.random.default_rng(1)
    t, s = dev(np.zeros(16, np.uint8)), dev(np.zeros(4, np.float32))
    refused(fresh.fp8_weight, t, s, 1 << 24, 1 << 20)
    small_product(fresh, rng)
    refused(fresh.fp8_weight_quantize, s, rocm.F32, 1 << 24, 1 << 20)
    small_product(fresh, rng)


def test_an_expert_layer_that_does_not_fit(fresh):
    """512 experts of three 65536 x 65536 projections are 6 TiB."""
    rng = np.random.default_rng(2)
    t, s = dev(np.zeros(1 << 12, np.uint8)), dev(np.zeros(1 << 12, np.float32))
    big = rocm.MoeConfig(experts=512, top_k=1, hidden=65536, ff=65536, renormalize=0)
    refused(fresh.moe, big, s, rocm.F32, (t, s), (t, s), (t, s))
    small = rocm.MoeConfig(experts=2, top_k=1, hidden=32, ff=16, renormalize=0)
    moe = fresh.moe(small, s, rocm.F32, (t, s), (t, s), (t, s))
    x, y = dev(np.ones((3, 32), np.float32)), dev(np.ones((3, 32), np.float32))
    moe.forward(x, rocm.F32, 3, y)
    fresh.sync()
    assert (y == 0).all()
    moe.free()
    small_product(fresh, rng)


def test_a_workspace_that_does_not_fit(fresh):
    """2^24 rows of 2^20 values: the codes of x alone are 16 TiB, and x is not read."""
    rng = np.random.default_rng(3)
    codes, scales = make_weight(rng, 1, 1 << 20)
    w = fresh.fp8_weight(dev(codes), dev(scales), 1, 1 << 20)
    x = dev(np.zeros(4, np.float32))
    refused(fresh.fp8_linear, w, x, rocm.F32, 1 << 24, x, rocm.F32)
    small_product(fresh, rng)
    w.free()


def test_a_device_allocation_that_does_not_fit(fresh):
    out = ctypes.c_void_p()
    refused(lambda: fresh._check(rocm.load().dz_alloc(fresh.handle, 1 << 44, ctypes.byref(out))))
    small_product(fresh, np.random.default_rng(4))
