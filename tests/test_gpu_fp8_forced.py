"""A forced variant of the "fp8" family runs its own kernel, but for the one that the header excepts: f32 outputs of
256x256 take 256x128 tiles."""
import re
from pathlib import Path

import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty, launched
from tests.test_gpu_fp8 import VARIANTS, _torch, make_weight

HEADER = Path(__file__).resolve().parent.parent / "include" / "decisive_rocm.h"
FORMS = {"rows16": "fp8_rows_kernel<1,", "rows32": "fp8_rows_kernel<2,", "32x32k4": "fp8_tile_kernel<32, 32, 2, 1, 4,",
         "64x32k4": "fp8_tile_kernel<64, 32, 2, 1, 4,", "64x64k4": "fp8_tile_kernel<64, 64, 2, 2, 4,",
         "64x64": "fp8_tile_kernel<64, 64, 2, 2, 1,", "64x64k2": "fp8_tile_kernel<64, 64, 2, 1, 2,",
         "128x128": "fp8_tile_kernel<128, 128,", "256x128": "fp8_tile_kernel<256, 128,",
         "256x256": "fp8_tile_kernel<256, 256,"}


def test_the_header_says_what_f32_outputs_take():
    listed = re.search(r'\n \*   "fp8" (.*?)\*/', HEADER.read_text(), re.S).group(1)
    assert re.search(r"f32\s+outputs\s+of\s+256x256\s+take\s+256x128", listed.replace("\n *", " "))


@pytest.mark.gpu
@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.F16, rocm.BF16])
@pytest.mark.parametrize("variant", VARIANTS)
def test_the_kernel_that_runs(ctx, variant, y_dtype):
    import numpy as np
    rng = np.random.default_rng(7)
    m, n, k = 90, 200, 300
    codes, scales = make_weight(rng, n, k)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    x, y = dev(rng.standard_normal((m, k)).astype(np.float32)), empty((m, n), _torch(y_dtype))
    ctx.select_variant("fp8", variant)
    try:
        assert ctx.info()["variants"]["fp8"] == variant
        names = launched(ctx, lambda: ctx.fp8_linear(w, x, rocm.F32, m, y, y_dtype))
    finally:
        ctx.select_variant("fp8", "auto")
    form = FORMS["256x128" if variant == "256x256" and y_dtype == rocm.F32 else variant]
    assert any(form in name for name in names), names
    w.free()
