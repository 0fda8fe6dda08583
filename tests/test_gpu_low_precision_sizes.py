"""The 4-bit floating point products, the norm with codes and the choice of experts at the ends of what they take: the
widest rows, the most rows, and weights, codes, activations and outputs of more than 2^32 bytes or 2^31 values. Compared at
the far ends, with the tolerances of test_gpu_mx4 and, of norms and choices, bit by bit."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_add_norm import definition as normed
from tests.test_gpu_fp8 import _torch, f64, quantize as to_fp8
from tests.test_gpu_mx4 import buffers, check, make_weight, product, quantize, values
from tests.test_gpu_select import definition as chosen, rule_of

pytestmark = pytest.mark.gpu

WIDEST, LONGEST = 1 << 20, 1 << 24


def ends(rng, count, size, tail):
    """`count` places below `size`, its first and last ones among them."""
    return np.unique(np.concatenate([[0], rng.integers(0, size, count), np.arange(size - tail, size)]))


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("m", [1, 4, 20, 300])
def test_the_widest_rows(ctx, m, y_dtype):
    rng = np.random.default_rng(m)
    n, k = 20, WIDEST
    w, wide = make_weight(ctx, rng, n, k)
    x = (0.01 * rng.standard_normal((m, k))).astype(np.float32)
    xd, y = dev(x), empty((m, n), _torch(y_dtype))
    ctx.mx4_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    few = sorted({0, m // 2, m - 1})
    want, mags = product(values(*quantize(x[few]), k), wide)
    check(f64(y[few]), want, mags, k, y_dtype)
    assert np.isfinite(f64(y)).all()
    w.free()


@pytest.mark.parametrize("m", [1, 3, 40])
def test_the_most_rows_of_a_weight(ctx, m):
    import torch
    rng = np.random.default_rng(m)
    n, k = LONGEST, 5
    w, wide = make_weight(ctx, rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    y = empty((m, n), torch.float32)
    ctx.mx4_linear(w, dev(x), rocm.F32, m, y, rocm.F32)
    ctx.sync()
    few = sorted({0, m - 1})
    want, mags = product(values(*quantize(x[few]), k), wide)
    check(f64(y[few]), want, mags, k, rocm.F32)
    assert torch.isfinite(y).all()
    d = empty((n, k), torch.float32)
    ctx.mx4_dequant(w, d)
    ctx.sync()
    assert torch.equal(d, torch.from_numpy(wide.astype(np.float32)).cuda())
    w.free()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.F16])
def test_the_most_rows_of_activations(ctx, y_dtype):
    import torch
    rng = np.random.default_rng(3)
    m, n, k = LONGEST, 2, 3
    w, wide = make_weight(ctx, rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda")
    xd = dev(x)
    ctx.mx4_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    rows = ends(rng, 300, m, 300)
    want, mags = product(values(*quantize(x[rows]), k), wide)
    check(f64(y[torch.from_numpy(rows).cuda()]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()


@pytest.mark.parametrize("m", [1, 16, 40])
def test_a_weight_past_32_bits(ctx, m):
    """More than 2^32 bytes of codes."""
    import torch
    rng = np.random.default_rng(m)
    n, k = (1 << 23) + 96, 1024
    g = torch.Generator(device="cuda").manual_seed(m)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(118, 123, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    w = ctx.mx4_weight(codes, scales, n, k)
    assert w.device_bytes > 1 << 32
    x = (0.1 * rng.standard_normal((m, k))).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    xd = dev(x)
    ctx.mx4_linear(w, xd, rocm.F32, m, y, rocm.BF16)
    ctx.sync()
    cols = ends(rng, 60, n, 200)
    at = torch.from_numpy(cols).cuda()
    packed = codes[at].cpu().numpy()
    some = np.stack([packed & 15, packed >> 4], -1).reshape(len(cols), k)
    want, mags = product(values(*quantize(x), k), values(some, scales[at].cpu().numpy(), k))
    check(f64(y[:, at]), want, mags, k, rocm.BF16)
    assert torch.isfinite(y).all()
    w.free()
    del codes, y
    torch.cuda.empty_cache()


def test_activations_past_32_bits(ctx):
    """More than 2^32 bytes of codes and 2^33 of activations."""
    import torch
    rng = np.random.default_rng(5)
    m, n, k = (1 << 23) + 96, 33, 1024
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16).mul_(0.1)
    w, wide = make_weight(ctx, rng, n, k)
    y = torch.full((m, n), float("nan"), dtype=torch.float32, device="cuda")
    q, s = buffers(m, k)
    assert q.numel() > 1 << 32
    torch.cuda.synchronize()
    ctx.mx4_quantize(x, rocm.BF16, m, k, q, s)
    ctx.mx4_linear_q4(w, q, s, m, y, rocm.F32)
    ctx.sync()
    rows = ends(rng, 300, m, 300)
    at = torch.from_numpy(rows).cuda()
    want, mags = product(values(*quantize(x[at].float().cpu().numpy()), k), wide)
    check(f64(y[at]), want, mags, k, rocm.F32)
    assert torch.isfinite(y).all()
    w.free()
    del x, y, q, s
    torch.cuda.empty_cache()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.F16])
def test_outputs_past_32_bits(ctx, y_dtype):
    import torch
    rng = np.random.default_rng(7)
    m, n, k = 70001, 31001, 130
    w, wide = make_weight(ctx, rng, n, k)
    x = (0.1 * rng.standard_normal((m, k))).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=_torch(y_dtype), device="cuda")
    xd = dev(x)
    ctx.mx4_linear(w, xd, rocm.F32, m, y, y_dtype)
    ctx.sync()
    rows = ends(rng, 20, m, 20)
    want, mags = product(values(*quantize(x[rows]), k), wide)
    check(f64(y[torch.from_numpy(rows).cuda()]), want, mags, k, y_dtype)
    assert torch.isfinite(y).all()
    w.free()
    del y
    torch.cuda.empty_cache()


def test_a_form_whose_grid_would_be_too_large(ctx):
    """8.4 million tiles of 32 x 32, of 512 threads each: more than a grid's 2^32 threads, so another form takes them."""
    import torch
    rng = np.random.default_rng(8)
    m, n, k = 140001, 61441, 32
    w, wide = make_weight(ctx, rng, n, k)
    x = (0.1 * rng.standard_normal((m, k))).astype(np.float32)
    y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    xd = dev(x)
    ctx.select_variant("mx4", "32x32k4")
    try:
        ctx.mx4_linear(w, xd, rocm.F32, m, y, rocm.BF16)
        ctx.sync()
    finally:
        ctx.select_variant("mx4", "auto")
    rows = ends(rng, 20, m, 20)
    want, mags = product(values(*quantize(x[rows]), k), wide)
    check(f64(y[torch.from_numpy(rows).cuda()]), want, mags, k, rocm.BF16)
    w.free()
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("m,d", [(3, WIDEST), (LONGEST, 3), (LONGEST, 600), ((1 << 21) + 5, 2050)])
def test_norms_of_the_widest_and_the_most_rows(ctx, form, m, d):
    """The far rows' sums, codes and scales; the last two shapes pass 2^32 bytes in each 16-bit array, and need as many
    workgroups as a grid's side has, or rows of a workgroup each."""
    import torch
    rng = np.random.default_rng(d)
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(m, d, generator=g, device="cuda", dtype=torch.bfloat16)
    total = torch.empty_like(x)
    w = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    rows = ends(rng, 40, m, min(m, 70))
    at = torch.from_numpy(rows).cuda()
    wd, blocks = dev(w), -(-d // 128)
    _, y = normed((2 * x[at].float()).cpu().numpy(), None, w, 1e-6, False, rocm.BF16)
    if form == "fp8":
        q, s = torch.empty(m, blocks * 128, dtype=torch.uint8, device="cuda"), torch.empty(blocks, m, device="cuda")
        torch.cuda.synchronize()
        ctx.add_rmsnorm_fp8(x, x, rocm.BF16, m, d, wd, 1e-6, total, q, s, zero_centered=False)
        ctx.sync()
        wq, ws = to_fp8(y)
        assert np.array_equal(q[at].cpu().numpy(), wq) and np.array_equal(s[:, at].cpu().numpy(), ws)
    else:
        q, s = buffers(m, d)
        ctx.add_rmsnorm_mx4(x, x, rocm.BF16, m, d, wd, 1e-6, total, q, s, zero_centered=False)
        ctx.sync()
        wq, ws = quantize(y)
        tile, lane = at // 16, at % 16
        b = q.view(-1, blocks, 4, 16, 16)[tile, :, :, lane].cpu().numpy()
        codes = np.stack([b & 15, b >> 4], -1).reshape(len(rows), -1)
        scales = s.view(-1, blocks, 4, 16, 4)[at // 64, :, :, lane, tile % 4].cpu().numpy().reshape(len(rows), -1)
        assert np.array_equal(codes, wq) and np.array_equal(scales, ws)
    assert torch.equal(total[at], 2 * x[at])
    del x, total, q, s
    torch.cuda.empty_cache()


@pytest.mark.parametrize("experts,top", [(1, 1), (300, 4)])
def test_the_choice_for_the_most_tokens(ctx, experts, top):
    """2^24 tokens; 300 experts of them are more than 2^32 values."""
    import torch
    rng = np.random.default_rng(experts)
    g = torch.Generator(device="cuda").manual_seed(experts)
    logits = torch.randn(LONGEST, experts, generator=g, device="cuda", dtype=torch.bfloat16)
    ids = torch.full((LONGEST, top), -1, dtype=torch.int32, device="cuda")
    shares = torch.full((LONGEST, top), float("nan"), device="cuda")
    torch.cuda.synchronize()
    rule = rule_of(experts, top)
    ctx.moe_select(rule, logits, rocm.BF16, LONGEST, None, ids, shares)
    ctx.sync()
    at = torch.from_numpy(ends(rng, 100, LONGEST, 100)).cuda()
    want_ids, want = chosen(rule, logits[at].float().cpu().numpy(), None)
    assert np.array_equal(ids[at].cpu().numpy(), want_ids)
    err = np.abs(shares[at].double().cpu().numpy() - want)
    assert (err <= (2.0 ** -24 + 2.0 ** -40) * np.abs(want)).all()
    assert int(ids.min()) >= 0 and torch.isfinite(shares).all()
    del logits, ids, shares
    torch.cuda.empty_cache()
