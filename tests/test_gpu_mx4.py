"""Microscaled 4-bit floating point: its quantization bit by bit, and products against the definition in 64 bits.

Tolerances. Products of codes and their sum over a block of 32 are exact; each block and each partial sum of a split k is
then added in f32, which is off by at most one step, 2^-23, of the magnitudes added. With S = sum |x w| over a row's
values, a product of k values is off by at most (k / 32 + 32) 2^-23 S (32: more than the partial sums of any split)
before the output's own rounding, eps / 2 of the value, or half the smallest subnormal."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import bits_equal, dev, empty, host
from tests.test_gpu_fp8 import DTYPES, EPS, LEAST, _torch, f64, rows_to

pytestmark = pytest.mark.gpu

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def quantize(x):
    """Codes [m x 128 G] and scale bytes [m x 4 G] of f32 rows, as the definition makes them."""
    m, k = x.shape
    g = -(-k // 128)
    v = np.zeros((m, g * 128))
    v[:, :k] = x.astype(np.float64)
    v = v.reshape(m, 4 * g, 32)
    bad = ~np.isfinite(v).all(2)
    v[bad] = 0
    most = np.abs(v).max(2)
    e = np.where(most > 0, np.maximum(np.frexp(most)[1] - 3, -127), -127)
    a = np.abs(v) * 2.0 ** -e[..., None].astype(np.float64)
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    code = np.zeros(a.shape, np.int64)
    for i, edge in enumerate(edges):  # a tie goes to the even code: up to code i + 1 where that is even
        code += (a >= edge) if i % 2 else (a > edge)
    code |= np.where(np.signbit(v), 8, 0)
    code[bad] = 0
    return code.reshape(m, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def unpack(q, s, m, k):
    """The codes [m x 128 G] and scale bytes [m x 4 G] of the native layout."""
    g, tiles, panels = -(-k // 128), -(-m // 16), -(-m // 64)
    b = q.reshape(tiles, g, 4, 16, 16)
    codes = np.stack([b & 15, b >> 4], -1).reshape(tiles, g, 4, 16, 32).transpose(0, 3, 1, 2, 4).reshape(tiles * 16, -1)
    scales = s.reshape(panels, g, 4, 16, 4).transpose(0, 4, 3, 1, 2).reshape(panels * 64, -1)
    return codes[:m], scales[:m]


def values(codes, scales, k):
    """What codes and scale bytes stand for (64 bits)."""
    return (VALUES[codes] * np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, 1))[:, :k]


def buffers(m, k):
    import torch
    return [empty((b,), torch.uint8) for b in rocm.mx4_bytes(m, k)]


def make_weight(ctx, rng, n, k, spread=0.5):
    """(handle, its values in 64 bits) of a weight whose blocks differ in size."""
    codes = rng.integers(0, 16, (n, k)).astype(np.uint8)
    scales = np.clip(np.rint(120 + spread * rng.standard_normal((n, -(-k // 32)))), 1, 250).astype(np.uint8)
    padded = np.zeros((n, k + k % 2), np.uint8)
    padded[:, :k] = codes
    if k % 2:
        padded[:, k] = 7  # what stands past an odd row's end is no value
    w = ctx.mx4_weight(dev(padded[:, 0::2] | padded[:, 1::2] << 4), dev(scales), n, k)
    wide = np.zeros((n, -(-k // 32) * 32), np.uint8)
    wide[:, :k] = codes
    return w, values(wide, scales, k)


def product(x, w):
    """(y, S) in 64 bits."""
    import torch
    a, b = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    return (a @ b.t()).cpu().numpy(), (a.abs() @ b.abs().t()).cpu().numpy()


def check(got, want, mags, k, dtype):
    tol = (1 + EPS[dtype]) * (k / 32 + 32) * 2.0 ** -23 * mags + EPS[dtype] * np.abs(want) + LEAST[dtype]
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 33), (16, 128), (17, 1000), (40, 1111), (65, 95), (130, 520)])
def test_quantize_gives_the_definition_s_codes_and_scales(ctx, dtype, m, k):
    rng = np.random.default_rng(m * 5 + k)
    x = rng.standard_normal((m, k)).astype(np.float32) * np.exp(2 * rng.standard_normal((m, k))).astype(np.float32)
    x[0, : k // 2] = 0
    if m > 2:
        x[2] = 0  # a row of nothing
    xd, xf = rows_to(x, dtype)
    q, s = buffers(m, k)
    ctx.mx4_quantize(xd, dtype, m, k, q, s)
    codes, scales = unpack(host(ctx, q), host(ctx, s), m, k)
    want_codes, want_scales = quantize(xf)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)


def test_quantize_on_the_borders_of_codes_and_scales(ctx):
    """Every midpoint and its f32 neighbours at every scale; largest values next to a power of two; the ends of f32."""
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 6.0, 7.0, 7.5])
    rows = []
    for e in range(-149, 128):
        v = np.zeros(96)
        v[0], v[32], v[64] = 4.0, 7.9, 6.0
        v[1:12], v[33:44], v[65:76] = mid, -mid, mid
        with np.errstate(over="ignore", under="ignore"):
            r = (v * 2.0 ** (e - 2)).astype(np.float32)
        r[1:12] = np.nextafter(r[1:12], np.float32(0))
        r[65:76] = np.nextafter(r[65:76], np.float32(np.inf))
        rows.append(np.where(np.isfinite(r), r, np.float32(3.4028235e38)))
    x = np.array(rows, np.float32)
    m, k = x.shape
    q, s = buffers(m, k)
    ctx.mx4_quantize(dev(x), rocm.F32, m, k, q, s)
    codes, scales = unpack(host(ctx, q), host(ctx, s), m, k)
    want_codes, want_scales = quantize(x)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes)


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_are_not_finite(ctx, dtype):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 200)).astype(np.float32)
    x[1, 5], x[2, 63], x[3, 199], x[4, 64] = np.nan, np.inf, -np.inf, -np.nan
    xd, xf = rows_to(x, dtype)
    q, s = buffers(6, 200)
    ctx.mx4_quantize(xd, dtype, 6, 200, q, s)
    codes, scales = unpack(host(ctx, q), host(ctx, s), 6, 200)
    want_codes, want_scales = quantize(xf)
    assert (want_scales == 255).sum() == 4
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)


def test_rows_past_the_last_are_left_as_they_were(ctx):
    m, k = 18, 300
    q, s = buffers(m, k)
    q.fill_(0x5a), s.fill_(0xa5)
    x = dev(np.random.default_rng(1).standard_normal((m, k)).astype(np.float32))
    ctx.mx4_quantize(x, rocm.F32, m, k, q, s)
    codes, scales = unpack(host(ctx, q), host(ctx, s), 32, k)
    assert (codes[m:, 0::2] == 0xa).all() and (codes[m:, 1::2] == 5).all()
    assert (host(ctx, s).reshape(3, 4, 16, 4)[:, :, m - 16:, 1] == 0xa5).all()
    assert (host(ctx, s).reshape(3, 4, 16, 4)[:, :, :, 2:] == 0xa5).all()


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 33), (70, 1111), (130, 129)])
def test_weight_from_arrays_then_dequant(ctx, n, k):
    import torch
    w, wide = make_weight(ctx, np.random.default_rng(n + k), n, k, spread=20)
    y = empty((n, k), torch.float32)
    ctx.mx4_dequant(w, y)
    assert bits_equal(host(ctx, y), wide.astype(np.float32))
    assert (w.rows, w.cols, w.device_bytes) == (n, k, sum(rocm.mx4_bytes(n, k)))
    w.free()


def test_dequant_at_the_ends_of_the_scales(ctx):
    import torch
    codes = np.tile(np.arange(16, dtype=np.uint8), 2 * 256).reshape(256, 32)
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)[:255]
    codes = codes[:255]
    w = ctx.mx4_weight(dev(codes[:, 0::2] | codes[:, 1::2] << 4), dev(scales), 255, 32)
    y = empty((255, 32), torch.float32)
    ctx.mx4_dequant(w, y)
    with np.errstate(over="ignore"):
        want = values(codes, scales, 32).astype(np.float32)
    assert bits_equal(host(ctx, y), want)
    w.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (19, 130), (64, 256), (100, 1000)])
def test_weight_quantize_then_dequant(ctx, dtype, n, k):
    import torch
    rng = np.random.default_rng(n)
    vd, vf = rows_to(rng.standard_normal((n, k)).astype(np.float32) * 0.02, dtype)
    w = ctx.mx4_weight_quantize(vd, dtype, n, k)
    y = empty((n, k), torch.float32)
    ctx.mx4_dequant(w, y)
    assert np.array_equal(host(ctx, y), values(*quantize(vf), k).astype(np.float32))
    w.free()


# rows, columns of y, k: a row or a few, a tile and around it, many tiles, k within and past a block, short and long
SHAPES = [(1, 1, 1), (1, 16, 32), (1, 300, 1000), (2, 17, 129), (5, 40, 33), (15, 64, 2050), (16, 128, 128),
          (17, 130, 300), (31, 33, 640), (33, 257, 96), (63, 65, 1111), (64, 256, 512), (65, 31, 4100), (100, 500, 260),
          (129, 129, 129), (200, 1000, 70), (257, 300, 900), (300, 513, 384), (520, 1030, 600)]


@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_against_64_bits(ctx, m, n, k, x_dtype):
    rng = np.random.default_rng(m * 3 + n + k)
    w, wide = make_weight(ctx, rng, n, k)
    xd, xf = rows_to((rng.standard_normal((m, k)) * np.exp(rng.standard_normal((1, k)))).astype(np.float32), x_dtype)
    want, mags = product(values(*quantize(xf), k), wide)
    q, s = buffers(m, k)
    ctx.mx4_quantize(xd, x_dtype, m, k, q, s)
    for y_dtype in DTYPES:
        y, other = empty((m, n), _torch(y_dtype)), empty((m, n), _torch(y_dtype))
        ctx.mx4_linear(w, xd, x_dtype, m, y, y_dtype)
        ctx.mx4_linear_q4(w, q, s, m, other, y_dtype)
        ctx.sync()
        check(f64(y), want, mags, k, y_dtype)
        assert bits_equal(host(ctx, y.float()), host(ctx, other.float()))
    w.free()


VARIANTS = ["rows16", "32x32", "32x32k4", "64x64", "64x64k2", "64x128", "128x128", "256x256"]


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (70, 131, 2600), (300, 70, 1111), (257, 513, 129), (33, 300, 5000)])
def test_every_variant_against_64_bits(ctx, variant, m, n, k):
    rng = np.random.default_rng(m + n + k)
    w, wide = make_weight(ctx, rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    want, mags = product(values(*quantize(x), k), wide)
    q, s = buffers(m, k)
    q.fill_(0x77), s.fill_(255)  # what stands past the rows
    ctx.mx4_quantize(dev(x), rocm.F32, m, k, q, s)
    ctx.select_variant("mx4", variant)
    try:
        for y_dtype in DTYPES:
            y = empty((m, n), _torch(y_dtype))
            ctx.mx4_linear_q4(w, q, s, m, y, y_dtype)
            ctx.sync()
            check(f64(y), want, mags, k, y_dtype)
    finally:
        ctx.select_variant("mx4", "auto")
    w.free()


@pytest.mark.parametrize("y_dtype", [rocm.F32, rocm.BF16])
@pytest.mark.parametrize("k", [1, 200, 513, 640, 1100])
@pytest.mark.parametrize("variant,m,n", [("32x32", 1601, 2900), ("64x64", 1700, 4200), ("64x128", 2100, 5001),
                                         ("256x256", 4100, 4400), ("128x128", 2300, 2200), ("32x32k4", 1001, 1100)])
def test_tiles_in_turn_on_one_workgroup(ctx, variant, m, n, k, y_dtype):
    """More tiles than the units hold at once (the last two forms launch a workgroup each), with fewer 128-blocks of k than
    stages, as many, and an odd number."""
    import torch
    rng = np.random.default_rng(m + k)
    w, wide = make_weight(ctx, rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    want, mags = product(values(*quantize(x), k), wide)
    q, s = buffers(m, k)
    ctx.mx4_quantize(dev(x), rocm.F32, m, k, q, s)
    y = empty((m, n), _torch(y_dtype))
    ctx.select_variant("mx4", variant)
    try:
        for _ in range(2):
            y.fill_(float("nan"))
            torch.cuda.synchronize()
            ctx.mx4_linear_q4(w, q, s, m, y, y_dtype)
            ctx.sync()
            check(f64(y), want, mags, k, y_dtype)
    finally:
        ctx.select_variant("mx4", "auto")
    w.free()


@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 3, 20, 70, 300])
def test_a_row_that_is_not_finite_makes_its_own_outputs_nan(ctx, m, x_dtype):
    import torch
    rng = np.random.default_rng(m)
    n, k = 150, 700
    w, wide = make_weight(ctx, rng, n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    bad = {0: np.nan, m // 2: np.inf, m - 1: -np.inf}
    clean = rows_to(x, x_dtype)[1]
    for r, v in bad.items():
        x[r, (r * 37 + 5) % k] = v
    xd, _ = rows_to(x, x_dtype)
    y = empty((m, n), torch.float32)
    ctx.mx4_linear(w, xd, x_dtype, m, y, rocm.F32)
    got = host(ctx, y)
    want, mags = product(values(*quantize(clean), k), wide)
    good = [r for r in range(m) if r not in bad]
    assert np.isnan(got[list(bad)]).all()
    check(got[good], want[good], mags[good], k, rocm.F32)
    w.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 40, 130])
def test_rows_at_odd_addresses_and_bytes_around_the_output_left_alone(ctx, dtype, m):
    import torch
    rng = np.random.default_rng(9)
    n, k = 77, 333
    w, wide = make_weight(ctx, rng, n, k)
    xs = torch.zeros(m * k + 3, dtype=_torch(dtype), device="cuda")
    x = xs[3:].view(m, k)
    x.copy_(torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)))
    want, mags = product(values(*quantize(x.float().cpu().numpy()), k), wide)
    whole = torch.full((m * n + 66,), 7.0, dtype=_torch(dtype), device="cuda")
    y = whole[33:33 + m * n].view(m, n)
    torch.cuda.synchronize()
    ctx.mx4_linear(w, x, dtype, m, y, dtype)
    ctx.sync()
    check(f64(y), want, mags, k, dtype)
    assert (whole[:33] == 7).all() and (whole[33 + m * n:] == 7).all()
    w.free()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_scales_from_end_to_end_of_their_range(ctx, m):
    """Rows of 2^-120 against weights of 2^60 and the other way round: the scales' sum counts, not each."""
    import torch
    rng = np.random.default_rng(m)
    n, k = 90, 260
    codes = rng.integers(0, 16, (n, 288)).astype(np.uint8)
    codes[:, k:] = 0
    scales = np.full((n, 9), 187, np.uint8)
    scales[45:] = 67
    w = ctx.mx4_weight(dev((codes[:, 0::2] | codes[:, 1::2] << 4)[:, :130]), dev(scales), n, k)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[0::2] *= np.float32(2.0 ** -110)
    x[1::2] *= np.float32(2.0 ** 50)
    y = empty((m, n), torch.float32)
    ctx.mx4_linear(w, dev(x), rocm.F32, m, y, rocm.F32)
    want, mags = product(values(*quantize(x), k), values(codes, scales, k))
    check(host(ctx, y), want, mags, k, rocm.F32)
    w.free()


@pytest.mark.parametrize("y_dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 16, 40, 300])
def test_results_below_the_smallest_normal_value(ctx, m, y_dtype):
    """Outputs of some 2^-130 (f16: 2^-18) are rounded to subnormal values, not to 0. A subnormal f32 sum is off by half
    its last place, 2^-150, for each block that is added."""
    rng = np.random.default_rng(m)
    n, k = 90, 260
    codes = rng.integers(0, 16, (n, 288)).astype(np.uint8)
    codes[:, k:] = 0
    scales = np.full((n, 9), 127 - (16 if y_dtype == rocm.F16 else 50), np.uint8)
    w = ctx.mx4_weight(dev((codes[:, 0::2] | codes[:, 1::2] << 4)[:, :130]), dev(scales), n, k)
    x = rng.standard_normal((m, k)).astype(np.float32) * np.float32(2.0 ** (-8 if y_dtype == rocm.F16 else -88))
    y = empty((m, n), _torch(y_dtype))
    ctx.mx4_linear(w, dev(x), rocm.F32, m, y, y_dtype)
    ctx.sync()
    want, mags = product(values(*quantize(x), k), values(codes, scales, k))
    got = f64(y)
    tol = (1 + EPS[y_dtype]) * ((k / 32 + 32) * (2.0 ** -23 * mags + 2.0 ** -150)) + EPS[y_dtype] * np.abs(want) + LEAST[y_dtype]
    assert (np.abs(got - want) <= tol).all()
    if y_dtype != rocm.BF16:  # whose least value, 2^-133, is as large as these
        assert np.count_nonzero(got) > 0.9 * got.size
    w.free()


def test_refusals(ctx):
    import torch
    n, k, m = 32, 256, 4
    codes, scales = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda"), \
        torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    x, y = torch.zeros(m, k, device="cuda"), torch.zeros(m, n, device="cuda")
    q, s = buffers(m, k)
    torch.cuda.synchronize()
    w = ctx.mx4_weight(codes, scales, n, k)
    wrong = scales.clone()
    wrong[31, 7] = 255
    values_ = torch.zeros(n, k, device="cuda")
    values_[3, 200] = float("inf")
    torch.cuda.synchronize()

    def refused(code, call, *args):
        with pytest.raises(rocm.DzError) as e:
            call(*args)
        assert e.value.code == code, args

    refused("INVALID_CHECKPOINT", ctx.mx4_weight, codes, wrong, n, k)
    refused("INVALID_CHECKPOINT", ctx.mx4_weight_quantize, values_, rocm.F32, n, k)
    for rows, cols in ((0, k), (n, 0), ((1 << 24) + 1, k), (n, (1 << 20) + 1)):
        refused("INVALID_PARAMETERS", ctx.mx4_weight, codes, scales, rows, cols)
        refused("INVALID_PARAMETERS", ctx.mx4_weight_quantize, x, rocm.F32, rows, cols)
    refused("INVALID_REQUEST", ctx.mx4_weight, None, scales, n, k)
    refused("INVALID_REQUEST", ctx.mx4_weight, codes, None, n, k)
    refused("INVALID_REQUEST", ctx.mx4_weight_quantize, None, rocm.F32, n, k)
    refused("INVALID_PARAMETERS", ctx.mx4_weight_quantize, x, 3, 4, k)
    refused("INVALID_REQUEST", ctx.mx4_dequant, w, None)
    for args in ((None, rocm.F32, m, k, q, s), (x, rocm.F32, m, k, None, s), (x, rocm.F32, m, k, q, None)):
        refused("INVALID_REQUEST", ctx.mx4_quantize, *args)
    refused("INVALID_PARAMETERS", ctx.mx4_quantize, x, 5, m, k, q, s)
    refused("INVALID_PARAMETERS", ctx.mx4_quantize, x, rocm.F32, m, 0, q, s)
    refused("INVALID_PARAMETERS", ctx.mx4_quantize, x, rocm.F32, m, (1 << 20) + 1, q, s)
    refused("INPUT_TOO_LONG", ctx.mx4_quantize, x, rocm.F32, (1 << 24) + 1, k, q, s)
    refused("INVALID_PARAMETERS", ctx.mx4_quantize, x, rocm.F32, m, k, q.data_ptr() + 4, s)
    refused("INVALID_PARAMETERS", ctx.mx4_quantize, x, rocm.F32, m, k, q, s.data_ptr() + 4)
    for args in ((None, rocm.F32, m, y, rocm.F32), (x, rocm.F32, m, None, rocm.F32)):
        refused("INVALID_REQUEST", ctx.mx4_linear, w, *args)
    refused("INVALID_PARAMETERS", ctx.mx4_linear, w, x, -1, m, y, rocm.F32)
    refused("INVALID_PARAMETERS", ctx.mx4_linear, w, x, rocm.F32, m, y, 3)
    refused("INPUT_TOO_LONG", ctx.mx4_linear, w, x, rocm.F32, (1 << 24) + 1, y, rocm.F32)
    refused("INVALID_REQUEST", ctx.mx4_linear_q4, w, None, s, m, y, rocm.F32)
    refused("INVALID_REQUEST", ctx.mx4_linear_q4, w, q, None, m, y, rocm.F32)
    refused("INVALID_REQUEST", ctx.mx4_linear_q4, w, q, s, m, None, rocm.F32)
    refused("INVALID_PARAMETERS", ctx.mx4_linear_q4, w, q, s, m, y, 7)
    refused("INVALID_PARAMETERS", ctx.mx4_linear_q4, w, q.data_ptr() + 8, s, m, y, rocm.F32)
    refused("INPUT_TOO_LONG", ctx.mx4_linear_q4, w, q, s, (1 << 24) + 1, y, rocm.F32)
    ctx.mx4_quantize(None, rocm.F32, 0, k, None, None)
    ctx.mx4_linear(w, None, rocm.F32, 0, None, rocm.F32)
    ctx.mx4_linear_q4(w, None, None, 0, None, rocm.F32)
    w.free()


@pytest.mark.parametrize("m", [1, 40, 200])
def test_captured_products_replayed(ctx, m):
    """Two products of one recording take the workspace in turn; every replay gives the eager bits."""
    import torch
    rng = np.random.default_rng(22)
    n, k = 260, 1500
    w, _ = make_weight(ctx, rng, n, k)
    back, _ = make_weight(ctx, rng, n, n)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        x, h, y = empty((m, k), torch.bfloat16), empty((m, n), torch.float32), empty((m, n), torch.bfloat16)
        eager = torch.empty_like(y)
        x.zero_()
        torch.cuda.synchronize()

        def run(out):
            ctx.mx4_linear(w, x, rocm.BF16, m, h, rocm.F32)
            ctx.mx4_linear(back, h, rocm.F32, m, out, rocm.BF16)

        run(y)
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with rocm.capture(graph, stream):
            run(y)
            capture = ctx.capture_id()
        for i in range(4):
            x.copy_(torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            torch.cuda.synchronize()
            run(eager)
            ctx.sync()
            assert y.abs().max() > 0 and torch.equal(y, eager), i
        del graph
        ctx.capture_release(capture)
    finally:
        ctx.set_stream(None)
    w.free()
    back.free()
