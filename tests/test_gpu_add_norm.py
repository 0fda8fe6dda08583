"""The residual's addition, the RMS norm and the codes of its rows in one call, against the definition: h, the norm's
factor and the normed values are f32 (or T) roundings of stated quantities, so that codes and scales are compared bit by
bit. The factor's sum of squares is held in 64 bits on both sides; its order decides only where 1 / sqrt lies within
2^-40 of a rounding border, which no row here does."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import bits_equal, dev, empty, host
from tests.test_gpu_fp8 import DTYPES, _torch, quantize as to_fp8, rows_to
from tests.test_gpu_mx4 import quantize as to_mx4, unpack

pytestmark = pytest.mark.gpu


def definition(x, r, w, eps, centered, dtype):
    """(h, y) as f32 arrays of rows x and r of `dtype`, given as f32."""
    import torch
    h = x if r is None else rows_to(x + r, dtype)[1]
    wide = h.astype(np.float64)
    with np.errstate(all="ignore"):
        i = (1 / np.sqrt((wide * wide).sum(1, keepdims=True) / x.shape[1] + np.float64(np.float32(eps)))).astype(np.float32)
        y = (h * i) * (np.float32(1) + w if centered else w)
    return h, y.astype(np.float32)


def call(ctx, form, x, r, dtype, m, d, w, eps, centered, total, y):
    """(codes, scales) as the definition lays them out."""
    import torch
    if form == "fp8":
        g = -(-d // 128)
        q, s = empty((m, g * 128), torch.uint8), empty((g, m), torch.float32)
        ctx.add_rmsnorm_fp8(x, r, dtype, m, d, w, eps, total, q, s, y=y, zero_centered=centered)
        return host(ctx, q), host(ctx, s)
    q, s = (empty((b,), torch.uint8) for b in rocm.mx4_bytes(m, d))
    ctx.add_rmsnorm_mx4(x, r, dtype, m, d, w, eps, total, q, s, y=y, zero_centered=centered)
    return unpack(host(ctx, q), host(ctx, s), m, d)


SHAPES = [(1, 1), (1, 128), (2, 31), (3, 129), (5, 1000), (17, 2048), (16, 2056), (70, 1111), (4, 4096), (3, 4104),
          (2, 8192), (3, 8200), (2, 20001), (130, 96)]


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", SHAPES)
def test_codes_and_sums_are_the_definition_s(ctx, form, dtype, m, d):
    import torch
    rng = np.random.default_rng(m * 11 + d)
    xd, x = rows_to((rng.standard_normal((m, d)) * np.exp(rng.standard_normal((1, d)))).astype(np.float32), dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32) * 3, dtype)
    w = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    for residual, keeps, centered in ((True, True, False), (True, False, True), (False, False, False)):
        total, y = empty((m, d), _torch(dtype)), empty((m, d), _torch(dtype))
        total.fill_(7)
        torch.cuda.synchronize()
        codes, scales = call(ctx, form, xd, rd if residual else None, dtype, m, d, dev(w), 1e-6, centered,
                             total if keeps else None, y)
        h, want = definition(x, r if residual else None, w, 1e-6, centered, dtype)
        wq, ws = to_fp8(want) if form == "fp8" else to_mx4(want)
        assert bits_equal(scales, ws)
        assert np.array_equal(codes, wq)
        assert np.array_equal(host(ctx, y.float()), rows_to(want, dtype)[1])
        assert (host(ctx, total.float()) == (h if keeps else 7)).all()


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [300, 9000])
def test_in_place(ctx, form, dtype, d):
    """The sum in the residual's place and the normed rows in x's, as a decoder keeps them."""
    rng = np.random.default_rng(d)
    m = 9
    xd, x = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    w = rng.standard_normal(d).astype(np.float32)
    codes, scales = call(ctx, form, xd, rd, dtype, m, d, dev(w), 1e-5, True, rd, xd)
    h, y = definition(x, r, w, 1e-5, True, dtype)
    wq, ws = to_fp8(y) if form == "fp8" else to_mx4(y)
    assert np.array_equal(codes, wq) and bits_equal(scales, ws)
    assert np.array_equal(host(ctx, rd.float()), h)
    assert np.array_equal(host(ctx, xd.float()), rows_to(y, dtype)[1])
    # without a residual, the normed rows over x
    xd, x = rows_to(x, dtype)
    codes, scales = call(ctx, form, xd, None, dtype, m, d, dev(w), 1e-5, True, None, xd)
    _, y = definition(x, None, w, 1e-5, True, dtype)
    wq, ws = to_fp8(y) if form == "fp8" else to_mx4(y)
    assert np.array_equal(codes, wq) and bits_equal(scales, ws)
    assert np.array_equal(host(ctx, xd.float()), rows_to(y, dtype)[1])


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [260, 8300])
def test_a_row_that_is_not_finite_touches_no_other(ctx, form, dtype, d):
    rng = np.random.default_rng(6)
    m = 12
    x = rng.standard_normal((m, d)).astype(np.float32)
    x[1, 3], x[4, d - 1], x[7, 200] = np.nan, np.inf, -np.inf
    xd, x = rows_to(x, dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    w = np.ones(d, np.float32)
    codes, scales = call(ctx, form, xd, rd, dtype, m, d, dev(w), 1e-6, False, None, None)
    _, y = definition(x, r, w, 1e-6, False, dtype)
    rows = scales.T if form == "fp8" else scales
    nan = np.isnan(rows.astype(np.float32)) if form == "fp8" else rows == 255
    assert nan.any(1).tolist() == [i in (1, 4, 7) for i in range(m)]
    good = [i for i in range(m) if i not in (1, 4, 7)]
    wq, ws = to_fp8(y) if form == "fp8" else to_mx4(y)
    assert np.array_equal(codes[good], wq[good])
    assert np.array_equal(rows[good], (ws.T if form == "fp8" else ws)[good])


def test_rows_of_nothing_and_the_ends_of_f32(ctx):
    rng = np.random.default_rng(8)
    m, d = 5, 1030
    x = rng.standard_normal((m, d)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-30)
    x[2] *= np.float32(1e30)      # squares past f32
    x[3] *= np.float32(1e-42)     # subnormals
    w = np.ones(d, np.float32)
    for form in ("fp8", "mx4"):
        codes, scales = call(ctx, form, dev(x), None, rocm.F32, m, d, dev(w), 1e-6, False, None, None)
        _, y = definition(x, None, w, 1e-6, False, rocm.F32)
        wq, ws = to_fp8(y) if form == "fp8" else to_mx4(y)
        assert np.array_equal(codes, wq) and bits_equal(scales, ws)


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_odd_addresses_and_bytes_around_the_outputs_left_alone(ctx, form, dtype):
    import torch
    rng = np.random.default_rng(9)
    m, d, guard = 20, 333, 5

    def within(fill):
        whole = torch.full((m * d + 2 * guard,), fill, dtype=_torch(dtype), device="cuda")
        return whole, whole[guard:guard + m * d].view(m, d)

    xs, x = within(0.0)
    rs, r = within(0.0)
    totals, total = within(7.0)
    ys, y = within(7.0)
    ws = torch.zeros(d + 1, device="cuda")
    w = ws[1:]
    x.copy_(torch.from_numpy(rng.standard_normal((m, d)).astype(np.float32)))
    r.copy_(torch.from_numpy(rng.standard_normal((m, d)).astype(np.float32)))
    w.copy_(torch.from_numpy(rng.standard_normal(d).astype(np.float32)))
    torch.cuda.synchronize()
    codes, scales = call(ctx, form, x, r, dtype, m, d, w, 1e-6, False, total, y)
    h, want = definition(x.float().cpu().numpy(), r.float().cpu().numpy(), w.cpu().numpy(), 1e-6, False, dtype)
    wq, wsc = to_fp8(want) if form == "fp8" else to_mx4(want)
    assert np.array_equal(codes, wq) and bits_equal(scales, wsc)
    assert np.array_equal(host(ctx, total.float()), h)
    for whole in (totals, ys):
        assert (whole[:guard] == 7).all() and (whole[-guard:] == 7).all()


def test_refusals(ctx):
    import torch
    m, d = 4, 256
    x, w = torch.zeros(m, d, device="cuda"), torch.zeros(d, device="cuda")
    q8, s8 = empty((m, d), torch.uint8), empty((2, m), torch.float32)
    q4, s4 = (empty((b,), torch.uint8) for b in rocm.mx4_bytes(m, d))
    for name, q, s in (("add_rmsnorm_fp8", q8, s8), ("add_rmsnorm_mx4", q4, s4)):
        norm = getattr(ctx, name)

        def refused(code, *args, **kw):
            with pytest.raises(rocm.DzError) as e:
                norm(*args, **kw)
            assert e.value.code == code, args

        refused("INVALID_REQUEST", None, x, rocm.F32, m, d, w, 1e-6, None, q, s)
        refused("INVALID_REQUEST", x, x, rocm.F32, m, d, None, 1e-6, None, q, s)
        refused("INVALID_REQUEST", x, x, rocm.F32, m, d, w, 1e-6, None, None, s)
        refused("INVALID_REQUEST", x, x, rocm.F32, m, d, w, 1e-6, None, q, None)
        refused("INVALID_REQUEST", x, None, rocm.F32, m, d, w, 1e-6, x, q, s)
        refused("INVALID_PARAMETERS", x, x, 3, m, d, w, 1e-6, None, q, s)
        refused("INVALID_PARAMETERS", x, x, rocm.F32, m, 0, w, 1e-6, None, q, s)
        refused("INVALID_PARAMETERS", x, x, rocm.F32, m, (1 << 20) + 1, w, 1e-6, None, q, s)
        for eps in (-1e-6, float("nan"), float("inf")):
            refused("INVALID_PARAMETERS", x, x, rocm.F32, m, d, w, eps, None, q, s)
        refused("INVALID_PARAMETERS", x, x, rocm.F32, m, d, w, 1e-6, None, q, s, zero_centered=2)
        refused("INVALID_PARAMETERS", x, x, rocm.F32, m, d, w, 1e-6, None, q.data_ptr() + 8, s)
        refused("INPUT_TOO_LONG", x, x, rocm.F32, (1 << 24) + 1, d, w, 1e-6, None, q, s)
        norm(None, None, rocm.F32, 0, d, None, 1e-6, None, None, None)
    with pytest.raises(rocm.DzError) as e:
        ctx.add_rmsnorm_mx4(x, x, rocm.F32, m, d, w, 1e-6, None, q4, s4.data_ptr() + 4)
    assert e.value.code == "INVALID_PARAMETERS"


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_norm_then_the_products_on_its_codes(ctx, dtype):
    """The codes are those that the products make of the normed rows by themselves."""
    import torch
    rng = np.random.default_rng(12)
    m, d, n = 37, 520, 200
    xd, x = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    w = rng.standard_normal(d).astype(np.float32)
    _, y = definition(x, r, w, 1e-6, True, dtype)
    yd = dev(y)
    values = dev((rng.standard_normal((n, d)) * 0.05).astype(np.float32))
    w8, w4 = ctx.fp8_weight_quantize(values, rocm.F32, n, d), ctx.mx4_weight_quantize(values, rocm.F32, n, d)
    q8, s8 = empty((m, 640), torch.uint8), empty((5, m), torch.float32)
    q4, s4 = (empty((b,), torch.uint8) for b in rocm.mx4_bytes(m, d))
    got, want = [empty((m, n), torch.float32) for _ in range(2)], [empty((m, n), torch.float32) for _ in range(2)]
    ctx.add_rmsnorm_fp8(xd, rd, dtype, m, d, dev(w), 1e-6, None, q8, s8)
    ctx.fp8_linear_q8(w8, q8, s8, m, got[0], rocm.F32)
    ctx.add_rmsnorm_mx4(xd, rd, dtype, m, d, dev(w), 1e-6, None, q4, s4)
    ctx.mx4_linear_q4(w4, q4, s4, m, got[1], rocm.F32)
    ctx.fp8_linear(w8, yd, rocm.F32, m, want[0], rocm.F32)
    ctx.mx4_linear(w4, yd, rocm.F32, m, want[1], rocm.F32)
    ctx.sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.abs().max() > 0
    w8.free()
    w4.free()
