"""The norm with codes on the forms that a row's length and the number of rows pick: rows that are read twice, rows of a
wave each, and rows whose normed values are not finite. Bit by bit against the definition of test_gpu_add_norm."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import bits_equal, dev, empty, host
from tests.test_gpu_add_norm import call, definition
from tests.test_gpu_fp8 import DTYPES, _torch, quantize as to_fp8, rows_to
from tests.test_gpu_mx4 import quantize as to_mx4

pytestmark = pytest.mark.gpu


def coded(form, y):
    return to_fp8(y) if form == "fp8" else to_mx4(y)


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [12288, 12289, 13001, 16384])
@pytest.mark.parametrize("places", ["residual and x", "x and residual", "x and another", "no sum, over x",
                                    "no sum, over the residual", "neither", "no residual"])
def test_long_rows_in_place(ctx, form, dtype, d, places):
    """Rows past 12288 read h a second time, from where it was stored, or x and the residual again: in every place that
    the sum and the normed rows may take."""
    rng = np.random.default_rng(d)
    m = 7
    xd, x = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    other = empty((m, d), _torch(dtype))
    w = rng.standard_normal(d).astype(np.float32)
    total, out = {"residual and x": (rd, xd), "x and residual": (xd, rd), "x and another": (xd, other),
                  "no sum, over x": (None, xd), "no sum, over the residual": (None, rd), "neither": (None, None),
                  "no residual": (None, xd)}[places]
    residual = None if places == "no residual" else rd
    codes, scales = call(ctx, form, xd, residual, dtype, m, d, dev(w), 1e-5, True, total, out)
    h, y = definition(x, None if residual is None else r, w, 1e-5, True, dtype)
    wq, ws = coded(form, y)
    assert np.array_equal(codes, wq) and bits_equal(scales, ws)
    if total is not None:
        assert np.array_equal(host(ctx, total.float()), h)
    if out is not None:
        assert np.array_equal(host(ctx, out.float()), rows_to(y, dtype)[1])
    for t, before in ((xd, x), (rd, r)):
        if t is not total and t is not out:
            assert np.array_equal(host(ctx, t.float()), before)


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [12300, 13001])
def test_a_long_row_that_is_not_finite_touches_no_other(ctx, form, dtype, d):
    rng = np.random.default_rng(6)
    m = 12
    x = rng.standard_normal((m, d)).astype(np.float32)
    x[1, 3], x[4, d - 1], x[7, 12290] = np.nan, np.inf, -np.inf
    xd, x = rows_to(x, dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    w = np.ones(d, np.float32)
    _, y = definition(x, r, w, 1e-6, False, dtype)
    wq, ws = coded(form, y)
    good = [i for i in range(m) if i not in (1, 4, 7)]
    for keeps in (False, True):
        codes, scales = call(ctx, form, xd, rd, dtype, m, d, dev(w), 1e-6, False, rd if keeps else None, None)
        rows, want = (scales.T, ws.T) if form == "fp8" else (scales, ws)
        nan = np.isnan(rows) if form == "fp8" else rows == 255
        assert nan.any(1).tolist() == [i in (1, 4, 7) for i in range(m)]
        assert np.array_equal(codes[good], wq[good]) and np.array_equal(rows[good], want[good])


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", [(4099, 517), (4096, 1023), (4099, 1029), (4101, 2047)])
def test_many_rows_of_a_wave_each(ctx, form, dtype, m, d):
    """The last workgroup's waves are not all rows, the last vectors not all values; sum and normed rows kept apart, then
    in the residual's and x's places."""
    rng = np.random.default_rng(m + d)
    xd, x = rows_to((rng.standard_normal((m, d)) * np.exp(rng.standard_normal((1, d)))).astype(np.float32), dtype)
    rd, r = rows_to(rng.standard_normal((m, d)).astype(np.float32), dtype)
    w = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
    h, y = definition(x, r, w, 1e-6, True, dtype)
    wq, ws = coded(form, y)
    kept = rows_to(y, dtype)[1]
    for total, out in ((empty((m, d), _torch(dtype)), empty((m, d), _torch(dtype))), (rd, xd)):
        codes, scales = call(ctx, form, xd, rd, dtype, m, d, dev(w), 1e-6, True, total, out)
        assert np.array_equal(codes, wq) and bits_equal(scales, ws)
        assert np.array_equal(host(ctx, total.float()), h)
        assert np.array_equal(host(ctx, out.float()), kept)


@pytest.mark.parametrize("form", ["fp8", "mx4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [100, 300, 1500, 13001])
def test_normed_values_that_are_not_finite_spoil_their_blocks(ctx, form, dtype, d):
    """A row of zeros without an epsilon is 0 times infinity; a large weight takes a row's values past f32's range: such
    blocks have NaN scales though the row itself is finite, and no other row or block has."""
    rng = np.random.default_rng(d)
    m = 9
    x = rng.standard_normal((m, d)).astype(np.float32)
    x[2] = 0
    x[5, d // 2] = 0
    x[6:, 70] = 9
    w = np.ones(d, np.float32)
    w[70] = 3e38
    xd, x = rows_to(x, dtype)
    for weight in (np.ones(d, np.float32), w):
        codes, scales = call(ctx, form, xd, None, dtype, m, d, dev(weight), 0.0, False, None, None)
        _, y = definition(x, None, weight, 0.0, False, dtype)
        wq, ws = coded(form, y)
        rows, want = (scales.T, ws.T) if form == "fp8" else (scales, ws)
        nan = np.isnan(want) if form == "fp8" else want == 255
        assert nan[2].sum() == -(-d // (128 if form == "fp8" else 32))
        assert (nan[6:].sum(1) == (weight is w)).all()  # channel 70's block alone
        assert np.array_equal(rows, want, equal_nan=form == "fp8")
        assert np.array_equal(codes, wq)
