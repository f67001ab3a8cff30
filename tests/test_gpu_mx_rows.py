"""The norm and its gradient over more rows than the chip takes at once: the forms that a prompt or a training step takes (more than 444 rows), and rings
of the gradient that come round more than once, against 64 bits."""
import numpy as np
import pytest

from spoc_b200 import _lib as L
from spoc_b200.plugin import _check
from tests import mx_ref as R
from tests.test_gpu_mx import keep, loud, norm_inputs, run_backward, run_norm  # noqa: F401  (a fixture among them)
from tests.test_gpu_mx_range import check_gradient

pytestmark = pytest.mark.gpu
ROWS, SMS = 600, 148


@pytest.mark.parametrize("fmt", [0, R.FP8, R.FP4])
@pytest.mark.parametrize("cols", [100, 255, 513, 1000, 1001, 1024, 1025, 2047, 2048, 3000, 4095, 4096, 4100, 8191, 8192, 12001, 16384, 20004, 32769])
def test_norm_of_many_rows(keep, device, cols, fmt):  # noqa: F811
    """A warp a row, blocks of every width and rows read twice; whole vectors, broken ones, and rows that start off 16 bytes."""
    x, r, w = norm_inputs(np.random.default_rng(cols), ROWS, cols)
    r = r if cols % 5 else None
    pad, offset, in_place = [(0, 0, "residual" if r is not None else "x"), (3, 1, "x"), (4, 0, None)][cols % 3]
    s, y, q = run_norm(keep, device, x, r, w, 1e-5, fmt, pad, offset, in_place)
    h, want = R.rmsnorm(x, r, w, 1e-5)
    assert np.array_equal(s, h)
    # the scale is two roundings off, and each of two products one: 4 of 2^-24
    assert np.all(np.abs(y - want) <= 2.0 ** -22 * np.abs(want))
    if fmt:
        codes, scales = R.quantize(want, fmt)
        assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("rows", [3, 500])
@pytest.mark.parametrize("cols,offset", [(96, 0), (700, 1), (1500, 0), (4001, 0), (8000, 0), (33000, 0), (33001, 1)])
def test_norm_over_both_operands(keep, device, rows, cols, offset):  # noqa: F811
    """sum and y take the places of x and the residual, either way round, and y alone that of x."""
    x, r, w = norm_inputs(np.random.default_rng(cols), rows, cols)
    h, want = R.rmsnorm(x, r, w, 1e-5)
    codes, scales = R.quantize(want, R.FP8)
    wd = keep.f32(w, offset=offset)
    for s_over, y_over in (("x", "r"), ("r", "x"), (None, "x"), (None, "r")):
        d = {"x": keep.f32(x, offset=offset), "r": keep.f32(r, offset=offset)}
        q = keep.mx(R.FP8, rows, cols)
        _check(L.load().sb200_rmsnorm_f32(device.id, 0, rows, cols, d["x"].ptr, cols, d["r"].ptr, cols, wd.ptr, 1e-5, d[s_over].ptr if s_over else 0,
                                          cols if s_over else 0, d[y_over].ptr, cols, R.FP8, q.codes.ptr, q.scales.ptr))
        y = d[y_over].download().reshape(rows, cols)
        assert np.all(np.abs(y - want) <= 2.0 ** -22 * np.abs(want)), (s_over, y_over)
        if s_over:
            assert np.array_equal(d[s_over].download().reshape(rows, cols), h)
        else:
            other = "r" if y_over == "x" else "x"
            assert np.array_equal(d[other].download().reshape(rows, cols), {"x": x, "r": r}[other])
        got = q.download()
        assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales)


# longest row of a group, groups a block, stages of its ring
RINGS = [(128, 32, 4), (256, 16, 4), (512, 8, 4), (1024, 4, 4), (2048, 4, 2), (4096, 2, 2), (8192, 1, 2)]


@pytest.mark.parametrize("cols", [60, 125, 200, 253, 400, 511, 1000, 1023, 1500, 2047, 3000, 4095, 4100, 8191, 8192])
def test_gradient_of_rows_that_come_round(keep, device, cols):  # noqa: F811
    """Every stage of every group's ring is filled three times, for some of them once more."""
    _, groups, stages = next(ring for ring in RINGS if cols <= ring[0])
    at_once = SMS * groups
    rows = at_once * (2 * stages + 1) + at_once // 3
    rng = np.random.default_rng(cols)
    h, w = loud(rng, rows, cols), rng.normal(size=cols).astype(np.float32)
    dy, ds = loud(rng, rows, cols), loud(rng, rows, cols) if cols % 2 else None
    h[rows // 2] *= np.float32(1e20)      # one row that is summed again beside the others
    pad, offset, in_place = [(0, 0, "dy"), (3, 1, None), (4, 0, "sum")][cols % 3]
    got = run_backward(keep, device, h, w, dy, ds, 1e-5, pad, offset, in_place)
    # additions on the way of a value of dweight: the rows of its group, the groups, every eighth part, eight of those
    check_gradient(got, h, w, dy, ds, 1e-5, 2 * stages + 2 + groups + -(-SMS // 8) + 8)
