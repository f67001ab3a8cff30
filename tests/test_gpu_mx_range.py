"""The norm and its gradient from float32's smallest values to its largest, against 64 bits."""
import numpy as np
import pytest

from tests import mx_ref as R
from tests.test_gpu_mx import keep, run_backward, run_norm  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24      # half a step of float32


def check_gradient(got, h, w, dy, dsum, eps, additions=None):
    """In units of U.  A float32 sum adds a value in 28 roundings at most (three within four values, four fours, five steps over a warp, sixteen warps), so
    that r is off by 14, 2 of the mean's own and 3 of the root: 19; n = h r by 20, g = dy w by 1, mean(g n) by 28 + 1 + 19 and three products, 51
    of mean(|g n|); r (g - n mean(g n)) by 1 + 1 + 20 of |g| and 71 + 2 + 20 of |n mean|, the addition of dsum by one more: 94.  Results below 2^-126
    are off by half of 2^-149 for each of the last two besides.  dweight adds a row at a time, or as few as `additions` says; the
    zeros of blocks without a row add exactly."""
    dx, dw = R.rmsnorm_backward(h, w, dy, dsum, eps)
    h, w, dy = (v.astype(np.float64) for v in (h, w, dy))
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, g = np.abs(h * r), np.abs(dy * w)
    size = r * (g + n * (g * n).mean(-1, keepdims=True)) + (0 if dsum is None else np.abs(dsum))
    assert np.all(np.abs(got[0] - dx) <= 94 * U * size + 2.0 ** -149)
    assert np.all(np.abs(got[1] - dw) <= ((additions or h.shape[0]) + 21) * U * (np.abs(dy) * n).sum(0))


# every width of a warp's, a block's and a cluster's row, and rows read twice
@pytest.mark.parametrize("cols", [1, 33, 128, 250, 400, 512, 1000, 2048, 4096, 4099, 8192, 9000, 20004, 65536, 65540, 70001])
def test_gradient_of_rows_from_the_smallest_to_the_largest(keep, device, cols):  # noqa: F811
    """Rows of 1e-37 to 1e37, whose squares lie up to 2^37 times past either end of float32, side by side."""
    rng = np.random.default_rng(cols)
    scale = np.array([1e-37, 1e-30, 1e-24, 1e-19, 1e-18, 1.0, 6e16, 3e17, 1e18, 1e19, 1e25, 1e31, 5e36])[:, None]
    rows = scale.size
    h = (rng.choice([-1.0, 1.0], (rows, cols)) * rng.uniform(1.0, 1.8, (rows, cols)) * scale).astype(np.float32)
    w, dy = rng.normal(size=cols).astype(np.float32), rng.normal(size=(rows, cols)).astype(np.float32)
    dsum = (rng.normal(size=(rows, cols)) / scale).astype(np.float32) if cols % 2 else None
    pad, offset, in_place = [(0, 0, "sum"), (3, 1, None), (4, 0, "dy")][cols % 3]
    check_gradient(run_backward(keep, device, h, w, dy, dsum, 0.0, pad, offset, in_place), h, w, dy, dsum, 0.0)


@pytest.mark.parametrize("eps", [1e-70, 1e-40, 1e-20, 1e30])
@pytest.mark.parametrize("cols", [100, 3000, 9001, 66000])
def test_gradient_of_zeros_and_small_rows_beside_eps(keep, device, cols, eps):  # noqa: F811
    """Where the squares vanish beside eps, n does and r is 1 / sqrt(eps)."""
    rng = np.random.default_rng(cols)
    h = (rng.normal(size=(6, cols)) * np.array([0.0, 1e-44, 1e-37, 1e-30, 1.0, 1e20])[:, None]).astype(np.float32)
    w, dy = rng.normal(size=cols).astype(np.float32), rng.normal(size=(6, cols)).astype(np.float32)
    check_gradient(run_backward(keep, device, h, w, dy, None, eps), h, w, dy, None, eps)


def test_gradient_of_large_gradients(keep, device):  # noqa: F811
    """Products of h and g past float32, whose mean is an ordinary number of g's size."""
    rng = np.random.default_rng(3)
    h = (rng.normal(size=(7, 700)) * 1e25).astype(np.float32)
    w, dy = rng.normal(size=700).astype(np.float32), (rng.normal(size=(7, 700)) * 1e20).astype(np.float32)
    check_gradient(run_backward(keep, device, h, w, dy, None, 1e-5), h, w, dy, None, 1e-5)


@pytest.mark.parametrize("fmt", [0, R.FP8, R.FP4])
@pytest.mark.parametrize("eps", [5e-324, 1e-300, 1e-140, 1e-120, 1e-100, 1e-30, 1e300, float("inf")])
@pytest.mark.parametrize("cols", [100, 1500, 33000])
def test_norm_of_zeros_beside_any_eps(keep, device, cols, eps, fmt):  # noqa: F811
    """A row of zeros has the norm zero wherever eps is not; rows beside it are what they are.  2^-22: the scale is off by two units of U, two products by one each."""
    rng = np.random.default_rng(cols)
    x = (rng.normal(size=(5, cols)) * np.array([0.0, 1.0, 0.0, 1e-44, 1e30])[:, None]).astype(np.float32)
    w = rng.normal(size=cols).astype(np.float32)
    _, y, q = run_norm(keep, device, x, None, w, eps, fmt, 1)
    want = R.rmsnorm(x, None, w, eps)[1]
    assert np.all(np.abs(y - want) <= 2.0 ** -22 * np.abs(want) + 2.0 ** -148 * np.maximum(1, np.abs(w)))
    assert np.all(y[[0, 2]] == 0)
    if fmt:
        codes, scales = R.quantize(want, fmt)
        assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("cols", [1, 32, 33, 100, 130, 600, 1057, 2100, 4097, 33000])
def test_rows_that_are_not_numbers_leave_what_is_past_them_zero(keep, device, cols, fmt):  # noqa: F811
    """Codes and scales past K are zeros whatever the row: NaN, infinite, or zero beside an eps of zero."""
    rng = np.random.default_rng(cols)
    x, w = rng.normal(size=(5, cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    x[0, 0], x[1, cols // 2], x[2] = np.nan, np.inf, 0.0
    _, _, (codes, scales) = run_norm(keep, device, x, None, w, 0.0, fmt)
    with np.errstate(invalid="ignore"):
        want_codes, want_scales = R.quantize(R.rmsnorm(x, None, w, 0.0)[1], fmt)
    assert np.array_equal(scales, want_scales)
    assert np.array_equal(codes[3:], want_codes[3:])
    per_byte = 2 if fmt == R.FP4 else 1
    assert not codes[:, -(-cols // per_byte):].any()
    if cols % per_byte:
        assert not (codes[:, cols // per_byte] >> 4).any()


def test_a_clamp_makes_zero_of_nan(keep, device):  # noqa: F811
    """Scales of NaN show in a product, and are zeros behind SB200_ACT_RELU, as in the product of float32."""
    a, b = np.ones((5, 64)), np.ones((7, 64))
    a[2, 3] = np.nan
    A, B, d = keep.mx(R.FP8, 5, 64, R.quantize(a, R.FP8)), keep.mx(R.FP4, 7, 64, R.quantize(b, R.FP4)), keep.out(35)
    want = np.full((5, 7), 64.0)
    for act, nan in ((0, np.nan), (1, 0.0)):
        want[2] = nan
        R.gemm_mx(device, A, B, d, act=act)
        keep.backend.Device.synchronize(device)
        assert np.array_equal(d.download().reshape(5, 7), want, equal_nan=True)
        x, y = keep.f32(a.astype(np.float32)), keep.f32(np.ascontiguousarray(b.T).astype(np.float32))
        assert R.L.load().sb200_gemm_f32(device.id, 0, R.L.MODE_3XTF32, 5, 7, 64, x.ptr, 64, y.ptr, 7, d.ptr, 7, 1.0, 0, 0, 0.0, 0, act) == 0
        keep.backend.Device.synchronize(device)
        assert np.array_equal(d.download().reshape(5, 7), want, equal_nan=True)


@pytest.mark.parametrize("fmt", R.FORMATS)
def test_norms_past_float32_are_infinite(keep, device, fmt):  # noqa: F811
    """Weights near float32's largest: blocks with a y of 2^128 and more have the scale NaN, the others the codes of 64 bits."""
    rng = np.random.default_rng(fmt)
    x = rng.normal(size=(40, 320)).astype(np.float32)
    w = np.where(np.arange(320) // 32 % 2 == 0, 3e38, 1e38).astype(np.float32)
    _, y, (codes, scales) = run_norm(keep, device, x, None, w, 1e-5, fmt)
    want = R.rmsnorm(x, None, w, 1e-5)[1]
    past = np.abs(want) >= 2.0 ** 128
    assert past.any() and np.all(np.isinf(y[past]))
    want_codes, want_scales = R.quantize(np.where(past, np.inf, want), fmt)
    assert 0 < (want_scales == 255).sum() < want_scales.size / 2 and np.array_equal(scales, want_scales)
    fine = ~np.pad(past, ((0, 0), (0, 64))).reshape(40, 12, 32).any(-1)
    per_block = 16 if fmt == R.FP4 else 32
    assert np.array_equal(codes.reshape(40, 12, per_block)[fine], want_codes.reshape(40, 12, per_block)[fine])
