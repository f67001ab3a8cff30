"""Microscaled operators and the norm on the GPU against numpy in 64 bits (tests/mx_ref.py).

Codes and scales are compared byte for byte: the definition leaves no freedom.  Tolerances of the products: the tensor core adds the exact products
of a k-step (32 or 64 values) to a float32 accumulator; a step rounds, or cuts, at 2^-23 of a magnitude that the sum of magnitudes bounds, and
so does each sum over a divided k-loop, alpha, beta and the bias: |error| <= (K / 32 + 16) 2^-23 (|alpha| sum |a b| + |beta c| + |bias|).
"""
import ctypes as C

import numpy as np
import pytest

from spoc_b200 import _lib as L
from spoc_b200.plugin import BackendError, _check
from tests import mx_ref as R
from tests.gpu_util import CANARY
from tests.mx_ref import FP4, FP8, FORMATS, Keep, gemm_mx

pytestmark = pytest.mark.gpu


@pytest.fixture
def keep(backend, device):
    with Keep(backend, device) as k:
        yield k
    backend.Device.synchronize(device)


def loud(rng, rows, cols):
    """Normal values, some columns and rows far above the others."""
    return (rng.normal(size=(rows, cols)) * np.exp(2 * rng.normal(size=cols)) * np.exp(3 * rng.normal(size=(rows, 1)))).astype(np.float32)


# ------------------------------------------------------------------ quantisation
SIZES = [(1, 1), (1, 31), (1, 128), (2, 33), (5, 127), (31, 129), (33, 256), (64, 255), (127, 513), (128, 384), (129, 1000), (257, 640), (300, 96)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("transposed", [0, 1])
@pytest.mark.parametrize("pad,offset", [(0, 0), (4, 0), (3, 1)])
@pytest.mark.parametrize("rows,k", SIZES)
def test_quantize(keep, device, fmt, transposed, rows, k, pad, offset):
    v = loud(np.random.default_rng(rows * 1000 + k), rows, k)
    held = v.T if transposed else v
    src = np.full((held.shape[0], held.shape[1] + pad), np.nan, np.float32)     # what lies between the rows is not read
    src[:, :held.shape[1]] = held
    x, q = keep.f32(src, offset=offset), keep.mx(fmt, rows, k)
    _check(L.load().sb200_mx_quantize(device.id, 0, fmt, rows, k, x.ptr, src.shape[1], transposed, q.codes.ptr, q.scales.ptr))
    codes, scales = R.quantize(v, fmt)
    got = q.download()
    assert np.array_equal(got[1], scales)
    assert np.array_equal(got[0], codes)


def special_blocks():
    """Rows of 32 that the rules single out."""
    tiny, big = 2.0 ** -149, float(np.finfo(np.float32).max)
    g8, g4 = R.grid(FP8), R.grid(FP4)
    rows = [np.zeros(32), np.full(32, -0.0), np.full(32, tiny), np.linspace(-1, 1, 32) * 2.0 ** -130, np.full(32, big), np.linspace(-1, 1, 32) * big,
            np.r_[big, np.full(31, tiny)], np.r_[1.0, np.full(31, 2.0 ** -60)], np.r_[np.inf, np.ones(31)], np.r_[np.ones(31), np.nan],
            np.r_[-np.inf, np.zeros(31)], np.r_[511.9, np.linspace(440, 480, 31)], np.r_[7.9, np.linspace(4.9, 7, 31)],
            np.r_[256.0, (g8[1:32] + g8[:31]) / 2], np.r_[448.0, (g8[95:126] + g8[96:127]) / 2], np.r_[4.0, np.tile((g4[1:] + g4[:-1]) / 2, 5)[:31]],
            np.r_[2.0, -np.linspace(0, 2, 31)], np.full(32, 2.0 ** -127), np.r_[2.0 ** -119, np.linspace(0, 2.0 ** -120, 31)]]
    with np.errstate(invalid="ignore"):
        return np.array(rows).astype(np.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("transposed", [0, 1])
def test_quantize_special_values(keep, device, fmt, transposed):
    """Zeros, values beside the smallest and the largest, middles between codes, what is held at the largest, NaN and infinities."""
    v = special_blocks()
    rows = v.shape[0]
    x, q = keep.f32(np.ascontiguousarray(v.T if transposed else v)), keep.mx(fmt, rows, 32)
    _check(L.load().sb200_mx_quantize(device.id, 0, fmt, rows, 32, x.ptr, rows if transposed else 32, transposed, q.codes.ptr, q.scales.ptr))
    codes, scales = R.quantize(v, fmt)
    got = q.download()
    assert np.array_equal(got[1], scales)
    fine = np.isfinite(v).all(-1)
    assert np.array_equal(got[0][fine], codes[fine])
    out = keep.out(rows * 32)
    _check(L.load().sb200_mx_dequantize(device.id, 0, fmt, rows, 32, q.codes.ptr, q.scales.ptr, out.ptr, 32))
    back = out.download().reshape(rows, 32)
    assert np.isnan(back[~fine]).all() and np.array_equal(back[fine], R.values(codes, scales, fmt, 32)[fine].astype(np.float32))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k,pad,offset", [(1, 1, 0, 0), (3, 130, 0, 0), (129, 256, 4, 0), (200, 999, 0, 0), (7, 64, 1, 3)])
def test_dequantize_every_code(keep, device, fmt, rows, k, pad, offset):
    rng = np.random.default_rng(k)
    codes = rng.integers(0, 256, (rows, -(-k // 128) * (64 if fmt == FP4 else 128)), dtype=np.uint8)
    scales = rng.integers(0, 256, R.mx_bytes(fmt, rows, k)[1], dtype=np.uint8)
    q, out = keep.mx(fmt, rows, k, (codes, scales)), keep.out(rows * (k + pad), offset=offset)
    _check(L.load().sb200_mx_dequantize(device.id, 0, fmt, rows, k, q.codes.ptr, q.scales.ptr, out.ptr, k + pad))
    got = out.download().reshape(rows, k + pad)
    with np.errstate(over="ignore"):        # 448 * 2^127 and the like are infinite as float32
        want = R.values(codes, scales, fmt, k).astype(np.float32)
    assert np.array_equal(got[:, :k], want, equal_nan=True) and np.all(got[:, k:] == CANARY)


# ------------------------------------------------------------------ products
PAIRS = [(FP8, FP8), (FP8, FP4), (FP4, FP8), (FP4, FP4)]


def random_mx(rng, fmt, rows, k):
    return R.quantize(loud(rng, rows, k), fmt)


def check_product(keep, device, fa, fb, m, n, k, epilogue, pad=0, in_place=False, seed=0):
    rng = np.random.default_rng(seed + m * 7 + n * 3 + k)
    qa, qb = random_mx(rng, fa, m, k), random_mx(rng, fb, n, k)
    a, b = R.values(*qa, fa, k), R.values(*qb, fb, k)
    alpha, beta = (1.5, -0.5) if epilogue else (1.0, 0.0)
    want, size = alpha * (a @ b.T), abs(alpha) * (np.abs(a) @ np.abs(b).T)
    bias = (rng.normal(size=n) * size.mean()).astype(np.float32)
    c = (rng.normal(size=(m, n + pad)) * size.mean()).astype(np.float32)
    A, B = keep.mx(fa, m, k, qa), keep.mx(fb, n, k, qb)
    cd, bd = (keep.f32(c), keep.f32(bias)) if epilogue else (None, None)
    d = cd if in_place else keep.out(m * (n + pad))
    gemm_mx(device, A, B, d, ldd=n + pad, alpha=alpha, c=cd, ldc=n + pad, beta=beta, bias=bd, act=int(epilogue))
    keep.backend.Device.synchronize(device)
    got = d.download().reshape(m, n + pad)
    if epilogue:
        want = np.maximum(want + beta * c[:, :n] + bias, 0)
        size = size + abs(beta) * np.abs(c[:, :n]) + np.abs(bias)
    assert np.all(np.abs(got[:, :n] - want) <= (k / 32 + 16) * 2.0 ** -23 * size)
    assert np.array_equal(got[:, n:], c[:, n:]) if in_place else np.all(got[:, n:] == CANARY)
    return got


# One row to several tiles of every width, k-loops of one chunk, an odd number of them, and long enough to be divided; last rows and columns alone
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 129, 31), (3, 40, 300), (8, 256, 4096), (9, 700, 129), (16, 128, 512), (17, 2050, 640), (31, 300, 1500), (33, 127, 257),
          (64, 1024, 1024), (65, 513, 383), (100, 200, 300), (128, 640, 2048), (129, 129, 129), (200, 4096, 260), (255, 257, 1023), (300, 500, 700),
          (520, 1000, 130), (700, 2100, 200)]


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(keep, device, fa, fb, m, n, k):
    check_product(keep, device, fa, fb, m, n, k, epilogue=False)


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k,pad,in_place", [(1, 300, 2000, 0, False), (50, 130, 257, 5, False), (129, 260, 100, 3, True), (64, 512, 4096, 0, True),
                                                (300, 520, 384, 4, False), (600, 1030, 70, 0, True)])
def test_product_with_epilogue(keep, device, fa, fb, m, n, k, pad, in_place):
    check_product(keep, device, fa, fb, m, n, k, epilogue=True, pad=pad, in_place=in_place)


@pytest.mark.parametrize("fa,fb", PAIRS)
def test_product_of_drawn_shapes(keep, device, fa, fb):
    """Every number of last rows and columns, beside the widths of tiles."""
    rng = np.random.default_rng(fa * 10 + fb)
    for _ in range(25):
        m, n, k = (int(rng.integers(1, high)) for high in rng.permutation([40, 300, 900]))
        check_product(keep, device, fa, fb, m, n, k, epilogue=bool(rng.integers(2)), pad=int(rng.integers(3)))


@pytest.mark.parametrize("fa,fb", PAIRS)
@pytest.mark.parametrize("m,n,k", [(5, 130, 1000), (64, 300, 4096), (300, 600, 512)])
def test_whole_numbers_are_exact(keep, device, fa, fb, m, n, k):
    """Sums below 2^24 of whole numbers are what they are, in any order."""
    rng = np.random.default_rng(k)
    a, b = rng.integers(-4, 5, (m, k)).astype(float), rng.integers(-4, 5, (n, k)).astype(float)
    a[:, ::32] = 4.0      # every block's scale is 1 in e2m1 and 2^-6 in e4m3: whole numbers up to 4 are values of both types
    b[:, ::32] = -4.0
    A, B, d = keep.mx(fa, m, k, R.quantize(a, fa)), keep.mx(fb, n, k, R.quantize(b, fb)), keep.out(m * n)
    assert np.array_equal(R.values(*A.download(), fa, k), a) and np.array_equal(R.values(*B.download(), fb, k), b)
    gemm_mx(device, A, B, d)
    assert np.array_equal(d.download().reshape(m, n), a @ b.T)


@pytest.mark.parametrize("fa,fb", PAIRS)
def test_scales_of_nan_stay_in_their_row_and_column(keep, device, fa, fb):
    """A NaN in a block makes the row (column) of the result NaN and no other, beside an odd chunk and past the last row too."""
    m, n, k = 130, 140, 384
    rng = np.random.default_rng(3)
    a, b = rng.normal(size=(m, k)), rng.normal(size=(n, k))
    a[129, 5] = np.nan
    a[3, 383] = np.inf
    b[139, 200] = np.nan
    A, B, d = keep.mx(fa, m, k, R.quantize(a, fa)), keep.mx(fb, n, k, R.quantize(b, fb)), keep.out(m * n)
    gemm_mx(device, A, B, d)
    got = np.isnan(d.download().reshape(m, n))
    want = np.zeros((m, n), bool)
    want[[3, 129]] = True
    want[:, 139] = True
    assert np.array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_far_apart(keep, device, fmt):
    """Scales from 2^-100 to 2^100 meet their inverses: the sums are ordinary numbers."""
    m, n, k = 70, 90, 512
    rng = np.random.default_rng(9)
    e = rng.integers(-100, 101, k // 32).repeat(32)
    a, b = np.ldexp(rng.normal(size=(m, k)), e), np.ldexp(rng.normal(size=(n, k)), -e)
    qa, qb = R.quantize(a, fmt), R.quantize(b, fmt)
    A, B, d = keep.mx(fmt, m, k, qa), keep.mx(fmt, n, k, qb), keep.out(m * n)
    gemm_mx(device, A, B, d)
    va, vb = R.values(*qa, fmt, k), R.values(*qb, fmt, k)
    assert np.all(np.abs(d.download().reshape(m, n) - va @ vb.T) <= (k / 32 + 16) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T))


def test_empty_products(keep, device):
    a, b = keep.mx(FP8, 3, 64, R.quantize(np.ones((3, 64)), FP8)), keep.mx(FP8, 5, 64, R.quantize(np.ones((5, 64)), FP8))
    d, c, bias = keep.out(15), keep.f32(np.arange(15, dtype=np.float32)), keep.f32(np.arange(5, dtype=np.float32))
    lib = L.load()
    gemm_mx(device, a, b, d, m=0)
    gemm_mx(device, a, b, d, n=0, ldd=5)
    assert np.all(d.download() == CANARY)
    _check(lib.sb200_gemm_mx(device.id, 0, FP8, FP4, 3, 5, 0, 0, 0, 0, 0, d.ptr, 5, 2.0, c.ptr, 5, 0.5, bias.ptr, 0))     # an empty sum
    assert np.array_equal(d.download().reshape(3, 5), 0.5 * np.arange(15).reshape(3, 5) + np.arange(5))
    for rows, k in ((0, 64), (3, 0)):
        _check(lib.sb200_mx_quantize(device.id, 0, FP8, rows, k, 0, 0, 0, 0, 0))
        _check(lib.sb200_mx_dequantize(device.id, 0, FP8, rows, k, 0, 0, 0, 0))


def test_buffers_of_the_library_are_checked_for_their_extent(backend, device):
    lib = L.load()
    small = backend.Memory.alloc(device, 256, np.float32)
    large = backend.Memory.alloc(device, 1 << 16, np.float32)
    try:
        s, g = small.ptr, large.ptr
        for rc in (lib.sb200_mx_quantize(device.id, 0, FP8, 8, 256, s, 256, 0, g, g + 65536),
                   lib.sb200_mx_quantize(device.id, 0, FP8, 9, 128, g, 128, 0, s, g + 65536),
                   lib.sb200_mx_quantize(device.id, 0, FP8, 8, 256, g, 256, 0, g + 65536, s + 512),
                   lib.sb200_mx_dequantize(device.id, 0, FP8, 8, 256, g, g + 65536, s, 256),
                   lib.sb200_gemm_mx(device.id, 0, FP8, FP8, 8, 64, 256, g, g + 65536, g, s + 32, g + 131072, 64, 1.0, 0, 0, 0.0, 0, 0),
                   lib.sb200_gemm_mx(device.id, 0, FP8, FP8, 8, 64, 256, g, g + 65536, g, g + 65536, s, 64, 1.0, 0, 0, 0.0, 0, 0),
                   lib.sb200_rmsnorm_f32(device.id, 0, 2, 256, s, 256, 0, 0, g, 1e-5, 0, 0, g, 256, 0, 0, 0),
                   lib.sb200_rmsnorm_backward_f32(device.id, 0, 2, 256, g, 256, g, 1e-5, g, 256, 0, 0, 0, 0, g, s, 2048)):
            assert rc == L.ERR_BOUNDS, lib.sb200_last_error_string()
    finally:
        backend.Memory.free(small)
        backend.Memory.free(large)


def test_unknown_device():
    assert L.load().sb200_gemm_mx(99, 0, FP8, FP8, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1.0, 0, 0, 0.0, 0, 0) == L.ERR_INVALID_VALUE


# ------------------------------------------------------------------ norm
# a warp a row, a block a row of each width, rows read twice; whole and broken vectors
COLS = [1, 3, 31, 32, 100, 128, 129, 256, 500, 512, 1000, 1024, 1025, 2048, 3000, 4096, 5001, 8192, 12000, 16384, 20000, 32768, 32769, 40000]


def norm_inputs(rng, rows, cols):
    x, r = loud(rng, rows, cols), loud(rng, rows, cols)
    return x, r, rng.normal(size=cols).astype(np.float32)


def run_norm(keep, device, x, residual, weight, eps, fmt, pad=0, offset=0, in_place=None):
    """sum, y and the two buffers; matrices with `pad` more columns, `offset` floats off alignment.  in_place: which operand sum is."""
    rows, cols = x.shape
    ld = cols + pad

    def padded(v):
        w = np.full((rows, ld), np.nan, np.float32)
        w[:, :cols] = v
        return keep.f32(w, offset=offset)

    xd, rd, wd = padded(x), None if residual is None else padded(residual), keep.f32(weight, offset=offset)
    sd = {"x": xd, "residual": rd, None: None}[in_place] or keep.out(rows * ld, offset=offset)
    yd, q = keep.out(rows * ld, offset=offset), keep.mx(fmt, rows, cols) if fmt else None
    _check(L.load().sb200_rmsnorm_f32(device.id, 0, rows, cols, xd.ptr, ld, rd.ptr if rd else 0, ld if rd else 0, wd.ptr, eps, sd.ptr, ld, yd.ptr, ld, fmt,
                                      q.codes.ptr if q else 0, q.scales.ptr if q else 0))
    s, y = sd.download().reshape(rows, ld), yd.download().reshape(rows, ld)
    assert np.all(y[:, cols:] == CANARY)
    return s[:, :cols], y[:, :cols], q.download() if q else None


@pytest.mark.parametrize("fmt", [0, FP8, FP4])
@pytest.mark.parametrize("cols", COLS)
def test_norm(keep, device, cols, fmt):
    rows = 130 if cols <= 128 else 5
    x, r, w = norm_inputs(np.random.default_rng(cols), rows, cols)
    pad, offset, in_place = [(0, 0, None), (3, 1, "x"), (4, 0, "residual")][cols % 3]
    s, y, q = run_norm(keep, device, x, r, w, 1e-5, fmt, pad, offset, in_place)
    h, want = R.rmsnorm(x, r, w, 1e-5)
    assert np.array_equal(s, h)
    # the root is four units in the last place off at most, the mean, two products and y round once each: 4 + 1/2 + 3 / 2 of 2^-23
    assert np.all(np.abs(y - want) <= 6 * 2.0 ** -23 * np.abs(want))
    if fmt:
        codes, scales = R.quantize(want, fmt)
        assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_codes_of_many_rows_are_the_roundings_of_64_bits(keep, device, fmt):
    """Two million values, some of which lie within float32's error of a border."""
    x, r, w = norm_inputs(np.random.default_rng(17), 1024, 2048)
    _, _, q = run_norm(keep, device, x, r, w, 1e-6, fmt)
    codes, scales = R.quantize(R.rmsnorm(x, r, w, 1e-6)[1], fmt)
    assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_codes_at_the_borders(keep, device, fmt):
    """Rows whose mean square is 1 and weights that put y on the middles between codes, on powers of two and right beside both."""
    g = R.grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    edge = np.r_[mid, 2.0 ** np.arange(-4, 3)].astype(np.float32)
    near = np.r_[edge, np.nextafter(edge, np.float32(0)), np.nextafter(edge, np.float32(1e9)), edge * np.float32(1 + 2.0 ** -20)]
    cols = 512
    w = np.resize(near, cols).astype(np.float32)
    w[::32] = np.float32(2.0 ** R.EMAX[fmt])        # the blocks' scale is 1
    x = np.where(np.arange(cols) % 2 == 0, 1.0, -1.0).astype(np.float32)[None].repeat(3, 0)
    for eps in (0.0, 1e-12, 1e-7, 2.0 ** -24):
        _, _, q = run_norm(keep, device, x, None, w, eps, fmt)
        codes, scales = R.quantize(R.rmsnorm(x, None, w, eps)[1], fmt)
        assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x_scale,w_scale", [(1e-38, 1.0), (1e-30, 1e30), (1e25, 1e-25), (1e30, 1.0), (1.0, 1e-38), (1.0, 1e37), (3e-42, 1.0)])
def test_norm_of_the_smallest_and_the_largest(keep, device, fmt, x_scale, w_scale):
    rng = np.random.default_rng(2)
    x, w = (rng.normal(size=(4, 300)) * x_scale).astype(np.float32), (rng.normal(size=300) * w_scale).astype(np.float32)
    w[:40] *= np.float32(1e-6)
    _, y, q = run_norm(keep, device, x, None, w, 0.0, fmt)
    want = R.rmsnorm(x, None, w, 0.0)[1]
    # as in test_norm, and a rounding to float32's smallest values, which a weight of a normal size keeps small
    assert np.all(np.abs(y - want) <= 6 * 2.0 ** -23 * np.abs(want) + 2.0 ** -148 * np.maximum(1, np.abs(w)))
    codes, scales = R.quantize(want, fmt)
    assert np.array_equal(q[1], scales) and np.array_equal(q[0], codes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_norm_of_zeros_and_of_what_is_not_a_number(keep, device, fmt):
    x = np.zeros((4, 160), np.float32)
    x[1, 7] = np.nan
    x[2, 100] = np.inf
    x[3, :64] = 2.0
    s, y, q = run_norm(keep, device, x, None, np.ones(160, np.float32), 1e-5, fmt)
    values = R.values(*q, fmt, 160)
    assert np.array_equal(s, x, equal_nan=True)
    assert np.all(values[0] == 0) and np.all(y[0] == 0)
    assert np.isnan(values[1]).all() and np.isnan(y[1]).all()      # the mean is NaN
    assert np.isnan(values[2, 96:128]).all() and np.all(values[2, :96] == 0) and np.all(values[2, 128:] == 0)     # inf * 0 beside zeros
    assert np.all(values[3, 64:] == 0) and np.all(values[3, :64] > 0)


def test_norm_results_alone(keep, device):
    """Each result without the others; without a sum nothing but the results is written."""
    rng = np.random.default_rng(4)
    x, r, w = norm_inputs(rng, 9, 260)
    lib = L.load()
    xd, rd, wd = keep.f32(x), keep.f32(r), keep.f32(w)
    _, y, q = run_norm(keep, device, x, r, w, 1e-5, FP8)
    only_y, only_q, only_s = keep.out(9 * 260), keep.mx(FP8, 9, 260), keep.out(9 * 260)
    _check(lib.sb200_rmsnorm_f32(device.id, 0, 9, 260, xd.ptr, 260, rd.ptr, 260, wd.ptr, 1e-5, 0, 0, only_y.ptr, 260, 0, 0, 0))
    _check(lib.sb200_rmsnorm_f32(device.id, 0, 9, 260, xd.ptr, 260, rd.ptr, 260, wd.ptr, 1e-5, 0, 0, 0, 0, FP8, only_q.codes.ptr, only_q.scales.ptr))
    _check(lib.sb200_rmsnorm_f32(device.id, 0, 9, 260, xd.ptr, 260, rd.ptr, 260, wd.ptr, 1e-5, only_s.ptr, 260, 0, 0, 0, 0, 0))
    assert np.array_equal(only_y.download(), y.ravel()) and np.array_equal(only_s.download().reshape(9, 260), x + r)
    assert all(np.array_equal(u, v) for u, v in zip(only_q.download(), q))
    assert np.array_equal(xd.download(), x.ravel()) and np.array_equal(rd.download(), r.ravel())


# ------------------------------------------------------------------ its gradient
def run_backward(keep, device, h, w, dy, dsum, eps, pad=0, offset=0, in_place=None, want=("dx", "dweight")):
    rows, cols = h.shape
    ld = cols + pad

    def padded(v):
        full = np.full((rows, ld), np.nan, np.float32)
        full[:, :cols] = v
        return keep.f32(full, offset=offset)

    hd, dyd, wd = padded(h), padded(dy), keep.f32(w, offset=offset)
    dsd = None if dsum is None else padded(dsum)
    dx = {"sum": hd, "dy": dyd, "dsum": dsd, None: None}[in_place] or keep.out(rows * ld, offset=offset)
    need = C.c_uint64()
    _check(L.load().sb200_rmsnorm_workspace_bytes(rows, cols, C.byref(need)))
    dw, ws = keep.out(cols, offset=offset), keep.bytes(need.value)
    _check(L.load().sb200_rmsnorm_backward_f32(device.id, 0, rows, cols, hd.ptr, ld, wd.ptr, eps, dyd.ptr, ld, dsd.ptr if dsd else 0, ld if dsd else 0,
                                               dx.ptr if "dx" in want else 0, ld, dw.ptr if "dweight" in want else 0, ws.ptr, need.value))
    keep.backend.Device.synchronize(device)
    got, gw = dx.download().reshape(rows, ld), dw.download()
    ws.download()
    return got[:, :cols], gw


def check_backward(got, h, w, dy, dsum, eps):
    """The two sums are trees of float32 additions over at most 32 terms a thread, 32 lanes and 32 warps: 48 roundings of 2^-24 of the sums of
    magnitudes; the other operations round a dozen times.  dweight: one after the other over the rows of a block, then over the parts."""
    dx, dw = R.rmsnorm_backward(h, w, dy, dsum, eps)
    h, w, dy = (v.astype(np.float64) for v in (h, w, dy))
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, g = np.abs(h * r), np.abs(dy * w)
    size = r * (g + n * (g * n).mean(-1, keepdims=True)) + (0 if dsum is None else np.abs(dsum))
    assert np.all(np.abs(got[0] - dx) <= 64 * 2.0 ** -24 * size)
    assert np.all(np.abs(got[1] - dw) <= (min(h.shape[0], 600) + 64) * 2.0 ** -24 * (np.abs(dy) * n).sum(0))


@pytest.mark.parametrize("cols", COLS)
def test_norm_backward(keep, device, cols):
    rng = np.random.default_rng(cols + 1)
    rows = 700 if cols <= 512 else 9
    h, w = loud(rng, rows, cols), rng.normal(size=cols).astype(np.float32)
    dy, ds = loud(rng, rows, cols), loud(rng, rows, cols) if cols % 2 else None
    pad, offset, in_place = [(0, 0, None), (3, 1, "dy"), (4, 0, "sum")][cols % 3]
    check_backward(run_backward(keep, device, h, w, dy, ds, 1e-5, pad, offset, in_place), h, w, dy, ds, 1e-5)


@pytest.mark.parametrize("rows", [1, 2, 147, 148, 296, 297, 444, 445, 600, 1500])
@pytest.mark.parametrize("cols", [36, 260, 1000])
def test_norm_backward_rows(keep, device, rows, cols):
    """From one row to several for every block, with the gradient of the sum and in its place."""
    rng = np.random.default_rng(rows)
    h, w = rng.normal(size=(rows, cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    dy, ds = rng.normal(size=(rows, cols)).astype(np.float32), rng.normal(size=(rows, cols)).astype(np.float32)
    check_backward(run_backward(keep, device, h, w, dy, ds, 1e-5, in_place="dsum" if rows % 2 else None), h, w, dy, ds, 1e-5)


@pytest.mark.parametrize("rows,cols", [(1, 8193), (300, 8196), (150, 12001), (75, 16384), (2, 16385), (180, 20004), (101, 24577), (77, 40000), (43, 49155),
                                       (31, 65535), (60, 65536), (3, 65537)])
def test_norm_backward_wide(keep, device, rows, cols):
    """Rows of two to eight blocks, up to five for a cluster, and those that no cluster takes."""
    rng = np.random.default_rng(cols)
    h, w = loud(rng, rows, cols), rng.normal(size=cols).astype(np.float32)
    dy, ds = loud(rng, rows, cols), loud(rng, rows, cols) if rows % 2 else None
    check_backward(run_backward(keep, device, h, w, dy, ds, 1e-5, 3 if rows % 5 == 0 else 0, 0, "dy" if rows % 3 == 0 else None), h, w, dy, ds, 1e-5)


def test_norm_backward_against_differences(keep, device):
    """The loss sum(c * y) changes by dx and dweight, to a difference's error: central differences of the formula in 64 bits."""
    rng = np.random.default_rng(8)
    x, r, w, c = (rng.normal(size=s).astype(np.float32) for s in ((3, 50), (3, 50), 50, (3, 50)))
    dx, dw = run_backward(keep, device, x + r, w, c, None, 1e-3)
    h = (x + r).astype(np.float64)

    def loss(h, w):
        return (c * (h * w / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-3))).sum()

    step = 1e-5
    for at in [(0, 0), (1, 20), (2, 49)]:
        e = np.zeros_like(h)
        e[at] = step
        # the third derivative is of order 1: step^2, and 2^-53 / step of the loss's terms
        assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * step) - dx[at]) <= 1e-5
    for at in (0, 31, 49):
        e = np.zeros(50)
        e[at] = step
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * step) - dw[at]) <= 1e-5


def test_norm_backward_results_alone(keep, device):
    rng = np.random.default_rng(5)
    for cols in (300, 302, 9000):
        h, w, dy = (rng.normal(size=s).astype(np.float32) for s in ((20, cols), cols, (20, cols)))
        dx, dw = run_backward(keep, device, h, w, dy, None, 1e-5)
        alone, untouched = run_backward(keep, device, h, w, dy, None, 1e-5, want=("dx",))
        assert np.array_equal(alone, dx) and np.all(untouched == CANARY)
        untouched, alone = run_backward(keep, device, h, w, dy, None, 1e-5, want=("dweight",))
        assert np.array_equal(alone, dw) and np.all(untouched == CANARY)


def test_norm_backward_of_no_rows(keep, device):
    dw = keep.out(33)
    _check(L.load().sb200_rmsnorm_backward_f32(device.id, 0, 0, 33, 0, 0, 0, 1e-5, 0, 0, 0, 0, 0, 0, dw.ptr, 0, 0))
    assert np.all(dw.download() == 0)


# ------------------------------------------------------------------ together
class Layer:
    """Norm to `fa`, product with `fb` weights, bias and clamp, and the gradients of its linear part, on one stream."""

    def __init__(self, keep, device, m, n, k, fa, fb, seed=0):
        rng = np.random.default_rng(seed)
        self.keep, self.device, self.m, self.n, self.k, self.fa, self.fb = keep, device, m, n, k, fa, fb
        self.gain, self.w = rng.normal(size=k).astype(np.float32), (rng.normal(size=(k, n)) / np.sqrt(k)).astype(np.float32)
        self.bias = rng.normal(size=n).astype(np.float32)
        self.dev = {name: keep.f32(getattr(self, name)) for name in ("gain", "w", "bias")}
        self.x, self.res, self.dd = keep.out(m * k), keep.out(m * k), keep.out(m * n)
        self.s, self.d, self.dx, self.dw = keep.out(m * k), keep.out(m * n), keep.out(m * k), keep.out(k * n)
        self.q, self.qw = keep.mx(fa, m, k), keep.mx(fb, n, k)
        self.dd_rows, self.w_rows, self.dd_cols, self.s_cols = keep.mx(FP8, m, n), keep.mx(FP8, k, n), keep.mx(FP8, n, m), keep.mx(FP8, k, m)

    def upload(self, seed):
        rng = np.random.default_rng(seed)
        x, res, dd = loud(rng, self.m, self.k), loud(rng, self.m, self.k), loud(rng, self.m, self.n)
        for dev, a in ((self.x, x), (self.res, res), (self.dd, dd)):
            dev.upload(a)
        return x, res, dd

    def calls(self, stream):
        lib, dev, m, n, k = L.load(), self.device.id, self.m, self.n, self.k

        def quantize(src, ld, transposed, to):
            _check(lib.sb200_mx_quantize(dev, stream, to.fmt, to.rows, to.k, src.ptr, ld, transposed, to.codes.ptr, to.scales.ptr))

        quantize(self.dev["w"], n, 1, self.qw)
        _check(lib.sb200_rmsnorm_f32(dev, stream, m, k, self.x.ptr, k, self.res.ptr, k, self.dev["gain"].ptr, 1e-5, self.s.ptr, k, 0, 0, self.fa,
                                     self.q.codes.ptr, self.q.scales.ptr))
        gemm_mx(self.device, self.q, self.qw, self.d, bias=self.dev["bias"], act=1, stream=stream)
        quantize(self.dd, n, 0, self.dd_rows)
        quantize(self.dev["w"], n, 0, self.w_rows)
        quantize(self.dd, n, 1, self.dd_cols)
        quantize(self.s, k, 1, self.s_cols)
        gemm_mx(self.device, self.dd_rows, self.w_rows, self.dx, stream=stream)
        gemm_mx(self.device, self.s_cols, self.dd_cols, self.dw, stream=stream)

    def check(self, inputs):
        x, res, dd = inputs
        h, y = R.rmsnorm(x, res, self.gain, 1e-5)

        def both(u, v, fu, fv):
            return (R.values(*R.quantize(p, f), f, p.shape[1]) for p, f in ((u, fu), (v, fv)))

        for got, (u, v), extra in ((self.d, both(y, self.w.T, self.fa, self.fb), self.bias), (self.dx, both(dd, self.w, FP8, FP8), None),
                                   (self.dw, both(h.T, dd.T, FP8, FP8), None)):
            want, size = u @ v.T, np.abs(u) @ np.abs(v).T
            if extra is not None:
                want, size = np.maximum(want + extra, 0), size + np.abs(extra)
            assert np.all(np.abs(got.download().reshape(want.shape) - want) <= (u.shape[1] / 32 + 16) * 2.0 ** -23 * size)


@pytest.mark.parametrize("m,n,k,fa,fb", [(1, 300, 256, FP8, FP4), (70, 260, 500, FP4, FP4), (200, 384, 640, FP8, FP8)])
def test_a_layer_and_its_gradients(keep, device, m, n, k, fa, fb):
    layer = Layer(keep, device, m, n, k, fa, fb)
    for seed in (1, 2):
        inputs = layer.upload(seed)
        layer.calls(0)
        layer.check(inputs)


def test_two_streams_side_by_side(keep, backend, device):
    layers = [Layer(keep, device, 90, 300, 400, FP8, FP4, seed) for seed in (0, 1)]
    streams = [backend.Stream.create(device) for _ in layers]
    inputs = [layer.upload(5 + i) for i, layer in enumerate(layers)]
    for _ in range(3):
        for layer, stream in zip(layers, streams):
            layer.calls(stream.handle)
    for stream in streams:
        backend.Stream.synchronize(stream)
        backend.Stream.destroy(stream)
    for layer, i in zip(layers, inputs):
        layer.check(i)


def test_captured_and_replayed(keep, backend, device):
    """Two graphs of different layers, replayed side by side on new inputs, and calls outside of them in between."""
    torch = pytest.importorskip("torch")
    layers = [Layer(keep, device, 33, 260, 390, FP8, FP4, 3), Layer(keep, device, 150, 130, 256, FP4, FP8, 4)]
    graphs, streams = [], [torch.cuda.Stream() for _ in layers]
    for layer, stream in zip(layers, streams):
        layer.upload(0)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            layer.calls(stream.cuda_stream)
    other = Layer(keep, device, 64, 200, 256, FP8, FP8, 9)
    for seed in (20, 30):
        inputs = [layer.upload(seed + i) for i, layer in enumerate(layers)]
        mine = other.upload(seed)
        torch.cuda.synchronize()
        for _ in range(2):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        other.calls(0)
        torch.cuda.synchronize()
        for layer, i in zip(layers, inputs):
            layer.check(i)
        other.check(mine)
    del graphs


def test_backward_captured_and_replayed(keep, device):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(6)
    rows, cols = 500, 1000
    h, w, dy = (rng.normal(size=s).astype(np.float32) for s in ((rows, cols), cols, (rows, cols)))
    hd, wd, dyd, dx, dw, ws = keep.f32(h), keep.f32(w), keep.f32(dy), keep.out(rows * cols), keep.out(cols), keep.bytes(rows * cols * 4)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()

    def call(st):
        _check(L.load().sb200_rmsnorm_backward_f32(device.id, st, rows, cols, hd.ptr, cols, wd.ptr, 1e-5, dyd.ptr, cols, 0, 0, dx.ptr, cols, dw.ptr, ws.ptr,
                                                   rows * cols * 4))

    with torch.cuda.graph(graph, stream=stream):
        call(stream.cuda_stream)
    for seed in (1, 2):
        dy = np.random.default_rng(seed).normal(size=(rows, cols)).astype(np.float32)
        dyd.upload(dy)
        graph.replay()
        torch.cuda.synchronize()
        check_backward((dx.download().reshape(rows, cols), dw.download()), h, w, dy, None, 1e-5)
    del graph


def test_the_same_bits_every_time(keep, backend, device):
    """Divided k-loops, sums over rows and all else in a fixed order."""
    rng = np.random.default_rng(12)
    for m, n, k in ((4, 500, 8192), (64, 300, 4096), (300, 700, 300)):
        a, b = keep.mx(FP8, m, k, random_mx(rng, FP8, m, k)), keep.mx(FP4, n, k, random_mx(rng, FP4, n, k))
        d = keep.out(m * n)
        seen = set()
        for _ in range(20):
            gemm_mx(device, a, b, d)
            seen.add(d.download().tobytes())
        assert len(seen) == 1
    h, w, dy = (rng.normal(size=s).astype(np.float32) for s in ((900, 640), 640, (900, 640)))
    assert len({b"".join(v.tobytes() for v in run_backward(keep, device, h, w, dy, None, 1e-5)) for _ in range(5)}) == 1


def test_rows_and_columns_that_are_not_there_stay_as_they_are(keep, device):
    """A last tile of one row and one column: D's neighbours keep their values."""
    for m, n in ((257, 129), (129, 257), (1, 1)):
        check_product(keep, device, FP8, FP8, m, n, 128, epilogue=True, pad=7, in_place=True)


def test_errors_carry_the_message(keep, device):
    with pytest.raises(BackendError, match="leading dimension"):
        gemm_mx(device, keep.mx(FP8, 4, 32), keep.mx(FP8, 9, 32), keep.out(36), ldd=8)


# ------------------------------------------------------------------ far and wide
def test_offsets_past_32_bits(keep, backend, device):
    """Five rows 2^30 + 4 floats apart, the last of which lie beyond 2^32 elements: read, summed, written."""
    rows, cols, ld = 5, 132, (1 << 30) + 4
    lib = L.load()
    rng = np.random.default_rng(0)
    x, w = rng.normal(size=(rows, cols)).astype(np.float32), rng.normal(size=cols).astype(np.float32)
    far = backend.Memory.alloc(device, (rows - 1) * ld + cols, np.float32)

    def put(a):
        for i in range(rows):
            row = np.ascontiguousarray(a[i])
            _check(lib.sb200_memcpy_htod(device.id, far.ptr + 4 * i * ld, row.ctypes.data_as(C.c_void_p), 4 * cols))

    def get():
        out = np.empty((rows, cols), np.float32)
        for i in range(rows):
            _check(lib.sb200_memcpy_dtoh(device.id, out[i].ctypes.data_as(C.c_void_p), far.ptr + 4 * i * ld, 4 * cols))
        return out

    try:
        q, wd, dw, ws = keep.mx(FP8, rows, cols), keep.f32(w), keep.out(cols), keep.bytes(rows * cols * 4)
        codes, scales = R.quantize(x, FP8)
        put(x)
        _check(lib.sb200_mx_quantize(device.id, 0, FP8, rows, cols, far.ptr, ld, 0, q.codes.ptr, q.scales.ptr))
        assert np.array_equal(q.download()[0], codes) and np.array_equal(q.download()[1], scales)
        put(np.zeros_like(x))
        _check(lib.sb200_mx_dequantize(device.id, 0, FP8, rows, cols, q.codes.ptr, q.scales.ptr, far.ptr, ld))
        assert np.array_equal(get(), R.values(codes, scales, FP8, cols).astype(np.float32))
        turned = keep.mx(FP4, cols, rows)
        put(x)
        _check(lib.sb200_mx_quantize(device.id, 0, FP4, cols, rows, far.ptr, ld, 1, turned.codes.ptr, turned.scales.ptr))
        assert np.array_equal(turned.download()[0], R.quantize(x.T, FP4)[0])
        _check(lib.sb200_rmsnorm_f32(device.id, 0, rows, cols, far.ptr, ld, far.ptr, ld, wd.ptr, 1e-5, far.ptr, ld, 0, 0, FP8, q.codes.ptr, q.scales.ptr))
        h, y = R.rmsnorm(x, x, w, 1e-5)
        assert np.array_equal(get(), h) and np.array_equal(q.download()[0], R.quantize(y, FP8)[0])
        _check(lib.sb200_rmsnorm_backward_f32(device.id, 0, rows, cols, far.ptr, ld, wd.ptr, 1e-5, far.ptr, ld, far.ptr, ld, far.ptr, ld, dw.ptr, ws.ptr,
                                              rows * cols * 4))
        backend.Device.synchronize(device)
        check_backward((get(), dw.download()), h, w, h, h, 1e-5)
        a, b = random_mx(rng, FP8, rows, 200), random_mx(rng, FP4, cols, 200)
        A, B = keep.mx(FP8, rows, 200, a), keep.mx(FP4, cols, 200, b)
        put(x)
        _check(lib.sb200_gemm_mx(device.id, 0, FP8, FP4, rows, cols, 200, A.codes.ptr, A.scales.ptr, B.codes.ptr, B.scales.ptr, far.ptr, ld, 1.0, far.ptr, ld,
                                 1.0, 0, 0))
        backend.Device.synchronize(device)
        va, vb = R.values(*a, FP8, 200), R.values(*b, FP4, 200)
        assert np.all(np.abs(get() - (va @ vb.T + x)) <= (200 / 32 + 16) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T + np.abs(x)))
    finally:
        backend.Memory.free(far)


@pytest.mark.parametrize("m,n,k", [(70001, 5, 40), (3, 150001, 64), (1, 1, 70000), (130, 2, 40000), (2, 131, 33000)])
def test_product_of_the_longest(keep, device, m, n, k):
    check_product(keep, device, FP8, FP4, m, n, k, epilogue=True)


@pytest.mark.parametrize("rows,cols", [(100003, 3), (1, 300001), (2, 262144), (65537, 36)])
def test_norm_of_the_longest(keep, device, rows, cols):
    rng = np.random.default_rng(cols)
    x, r, w = norm_inputs(rng, rows, cols)
    s, y, q = run_norm(keep, device, x, r, w, 1e-5, FP8)
    h, want = R.rmsnorm(x, r, w, 1e-5)
    codes, scales = R.quantize(want, FP8)
    assert np.array_equal(s, h) and np.array_equal(q[0], codes) and np.array_equal(q[1], scales)
    dy = rng.normal(size=(rows, cols)).astype(np.float32)
    check_backward(run_backward(keep, device, h, w, dy, x, 1e-5), h, w, dy, x, 1e-5)


@pytest.mark.parametrize("rows,k", [(100003, 1), (1, 300001), (3, 131072)])
@pytest.mark.parametrize("transposed", [0, 1])
def test_quantize_the_longest(keep, device, rows, k, transposed):
    v = np.random.default_rng(k).normal(size=(rows, k)).astype(np.float32)
    x, q = keep.f32(v.T if transposed else v), keep.mx(FP4, rows, k)
    _check(L.load().sb200_mx_quantize(device.id, 0, FP4, rows, k, x.ptr, rows if transposed else k, transposed, q.codes.ptr, q.scales.ptr))
    codes, scales = R.quantize(v, FP4)
    assert np.array_equal(q.download()[0], codes) and np.array_equal(q.download()[1], scales)
