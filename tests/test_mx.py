"""Microscaled operators and the norm without a GPU: sizes, refusals, and the reference that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from spoc_b200 import _lib as L
from spoc_b200.build import build_library
from tests import mx_ref as R

GOOD = 1 << 20      # an address that is aligned; nothing is read in a call that is refused
TOO_MANY = 1 << 31


@pytest.fixture(scope="module")
def lib():
    build_library()
    return L.load()


@pytest.mark.parametrize("fmt,rows,k,codes,scales", [(L.MX_FP8, 1, 1, 128, 512), (L.MX_FP4, 1, 1, 64, 512), (L.MX_FP8, 129, 128, 129 * 128, 1024),
                                                     (L.MX_FP4, 300, 4096, 300 * 2048, 3 * 32 * 512), (L.MX_FP8, 0, 7, 0, 0), (L.MX_FP8, 5, 0, 0, 0),
                                                     (L.MX_FP4, 1 << 20, 1 << 14, 1 << 33, 1 << 29)])
def test_sizes(lib, fmt, rows, k, codes, scales):
    assert R.mx_bytes(fmt, rows, k) == (codes, scales)


@pytest.mark.parametrize("rows,cols,need", [(0, 5, 0), (1, 5, 20), (511, 64, 511 * 256), (512, 64, 512 * 256), (100000, 64, 512 * 256)])
def test_workspace_sizes(lib, rows, cols, need):
    n = C.c_uint64()
    assert lib.sb200_rmsnorm_workspace_bytes(rows, cols, C.byref(n)) == 0 and n.value == need


QUANTIZE = dict(format=L.MX_FP8, rows=4, k=256, src=GOOD, ld=256, transposed=0, codes=GOOD, scales=GOOD)
DEQUANTIZE = dict(format=L.MX_FP4, rows=4, k=256, codes=GOOD, scales=GOOD, dst=GOOD, ld=256)
GEMM = dict(format_a=L.MX_FP8, format_b=L.MX_FP4, m=4, n=8, k=256, a_codes=GOOD, a_scales=GOOD, b_codes=GOOD, b_scales=GOOD, d=GOOD, ldd=8,
            alpha=1.0, c=GOOD, ldc=8, beta=1.0, bias=GOOD, act=0)
NORM = dict(rows=4, cols=256, x=GOOD, ldx=256, residual=GOOD, ldr=256, weight=GOOD, eps=1e-5, sum=GOOD, lds=256, y=GOOD, ldy=256,
            format=L.MX_FP8, codes=GOOD, scales=GOOD)
BACKWARD = dict(rows=4, cols=256, sum=GOOD, lds=256, weight=GOOD, eps=1e-5, dy=GOOD, lddy=256, dsum=GOOD, ldds=256, dx=GOOD, lddx=256,
                dweight=GOOD, workspace=GOOD, workspace_bytes=4096)
VALUE, ALIGN, LARGE = L.ERR_INVALID_VALUE, L.ERR_ALIGNMENT, L.ERR_TOO_LARGE

REFUSED = (
    [("mx_quantize", QUANTIZE, c, e) for c, e in [
        (dict(format=0), VALUE), (dict(format=6), VALUE), (dict(rows=-1), VALUE), (dict(k=-1), VALUE), (dict(rows=TOO_MANY), LARGE),
        (dict(k=TOO_MANY), LARGE), (dict(rows=1 << 30, k=1 << 20), LARGE), (dict(src=0), VALUE), (dict(src=GOOD + 2), ALIGN), (dict(ld=255), VALUE),
        (dict(transposed=1, ld=3), VALUE), (dict(codes=0), VALUE), (dict(scales=0), VALUE), (dict(codes=GOOD + 16), ALIGN),
        (dict(scales=GOOD + 8), ALIGN), (dict(ld=1 << 62), LARGE)]] +
    [("mx_dequantize", DEQUANTIZE, c, e) for c, e in [
        (dict(format=1), VALUE), (dict(rows=-2), VALUE), (dict(codes=0), VALUE), (dict(scales=GOOD + 4), ALIGN), (dict(dst=0), VALUE),
        (dict(dst=GOOD + 1), ALIGN), (dict(ld=255), VALUE)]] +
    [("gemm_mx", GEMM, c, e) for c, e in [
        (dict(format_a=5), VALUE), (dict(format_b=-4), VALUE), (dict(m=-1), VALUE), (dict(n=-1), VALUE), (dict(k=-1), VALUE), (dict(m=TOO_MANY), LARGE),
        (dict(n=TOO_MANY), LARGE), (dict(k=TOO_MANY), LARGE), (dict(a_codes=0), VALUE), (dict(b_scales=0), VALUE), (dict(a_scales=GOOD + 16), ALIGN),
        (dict(b_codes=GOOD + 16), ALIGN), (dict(d=0), VALUE), (dict(d=GOOD + 2), ALIGN), (dict(ldd=7), VALUE), (dict(ldc=7), VALUE),
        (dict(c=GOOD + 3), ALIGN), (dict(bias=GOOD + 1), ALIGN), (dict(act=2), VALUE)]] +
    [("rmsnorm_f32", NORM, c, e) for c, e in [
        (dict(format=3), VALUE), (dict(rows=-1), VALUE), (dict(cols=TOO_MANY), LARGE), (dict(x=0), VALUE), (dict(x=GOOD + 2), ALIGN),
        (dict(ldx=255), VALUE), (dict(ldr=255), VALUE), (dict(residual=GOOD + 1), ALIGN), (dict(weight=0), VALUE), (dict(weight=GOOD + 3), ALIGN),
        (dict(eps=-1e-9), VALUE), (dict(eps=float("nan")), VALUE), (dict(lds=255), VALUE), (dict(ldy=100), VALUE), (dict(y=GOOD + 2), ALIGN),
        (dict(codes=0), VALUE), (dict(scales=GOOD + 16), ALIGN), (dict(sum=0, y=0, format=0), VALUE)]] +
    [("rmsnorm_backward_f32", BACKWARD, c, e) for c, e in [
        (dict(rows=-1), VALUE), (dict(cols=-1), VALUE), (dict(sum=0), VALUE), (dict(weight=0), VALUE), (dict(dy=0), VALUE), (dict(dy=GOOD + 2), ALIGN),
        (dict(lds=1), VALUE), (dict(lddy=255), VALUE), (dict(ldds=255), VALUE), (dict(lddx=255), VALUE), (dict(dx=0, dweight=0), VALUE),
        (dict(workspace=0), VALUE), (dict(workspace_bytes=4095), VALUE), (dict(workspace=GOOD + 2), ALIGN), (dict(dweight=GOOD + 1), ALIGN),
        (dict(eps=-1.0), VALUE)]])


@pytest.mark.parametrize("name,good,change,error", REFUSED, ids=lambda v: str(v) if isinstance(v, (str, int)) else None)
def test_refusals(lib, name, good, change, error):
    """Every refusal is the host's: it comes before a device is asked for."""
    assert getattr(lib, "sb200_" + name)(0, 0, *{**good, **change}.values()) == error
    assert lib.sb200_last_error_string()


APART = dict(sum=GOOD + 4096, y=GOOD + 8192)
IN_PLACE = [("rmsnorm_f32", NORM, {}), ("rmsnorm_f32", NORM, dict(APART, sum=GOOD, lds=260)), ("rmsnorm_f32", NORM, dict(APART, y=GOOD, ldr=257)),
            ("rmsnorm_f32", NORM, dict(APART, y=GOOD, residual=0, ldy=300)), ("gemm_mx", GEMM, dict(ldd=9)), ("gemm_mx", GEMM, dict(ldc=12)),
            ("rmsnorm_backward_f32", BACKWARD, dict(lddx=257)), ("rmsnorm_backward_f32", BACKWARD, dict(lddy=260)),
            ("rmsnorm_backward_f32", BACKWARD, dict(ldds=260)), ("rmsnorm_backward_f32", BACKWARD, dict(lds=260))]


@pytest.mark.parametrize("name,good,change", IN_PLACE)
def test_refusals_in_place(lib, name, good, change):
    """A result that lies on an operand with other row lengths, and two results on each other."""
    assert getattr(lib, "sb200_" + name)(0, 0, *{**good, **change}.values()) == VALUE
    assert b"in place" in lib.sb200_last_error_string() or b"same matrix" in lib.sb200_last_error_string()


def test_refusals_of_sizes(lib):
    a, b = C.c_uint64(), C.c_uint64()
    assert lib.sb200_mx_bytes(7, 1, 1, C.byref(a), C.byref(b)) == VALUE
    assert lib.sb200_mx_bytes(L.MX_FP8, -1, 1, C.byref(a), C.byref(b)) == VALUE
    assert lib.sb200_mx_bytes(L.MX_FP8, 1, 1, None, C.byref(b)) == VALUE
    assert lib.sb200_rmsnorm_workspace_bytes(1, 1, None) == VALUE
    assert lib.sb200_rmsnorm_workspace_bytes(-1, 1, C.byref(a)) == VALUE


@pytest.mark.parametrize("fmt", R.FORMATS)
def test_reference_rounds_to_the_nearest(fmt):
    """Every value of the type is its own code; what lies between two goes to the nearer, the middle to the even one."""
    g = R.grid(fmt)
    assert np.array_equal(R.round_to(g, fmt), np.arange(g.size)) and np.array_equal(R.round_to(-g, fmt) % (8 if fmt == R.FP4 else 128), np.arange(g.size))
    mid = (g[1:] + g[:-1]) / 2
    even = np.arange(g.size - 1) + np.arange(g.size - 1) % 2
    assert np.array_equal(R.round_to(mid, fmt), even)
    assert np.array_equal(R.round_to(np.nextafter(mid, 0), fmt), np.arange(g.size - 1))
    assert np.array_equal(R.round_to(np.nextafter(mid, 1e9), fmt), np.arange(1, g.size))
    assert R.round_to(np.array([1e30]), fmt) == g.size - 1


@pytest.mark.parametrize("fmt", R.FORMATS)
def test_reference_is_within_half_a_step(fmt):
    """A value of the type is off by half a step of its block's largest binade at most, or held at the largest value."""
    rng = np.random.default_rng(1)
    v = rng.normal(size=(37, 200)) * np.exp(rng.normal(size=(37, 1)) * 10)
    got = R.values(*R.quantize(v, fmt), fmt, 200)
    top = np.abs(np.pad(v, ((0, 0), (0, 24))).reshape(37, 7, 32)).max(-1).repeat(32, 1)[:, :200]
    half_step = 2.0 ** (np.floor(np.log2(top)) - (3 if fmt == R.FP8 else 1) - 1)
    held = np.abs(v) > np.abs(got)
    largest = R.grid(fmt)[-1] * 2.0 ** (np.floor(np.log2(top)) - R.EMAX[fmt])
    assert np.all((np.abs(v - got) <= half_step) | (held & (np.abs(got) == largest)))
