"""Products of microscaled matrices in every form that sizes take (pairs of blocks, several tiles a block, rings that turn, accumulators that overlap), with whole
numbers: sums below 2^24 are what they are in any order, so that a wrong scale, row or wait shows in every bit.  tests/test_mx_plan.py shows that
these sizes and those of tests/test_gpu_mx.py take them all."""
import numpy as np
import pytest

from tests import mx_ref as R
from tests.mx_ref import FP4, FP8, gemm_mx
from tests.test_gpu_mx import PAIRS, keep  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

FORMS = [
    # a k-loop divided within a cluster: 16, 32, 64 and 128 rows a tile; and one longer than the ring that is not
    (17, 300, 2346), (18, 17, 3753), (36, 129, 2367), (33, 150, 4970), (70, 17, 3662), (67, 260, 6869), (1, 2702, 1413), (1, 300, 2600),
    # several tiles a block
    (5, 40001, 200), (30, 40003, 130), (60, 40005, 389), (129, 9916, 49), (288, 9500, 889), (514, 13001, 1400),
    # pairs, a tile of 128 rows each, or several
    (158, 9399, 3101), (131, 9369, 6799), (263, 9774, 2203), (261, 9740, 3850), (513, 9601, 1700),
    # pairs, a tile of 256 rows each, or several
    (137, 9751, 136), (130, 9553, 874), (261, 6274, 300), (129, 10122, 1731), (389, 14849, 853), (412, 14587, 1686), (518, 11308, 300), (1195, 13001, 300),
]
WHOLE = np.array([0, 1, 2, 3, 4, 6])
CODES = {FP8: np.array([0x00, 0x38, 0x40, 0x44, 0x48, 0x4C], np.uint8), FP4: np.array([0, 2, 4, 5, 6, 7], np.uint8)}


def operand(rng, rows, k):
    """Whole numbers, as values and as the buffers of either format: values up to 6, scales 1, 2 and 4."""
    kp = -(-k // 128) * 128
    at, minus = np.zeros((rows, kp), np.uint8), np.zeros((rows, kp), bool)
    at[:, :k], minus[:, :k] = rng.integers(0, WHOLE.size, (rows, k), dtype=np.uint8), rng.integers(0, 2, (rows, k), dtype=np.uint8)
    power = rng.integers(0, 3, (rows, kp // 32), dtype=np.uint8)
    power[:, -(-k // 32):] = 0
    v = np.where(minus, -1.0, 1.0) * WHOLE[at] * np.repeat(2.0 ** power, 32, axis=1)
    scales = np.zeros(-(-rows // 128) * 128 * kp // 32, np.uint8)
    scales[R.tile_offsets(rows, kp // 32)[:, :-(-k // 32)]] = 127 + power[:, :-(-k // 32)]
    c8, c4 = CODES[FP8][at] | minus.astype(np.uint8) << 7, CODES[FP4][at] | minus.astype(np.uint8) << 3
    return v[:, :k], {FP8: (c8, scales), FP4: (c4[:, 0::2] | c4[:, 1::2] << 4, scales)}


@pytest.mark.parametrize("m,n,k", FORMS)
def test_every_form_is_exact(keep, device, m, n, k):  # noqa: F811
    rng = np.random.default_rng(m + n + k)
    (a, qa), (b, qb) = operand(rng, m, k), operand(rng, n, k)
    assert 24 * 24 * k < 2 ** 23        # no sum of magnitudes, nor the same doubled, leaves 24 bits
    product = a @ b.T
    c, bias = rng.integers(-999, 1000, (m, n)).astype(np.float32), rng.integers(-999, 1000, n).astype(np.float32)
    with_epilogue = np.maximum(0.5 * product - 2 * c + bias, 0)
    A, B = {f: keep.mx(f, m, k, qa[f]) for f in qa}, {f: keep.mx(f, n, k, qb[f]) for f in qb}
    d, dc, bd = keep.out(m * n), keep.f32(c), keep.f32(bias)
    for fa, fb in PAIRS:
        d.upload(np.full(m * n, np.nan, np.float32))
        gemm_mx(device, A[fa], B[fb], d)
        keep.backend.Device.synchronize(device)
        assert np.array_equal(d.download().reshape(m, n), product), (fa, fb)
        dc.upload(c)
        gemm_mx(device, A[fa], B[fb], dc, alpha=0.5, c=dc, beta=-2.0, bias=bd, act=1)     # in place
        keep.backend.Device.synchronize(device)
        assert np.array_equal(dc.download().reshape(m, n), with_epilogue), (fa, fb)


@pytest.mark.parametrize("m,n,k", [(389, 14849, 853), (263, 9774, 2203), (1195, 13001, 300)])
def test_pairs_give_the_same_bits_every_time(keep, device, m, n, k):  # noqa: F811
    rng = np.random.default_rng(k)
    v = [rng.normal(size=(rows, k)).astype(np.float32) for rows in (m, n)]
    for fmt in (FP8, FP4):
        q = [keep.mx(fmt, x.shape[0], k) for x in v]
        for x, to in zip(v, q):
            src = keep.f32(x)
            assert R.L.load().sb200_mx_quantize(device.id, 0, fmt, to.rows, k, src.ptr, k, 0, to.codes.ptr, to.scales.ptr) == 0
        d = keep.out(m * n)
        seen = set()
        for _ in range(4):
            gemm_mx(device, q[0], q[1], d)
            keep.backend.Device.synchronize(device)
            seen.add(hash(d.download().tobytes()))
        assert len(seen) == 1
