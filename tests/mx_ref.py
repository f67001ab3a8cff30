"""Microscaled matrices, their products and the root-mean-square norm in numpy, in 64 bits, from their definitions."""
import ctypes as C

import numpy as np

from spoc_b200 import _lib as L
from spoc_b200.plugin import _check
from tests.gpu_util import Dev, dev_from

FP8, FP4 = L.MX_FP8, L.MX_FP4
FORMATS = [FP8, FP4]
EMAX = {FP8: 8, FP4: 2}


def grid(fmt):
    """The type's values from zero up; the index is the code without its sign."""
    if fmt == FP4:
        return np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    return np.array([c / 8 * 2.0 ** -6 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])


def round_to(v, fmt):
    """Codes of the values nearest to v, ties to the even code, held at the largest."""
    g = grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    i = np.searchsorted(mid, np.abs(v), side="left")
    tie = (i < mid.size) & (np.abs(v) == mid[np.minimum(i, mid.size - 1)])
    i = i + (tie & (i % 2 == 1))
    return i | np.signbit(v) * (8 if fmt == FP4 else 128)


def tile_offsets(rows, blocks):
    """Where the scale of each row and block lies."""
    r, b = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return (r // 128 * (blocks // 4) + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def quantize(v, fmt):
    """v: rows x K in 64 bits, finite or not.  The two buffers, as bytes."""
    v = np.asarray(v, dtype=np.float64)
    rows, k = v.shape
    kp = -(-k // 128) * 128
    w = np.zeros((rows, kp))
    w[:, :k] = v
    w = w.reshape(rows, kp // 32, 32)
    finite = np.isfinite(w).all(-1)
    w = np.where(finite[..., None], w, 0.0)
    top = np.abs(w).max(-1)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - EMAX[fmt], -127).clip(min=-127)
    codes = round_to(np.ldexp(w, -e[..., None]), fmt).reshape(rows, kp).astype(np.uint8)
    if fmt == FP4:
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    scales = np.zeros(-(-rows // 128) * 128 * kp // 32, np.uint8)
    scales[tile_offsets(rows, kp // 32)] = np.where(finite, e + 127, 255)
    return codes, scales


def values(codes, scales, fmt, k):
    """What the buffers stand for, in 64 bits."""
    rows = codes.shape[0]
    kp = -(-k // 128) * 128
    c = codes.astype(np.int64)
    if fmt == FP4:
        c = np.stack((c & 15, c >> 4), -1).reshape(rows, kp)
    half = 8 if fmt == FP4 else 128
    g = np.append(grid(fmt), np.nan) if fmt == FP8 else grid(fmt)
    q = np.where(c >= half, -1.0, 1.0) * g[c % half]
    s = scales[tile_offsets(rows, kp // 32)].astype(np.int64)
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (q.reshape(rows, kp // 32, 32) * scale[..., None]).reshape(rows, kp)[:, :k]


def rmsnorm(x, residual, weight, eps):
    h = x if residual is None else x + residual      # float32, as it is stored
    d = h.astype(np.float64)
    return h, d * weight.astype(np.float64) / np.sqrt((d * d).mean(-1, keepdims=True) + eps)


def rmsnorm_backward(h, weight, dy, dsum, eps):
    h, weight, dy = (v.astype(np.float64) for v in (h, weight, dy))
    r = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n, g = h * r, dy * weight
    dx = r * (g - n * (g * n).mean(-1, keepdims=True))
    return dx if dsum is None else dx + dsum, (dy * n).sum(0)


class Bytes:
    """A device buffer of bytes between two stretches that must stay as they are."""
    PAD, MARK = 256, 0xA5

    def __init__(self, backend, device, n):
        self.backend, self.n = backend, n
        self.buf = backend.Memory.alloc(device, n + 2 * self.PAD, np.uint8)
        self.clear()

    @property
    def ptr(self):
        return self.buf.ptr + self.PAD

    def clear(self):
        self.backend.Memory.host_to_device(src=np.full(self.n + 2 * self.PAD, self.MARK, np.uint8), dst=self.buf)

    def upload(self, a):
        host = np.full(self.n + 2 * self.PAD, self.MARK, np.uint8)
        host[self.PAD:self.PAD + self.n] = np.ascontiguousarray(a).view(np.uint8).ravel()
        self.backend.Memory.host_to_device(src=host, dst=self.buf)
        return self

    def download(self):
        host = np.empty(self.n + 2 * self.PAD, np.uint8)
        self.backend.Memory.device_to_host(src=self.buf, dst=host)
        assert (host[:self.PAD] == self.MARK).all() and (host[self.PAD + self.n:] == self.MARK).all(), "write outside the buffer"
        return host[self.PAD:self.PAD + self.n].copy()

    def free(self):
        self.backend.Memory.free(self.buf)


def mx_bytes(fmt, rows, k):
    c, s = C.c_uint64(), C.c_uint64()
    _check(L.load().sb200_mx_bytes(fmt, rows, k, C.byref(c), C.byref(s)))
    return c.value, s.value


class Mx:
    """A microscaled matrix on the device."""

    def __init__(self, backend, device, fmt, rows, k, buffers=None):
        self.fmt, self.rows, self.k = fmt, rows, k
        c, s = mx_bytes(fmt, rows, k)
        self.codes, self.scales = Bytes(backend, device, c), Bytes(backend, device, s)
        if buffers is not None:
            self.codes.upload(buffers[0])
            self.scales.upload(buffers[1])

    def download(self):
        return self.codes.download().reshape(self.rows, -1), self.scales.download()

    def free(self):
        self.codes.free()
        self.scales.free()


class Keep:
    """Device arrays that are given back together."""

    def __init__(self, backend, device):
        self.backend, self.device, self.held = backend, device, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for h in self.held:
            h.free()

    def _held(self, h):
        self.held.append(h)
        return h

    def f32(self, array, offset=0):
        return self._held(dev_from(self.backend, self.device, array, offset=offset))

    def out(self, n, offset=0):
        return self._held(Dev(self.backend, self.device, n, offset=offset))

    def mx(self, fmt, rows, k, buffers=None):
        return self._held(Mx(self.backend, self.device, fmt, rows, k, buffers))

    def bytes(self, n):
        return self._held(Bytes(self.backend, self.device, n))


def gemm_mx(device, a, b, d, ldd=None, alpha=1.0, c=None, ldc=None, beta=0.0, bias=None, act=0, stream=0, m=None, n=None):
    m, n = a.rows if m is None else m, b.rows if n is None else n
    _check(L.load().sb200_gemm_mx(device.id, stream, a.fmt, b.fmt, m, n, a.k, a.codes.ptr, a.scales.ptr, b.codes.ptr, b.scales.ptr, d.ptr,
                                  ldd or n, alpha, c.ptr if c else 0, ldc or n, beta, bias.ptr if bias else 0, act))
