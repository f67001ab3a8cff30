"""Performance cases of the microscaled operators: root-mean-square norm with the residual's addition and its gradient,
quantisation to 8 and 4 bits with a power-of-two scale for every 32 values, and products of such matrices.

A microscaled matrix of `rows` x `K` is held in two buffers: `codes`, row by row, K padded with zeros to a multiple of 128
(fp8: one e4m3 byte a value; fp4: two e2m1 values a byte, the first in the low half), and `scales`, one exponent byte (e8m0)
for every 32 values of a row, in tiles of 128 rows x 4 scales: byte (row % 32) * 16 + (row % 128) // 32 * 4 + scale % 4 of
tile (row // 128, scale // 4), tiles row by row, what is past the last row and K zero.  The scale of a block is 2^(floor(log2(
largest magnitude)) - e), e the exponent of the type's largest value (8 for e4m3, 2 for e2m1); values are rounded to the
nearest, ties to even, and held at the type's largest value.

Kinds of case:

* ``norm``: sum = x + residual (rounded to float32: the stream that the next layer adds to), y = sum * weight / sqrt(mean(sum^2)
  + eps), y in float32 or microscaled.  A code is the rounding of the exact y of that sum, so the plain form computes y in 64
  bits: in 32 bits values next to a rounding border would fall on either side;
* ``norm_backward``: gradients of x and weight from the gradient of y (a microscaled y passes its gradient through), plus the
  gradient that reaches the sum from the layers behind;
* ``quantize``: a float32 matrix, or its transpose, to codes and scales; the 4-bit cases read the values back;
* ``gemm``: D = act(alpha * A . B^T + beta * C + bias) of microscaled A (M x K) and B (N x K);
* ``layer``: norm to 8 bits and the product with 4-bit weights, as a layer of a network runs them;
* ``linear_backward``: both gradients of y = x . W^T in 8 bits: four quantisations and two products.

``listed`` gives the fixed cases, ``draw`` one more case of the same ranges, ``prepare`` what the program holds before the
call, ``run`` one pass (in elementary torch operations, or through the framework where ``own`` is true), ``work`` the bytes
and operations a pass cannot do without, ``exact`` the result in 64 bits.
"""
import numpy as np
import torch

own = False

BLOCK = 32
LARGEST = {"fp8": 448.0, "fp4": 6.0}        # largest value of the type
EMAX = {"fp8": 8, "fp4": 2}                 # its exponent
EMIN = {"fp8": -6, "fp4": 0}                # exponent of the smallest normal value
MANTISSA = {"fp8": 3, "fp4": 1}             # explicit mantissa bits
BITS = {"fp8": 8, "fp4": 4}
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
EPS = 1e-5
MOST_VALUES = 8192 * 8192
MOST_MACS = 8192 ** 3


def listed():
    return [
        # one token in front of a layer: a launch and a row of 4096, nearly all latency
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096, "format": "fp8", "residual": True},
        # a long prompt in front of a layer of 8192 columns: HBM bandwidth
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 8192, "format": "fp8", "residual": True},
        # rows that start off a 16-byte boundary, a last block of 31 values, y in float32
        {"name": "norm_ragged", "kind": "norm", "rows": 1531, "cols": 2047, "format": "f32", "residual": False},
        # a training step's backward pass through the norm
        {"name": "norm_backward", "kind": "norm_backward", "rows": 8192, "cols": 4096, "residual": True},
        # a weight matrix stored K x N brought into the form the product reads
        {"name": "quantize_weights", "kind": "quantize", "rows": 8192, "cols": 8192, "format": "fp8", "transposed": True},
        # 4 bits and back (training that sees its own rounding), ragged
        {"name": "quantize_ragged", "kind": "quantize", "rows": 2047, "cols": 1021, "format": "fp4", "transposed": False},
        # one token against 4-bit weights: the weights are read once
        {"name": "gemm_token", "kind": "gemm", "m": 1, "n": 4096, "k": 4096, "a": "fp8", "b": "fp4", "epilogue": False},
        # a small batch through a wide layer, bias and clamp
        {"name": "gemm_64_rows", "kind": "gemm", "m": 64, "n": 16384, "k": 4096, "a": "fp8", "b": "fp4", "epilogue": True},
        # a ragged product in 8 bits
        {"name": "gemm_ragged", "kind": "gemm", "m": 1531, "n": 2047, "k": 1021, "a": "fp8", "b": "fp8", "epilogue": True},
        # the largest product, 4 bits on both sides
        {"name": "gemm_8192_fp4", "kind": "gemm", "m": 8192, "n": 8192, "k": 8192, "a": "fp4", "b": "fp4", "epilogue": False},
        # a prompt through norm and product
        {"name": "layer_prompt", "kind": "layer", "m": 2048, "n": 4096, "k": 4096, "a": "fp8", "b": "fp4"},
        # the backward pass of a linear layer over a batch of tokens
        {"name": "linear_backward", "kind": "linear_backward", "m": 4096, "n": 4096, "k": 2048, "a": "fp8", "b": "fp8"},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def _size(rng, low, high):
    """A size between low and high, evenly in its logarithm; half of the time a multiple of 32."""
    v = _log(rng, low, high)
    return min(high, (v + 31) // 32 * 32) if rng.random() < 0.5 else v


def _dims(rng, low_m, limit):
    while True:
        m = _log(rng, low_m, 8192)
        n, k = _size(rng, 64, 16384), _size(rng, 32, 16384)
        if m * n * k <= limit:
            return {"m": m, "n": n, "k": k}


def draw(rng):
    kind = rng.choice(("norm", "norm", "norm_backward", "quantize", "quantize", "gemm", "gemm", "gemm", "layer", "linear_backward"))
    if kind in ("norm", "norm_backward", "quantize"):
        while True:
            rows, cols = _log(rng, 1, 16384), _size(rng, 32, 16384)
            if rows * cols <= MOST_VALUES:
                break
        case = {"kind": kind, "rows": rows, "cols": cols}
        if kind == "norm":
            return {**case, "format": rng.choice(("fp8", "fp8", "fp4", "f32")), "residual": rng.random() < 0.7}
        if kind == "norm_backward":
            return {**case, "residual": rng.random() < 0.7}
        return {**case, "format": rng.choice(("fp8", "fp4")), "transposed": rng.random() < 0.5}
    if kind == "gemm":
        a, b = rng.choice((("fp8", "fp8"), ("fp8", "fp4"), ("fp4", "fp4")))
        return {"kind": kind, **_dims(rng, 1, MOST_MACS), "a": a, "b": b, "epilogue": rng.random() < 0.5}
    if kind == "layer":
        a, b = rng.choice((("fp8", "fp8"), ("fp8", "fp4"), ("fp4", "fp4")))
        return {"kind": kind, **_dims(rng, 1, MOST_MACS // 4), "a": a, "b": b}
    return {"kind": kind, **_dims(rng, 64, MOST_MACS // 4), "a": "fp8", "b": "fp8"}


# ------------------------------------------------------------------ plain form
def _pow2(e):
    """2^e in float64 for whole e in [-1022, 1023]."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exponent(v):
    """floor(log2(|v|)), and a number below every exponent that counts for zero."""
    return torch.where(v == 0, -1000, torch.frexp(v)[1] - 1)


def _rounded(v, fmt):
    """v rounded to the nearest value of the type, ties to even, held at its largest."""
    step = _pow2(_exponent(v).clamp(EMIN[fmt], EMAX[fmt]) - MANTISSA[fmt])
    return ((v / step).round() * step).clamp(-LARGEST[fmt], LARGEST[fmt])


def _quantized(v, fmt):
    """Codes and scales of the rows of v."""
    rows, k = v.shape
    kp = (k + 127) // 128 * 128
    v = torch.nn.functional.pad(v.double(), (0, kp - k)).view(rows, kp // BLOCK, BLOCK)
    e = (_exponent(v.abs().amax(-1)) - EMAX[fmt]).clamp(min=-127)
    q = _rounded(v * _pow2(-e).unsqueeze(-1), fmt).view(rows, kp)
    if fmt == "fp8":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        level = torch.bucketize(q.abs(), torch.tensor(FP4_VALUES[:8], dtype=torch.float64, device=v.device)).to(torch.uint8)
        level |= torch.signbit(q).to(torch.uint8) << 3
        codes = level[:, 0::2] | level[:, 1::2] << 4
    tiles = (rows + 127) // 128
    s = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 0, 0, tiles * 128 - rows))
    return codes, s.view(tiles, 4, 32, kp // 128, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _values(codes, scales, fmt, k, dtype=torch.float32):
    """What codes and scales stand for."""
    rows = codes.shape[0]
    if fmt == "fp8":
        q = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        table = torch.tensor(FP4_VALUES, dtype=dtype, device=codes.device)
        q = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
    kp, tiles = (k + 127) // 128 * 128, (rows + 127) // 128
    s = scales.view(tiles, kp // 128, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles * 128, kp // BLOCK)[:rows]
    s = _pow2(s.to(torch.int64) - 127).to(dtype)
    return (q.reshape(rows, kp // BLOCK, BLOCK) * s.unsqueeze(-1)).view(rows, kp)[:, :k]


def _seen(codes, scales, fmt):
    """Codes and scales of 8 bits as numbers of their types."""
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def _plain_norm(s):
    h = s["x"] if s["residual"] is None else s["x"] + s["residual"]
    fmt = s["case"].get("format") or s["case"]["a"]
    if fmt == "f32":
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"]
        return h, y, None
    d = h.double()
    y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()
    return h, *_quantized(y, fmt)


def _plain_product(a, b, s, epilogue):
    d = a @ b.T
    if epilogue:
        d = s["alpha"] * d + s["bias"]
        if s["c"] is not None:
            d = d + s["beta"] * s["c"]
        d = d * (d > 0)
    return d


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        h, y, scales = _plain_norm(s)
        out = {} if s["residual"] is None else {"sum": h}
        if case["format"] == "f32":
            return {**out, "y": y}
        if case["format"] == "fp4":
            return {**out, "values": _values(y, scales, "fp4", case["cols"])}
        return {**out, **_seen(y, scales, "fp8")}
    if kind == "norm_backward":
        h, dy, w = s["h"], s["dy"], s["weight"]
        r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        n, g = h * r, dy * w
        dx = r * (g - n * (g * n).mean(-1, keepdim=True))
        if s["dsum"] is not None:
            dx = dx + s["dsum"]
        return {"dx": dx, "dweight": (dy * n).sum(0)}
    if kind == "quantize":
        codes, scales = _quantized(s["x"].T if case["transposed"] else s["x"], case["format"])
        if case["format"] == "fp4":
            return {"values": _values(codes, scales, "fp4", case["cols"])}
        return _seen(codes, scales, "fp8")
    if kind == "gemm":
        a = _values(*s["a"], case["a"], case["k"])
        b = _values(*s["b"], case["b"], case["k"])
        return _plain_product(a, b, s, case["epilogue"])
    if kind == "layer":
        h, codes, scales = _plain_norm(s)
        a = _values(codes, scales, case["a"], case["k"])
        return {"sum": h, "d": _plain_product(a, _values(*s["b"], case["b"], case["k"]), s, True)}
    back = [_values(*_quantized(v, f), f, v.shape[1]) for v, f in ((s["dy"], "fp8"), (s["w"].T, "fp8"), (s["dy"].T, "fp8"), (s["x"].T, "fp8"))]
    return {"dx": back[0] @ back[1].T, "dw": back[2] @ back[3].T}


# ------------------------------------------------------------------ the framework's calls
_loaded = None


def _library():
    global _loaded
    if _loaded is None:
        from spoc_b200 import Backend, _lib
        backend = Backend()
        backend.Device.init()
        backend.Device.set_current(backend.Device.get(0))
        _loaded = _lib.load()
    return _loaded


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _checked(code):
    if code:
        raise RuntimeError(_library().sb200_last_error_string().decode())


def _mx(fmt):
    return BITS.get(fmt, 0)     # SB200_MX_FP8, SB200_MX_FP4; 0: none


def _own_norm(lib, s, fmt, y, codes, scales):
    x, r, h = s["x"], s["residual"], s["sum"]
    rows, cols = x.shape
    _checked(lib.sb200_rmsnorm_f32(0, 0, rows, cols, x.data_ptr(), x.stride(0), _ptr(r), cols, s["weight"].data_ptr(), EPS, _ptr(h), cols,
                                   _ptr(y), cols, _mx(fmt), _ptr(codes), _ptr(scales)))


def _own_quantize(lib, fmt, x, transposed, codes, scales):
    rows, cols = x.shape[::-1] if transposed else x.shape
    _checked(lib.sb200_mx_quantize(0, 0, _mx(fmt), rows, cols, x.data_ptr(), x.stride(0), int(transposed), codes.data_ptr(), scales.data_ptr()))


def _own_gemm(lib, fmt_a, fmt_b, k, a, b, d, alpha=1.0, c=None, beta=0.0, bias=None, act=0):
    m, n = d.shape
    _checked(lib.sb200_gemm_mx(0, 0, _mx(fmt_a), _mx(fmt_b), m, n, k, a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(),
                               d.data_ptr(), n, alpha, _ptr(c), n, beta, _ptr(bias), act))
    return d


def _own(s):
    lib, case = _library(), s["case"]
    kind = case["kind"]
    if kind == "norm":
        fmt, out = case["format"], {} if s["residual"] is None else {"sum": s["sum"]}
        if fmt == "f32":
            _own_norm(lib, s, fmt, s["y"], None, None)
            return {**out, "y": s["y"]}
        _own_norm(lib, s, fmt, None, s["codes"], s["scales"])
        if fmt == "fp8":
            return {**out, **_seen(s["codes"], s["scales"], fmt)}
        _checked(lib.sb200_mx_dequantize(0, 0, _mx(fmt), case["rows"], case["cols"], s["codes"].data_ptr(), s["scales"].data_ptr(),
                                         s["y"].data_ptr(), case["cols"]))
        return {**out, "values": s["y"]}
    if kind == "norm_backward":
        h, dy = s["h"], s["dy"]
        rows, cols = h.shape
        _checked(lib.sb200_rmsnorm_backward_f32(0, 0, rows, cols, h.data_ptr(), cols, s["weight"].data_ptr(), EPS, dy.data_ptr(), cols,
                                                _ptr(s["dsum"]), cols, s["dx"].data_ptr(), cols, s["dweight"].data_ptr(),
                                                s["workspace"].data_ptr(), s["workspace"].numel()))
        return {"dx": s["dx"], "dweight": s["dweight"]}
    if kind == "quantize":
        fmt = case["format"]
        _own_quantize(lib, fmt, s["x"], case["transposed"], s["codes"], s["scales"])
        if fmt == "fp8":
            return _seen(s["codes"], s["scales"], fmt)
        _checked(lib.sb200_mx_dequantize(0, 0, _mx(fmt), case["rows"], case["cols"], s["codes"].data_ptr(), s["scales"].data_ptr(),
                                         s["y"].data_ptr(), case["cols"]))
        return {"values": s["y"]}
    if kind == "gemm":
        if not case["epilogue"]:
            return _own_gemm(lib, case["a"], case["b"], case["k"], s["a"], s["b"], s["d"])
        return _own_gemm(lib, case["a"], case["b"], case["k"], s["a"], s["b"], s["d"], s["alpha"], s["c"], s["beta"], s["bias"], 1)
    if kind == "layer":
        _own_norm(lib, s, case["a"], None, s["codes"], s["scales"])
        d = _own_gemm(lib, case["a"], case["b"], case["k"], (s["codes"], s["scales"]), s["b"], s["d"], s["alpha"], None, 0.0, s["bias"], 1)
        return {"sum": s["sum"], "d": d}
    m, n, k = case["m"], case["n"], case["k"]
    for x, transposed, to in ((s["dy"], False, s["dy_rows"]), (s["w"], True, s["w_cols"]), (s["dy"], True, s["dy_cols"]), (s["x"], True, s["x_cols"])):
        _own_quantize(lib, "fp8", x, transposed, *to)
    dx = _own_gemm(lib, "fp8", "fp8", n, s["dy_rows"], s["w_cols"], s["dx"])
    dw = _own_gemm(lib, "fp8", "fp8", m, s["dy_cols"], s["x_cols"], s["dw"])
    return {"dx": dx, "dw": dw}


# ------------------------------------------------------------------ state
def _buffers(rows, k, fmt):
    kp = (k + 127) // 128 * 128
    codes = torch.empty(rows, kp * BITS[fmt] // 8, dtype=torch.uint8, device="cuda")
    return codes, torch.empty((rows + 127) // 128 * 128 * kp // BLOCK, dtype=torch.uint8, device="cuda")


def _activations(g, rows, cols):
    """What a layer's input looks like: normal values, and a few columns that stand out."""
    x = torch.empty(rows, cols, device="cuda").normal_(0.0, 1.0, generator=g)
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _gradients(g, rows, cols):
    """Gradients of a batch: normal, each token with a magnitude of its own."""
    return torch.empty(rows, cols, device="cuda").normal_(0.0, 1e-3, generator=g) * torch.empty(rows, 1, device="cuda").uniform_(0.1, 3.0, generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    s = {"case": dict(case)}

    def normal(rows, cols, scale):
        return torch.empty(rows, cols, device="cuda").normal_(0.0, scale, generator=g)

    def norm_inputs(rows, cols, residual):
        s["x"] = _activations(g, rows, cols)
        s["residual"] = _activations(g, rows, cols) if residual else None
        s["weight"] = torch.empty(cols, device="cuda").uniform_(0.2, 1.8, generator=g)
        s["sum"] = torch.empty(rows, cols, device="cuda") if residual else None

    if kind == "norm":
        rows, cols, fmt = case["rows"], case["cols"], case["format"]
        norm_inputs(rows, cols, case["residual"])
        s["y"] = torch.empty(rows, cols, device="cuda") if fmt != "fp8" else None
        s["codes"], s["scales"] = _buffers(rows, cols, fmt) if fmt != "f32" else (None, None)
        return s
    if kind == "norm_backward":
        rows, cols = case["rows"], case["cols"]
        s["h"], s["dy"] = _activations(g, rows, cols), _gradients(g, rows, cols)
        s["dsum"] = _gradients(g, rows, cols) if case["residual"] else None
        s["weight"] = torch.empty(cols, device="cuda").uniform_(0.2, 1.8, generator=g)
        s["dx"], s["dweight"] = torch.empty(rows, cols, device="cuda"), torch.empty(cols, device="cuda")
        s["workspace"] = torch.empty(4 * cols * min(rows, 512), dtype=torch.uint8, device="cuda")    # partial sums of dweight
        return s
    if kind == "quantize":
        rows, cols, fmt = case["rows"], case["cols"], case["format"]
        s["x"] = normal(cols, rows, cols ** -0.5) if case["transposed"] else _activations(g, rows, cols)
        s["y"] = torch.empty(rows, cols, device="cuda") if fmt == "fp4" else None
        s["codes"], s["scales"] = _buffers(rows, cols, fmt)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "linear_backward":
        s["x"], s["w"], s["dy"] = _activations(g, m, k), normal(n, k, k ** -0.5), _gradients(g, m, n)
        s["dy_rows"], s["w_cols"] = _buffers(m, n, "fp8"), _buffers(k, n, "fp8")
        s["dy_cols"], s["x_cols"] = _buffers(n, m, "fp8"), _buffers(k, m, "fp8")
        s["dx"], s["dw"] = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda")
        return s
    s["b"] = _quantized(normal(n, k, k ** -0.5), case["b"])
    s["d"] = torch.empty(m, n, device="cuda")
    s["alpha"], s["beta"], s["c"] = 1.5, 0.5, None
    s["bias"] = normal(1, n, 0.1).view(n)
    if kind == "gemm":
        s["a"] = _quantized(_activations(g, m, k), case["a"])
        s["c"] = normal(m, n, 1.0) if case["epilogue"] else None
        return s
    norm_inputs(m, k, True)
    s["codes"], s["scales"] = _buffers(m, k, case["a"])
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work
def _mx_bytes(rows, k, fmt):
    return rows * k * BITS[fmt] / 8 + rows * ((k + BLOCK - 1) // BLOCK)


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_backward", "quantize"):
        rows, cols = case["rows"], case["cols"]
        values = rows * cols
        if kind == "norm_backward":
            return {"bytes": 4.0 * (values * (4 if case["residual"] else 3) + 2 * cols), "flops": 12.0 * values}
        fmt = case["format"]
        out = {"f32": 4.0 * values, "fp8": _mx_bytes(rows, cols, "fp8"), "fp4": 4.0 * values}[fmt]
        if kind == "quantize":
            return {"bytes": 4.0 * values + out, "flops": 3.0 * values}
        return {"bytes": 4.0 * (values * (3 if case["residual"] else 1) + cols) + out, "flops": 8.0 * values}
    m, n, k = case["m"], case["n"], case["k"]
    if kind == "linear_backward":
        return {"bytes": 4.0 * (m * n + 2 * m * k + 2 * n * k), "flops": 4.0 * m * n * k}
    b = _mx_bytes(n, k, case["b"])
    if kind == "layer":
        return {"bytes": 4.0 * (3 * m * k + k + n + m * n) + b, "flops": 2.0 * m * n * k + 8.0 * m * k}
    extra = m * n + n if case["epilogue"] else 0
    return {"bytes": _mx_bytes(m, k, case["a"]) + b + 4.0 * (m * n + extra), "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _power(e):
    """2^e for whole e in [-400, 400]."""
    return torch.from_numpy(np.ldexp(1.0, np.arange(-400, 401))).cuda()[e.long() + 400]


def _grid(fmt):
    """The type's values from zero up, in float64, by their definition: the index is the code."""
    if fmt == "fp4":
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    code = torch.arange(127, device="cuda")
    e, f = code // 8, (code % 8).double() / 8
    return torch.where(e == 0, f * 2.0 ** -6, (1 + f) * _power(e - 7))


def _nearest(v, fmt):
    """The index of the nearest value of the type to each |v|, an even one where two are as near."""
    grid = _grid(fmt)
    middle = (grid[1:] + grid[:-1]) / 2
    v = v.abs().contiguous()
    i = torch.bucketize(v, middle)
    tie = v == middle[i.clamp(max=middle.numel() - 1)]
    return i + (tie & (i % 2 == 1) & (i < middle.numel())).long()


def _exact_quantized(v, fmt):
    """The scaled values that the codes of v's rows stand for, its scales, and the values."""
    rows, k = v.shape
    kp = -(-k // 128) * 128
    wide = v.new_zeros(rows, kp)
    wide[:, :k] = v
    wide = wide.view(rows, -1, BLOCK)
    top = wide.abs().amax(-1).contiguous()
    powers = _power(torch.arange(-140, 129, device="cuda"))
    e = torch.bucketize(top, powers, right=True) - 1 - 140 - {"fp8": 8, "fp4": 2}[fmt]
    scale = _power(e.clamp(min=-127))
    scaled = wide / scale.unsqueeze(-1)
    q = _grid(fmt)[_nearest(scaled, fmt)] * torch.sign(scaled)
    return q, scale, (q * scale.unsqueeze(-1)).reshape(rows, kp)[:, :k]


def _exact_tiles(scale):
    """Scales in the order they are held in."""
    rows, blocks = scale.shape
    tiles = -(-rows // 128)
    held = torch.full((tiles * 128, blocks), 2.0 ** -127, dtype=torch.float64, device="cuda")
    held[:rows] = scale
    row = torch.arange(tiles * 128, device="cuda").view(-1, 1)
    col = torch.arange(blocks, device="cuda").view(1, -1)
    place = ((row // 128) * (blocks // 4) + col // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + col % 4
    out = torch.empty(held.numel(), dtype=torch.float64, device="cuda")
    out[place.reshape(-1)] = held.reshape(-1)
    return out


def _exact_of(codes, scales, fmt, k):
    """The values of a microscaled matrix in memory, byte by byte."""
    rows = codes.shape[0]
    kp = -(-k // 128) * 128
    byte = codes.long()
    nibbles = byte if fmt == "fp8" else torch.stack((byte % 16, byte // 16), 2).view(rows, kp)
    half = 128 if fmt == "fp8" else 8
    q = _grid(fmt)[nibbles % half] * (1 - 2 * (nibbles // half).double())
    row = torch.arange(rows, device="cuda").view(-1, 1)
    col = torch.arange(kp // BLOCK, device="cuda").view(1, -1)
    at = ((row // 128) * (kp // 128) + col // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + col % 4
    scale = _power(scales[at].long() - 127)
    return (q.view(rows, -1, BLOCK) * scale.unsqueeze(-1)).view(rows, kp)[:, :k]


def _exact_norm(s):
    h = (s["x"] if s["residual"] is None else s["x"] + s["residual"]).double()      # the sum is a float32 by definition
    length = torch.sqrt((h * h).sum(1) / h.shape[1] + EPS)
    return h, h * s["weight"].double() / length.view(-1, 1)


def _exact_product(s, a, b):
    d = s["alpha"] * (a @ b.transpose(0, 1)) + s["bias"].double()
    if s["c"] is not None:
        d += s["beta"] * s["c"].double()
    return torch.clamp(d, min=0.0)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h, y = _exact_norm(s)
        out = {"sum": h} if case["residual"] else {}
        if case["format"] == "f32":
            return {**out, "y": y}
        q, scale, values = _exact_quantized(y, case["format"])
        if case["format"] == "fp4":
            return {**out, "values": values}
        return {**out, "codes": q.reshape(case["rows"], -1), "scales": _exact_tiles(scale)}
    if kind == "norm_backward":
        h, dy, w = s["h"].double(), s["dy"].double(), s["weight"].double()
        cols = case["cols"]
        length = torch.sqrt((h * h).sum(1, keepdim=True) / cols + EPS)
        along = (dy * w * h).sum(1, keepdim=True) / cols
        dx = dy * w / length - h * along / length ** 3
        if case["residual"]:
            dx += s["dsum"].double()
        return {"dx": dx, "dweight": torch.einsum("rc,rc->c", dy, h / length)}
    if kind == "quantize":
        x = s["x"].double()
        q, scale, values = _exact_quantized(x.transpose(0, 1).contiguous() if case["transposed"] else x, case["format"])
        if case["format"] == "fp4":
            return {"values": values}
        return {"codes": q.reshape(case["rows"], -1), "scales": _exact_tiles(scale)}
    if kind == "linear_backward":
        dy, w, x = s["dy"].double(), s["w"].double(), s["x"].double()
        turned = [v.transpose(0, 1).contiguous() for v in (w, dy, x)]
        rows, w_cols, dy_cols, x_cols = (_exact_quantized(v, "fp8")[2] for v in (dy, *turned))
        return {"dx": rows @ w_cols.transpose(0, 1), "dw": dy_cols @ x_cols.transpose(0, 1)}
    b = _exact_of(*s["b"], case["b"], case["k"])
    if kind == "layer":
        h, y = _exact_norm(s)
        return {"sum": h, "d": _exact_product(s, _exact_quantized(y, case["a"])[2], b)}
    a = _exact_of(*s["a"], case["a"], case["k"])
    return _exact_product(s, a, b) if case["epilogue"] else a @ b.transpose(0, 1)
