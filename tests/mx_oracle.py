"""MXFP4 in 64 bits, plainly: what yl_mx_* compute, in numpy, block by block as include/yolo2_hip.h states it."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUES = np.concatenate([GRID, -GRID])


def blocks(k):
    return (k + 31) // 32


def quantize(x):
    """float64 [rows, k] (values of a narrower type) -> codes uint8 [rows, 32 * kb], scale bytes uint8 [rows, kb]."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    kb = blocks(k)
    full = np.zeros((rows, kb * 32))
    full[:, :k] = x
    full = full.reshape(rows, kb, 32)
    bad = ~np.isfinite(full).all(axis=2)
    full = np.where(bad[:, :, None], 0.0, full)
    top = np.abs(full).max(axis=2)
    _, e = np.frexp(top)                                  # top = m 2^e, 1/2 <= m < 1: floor(log2 top) = e - 1
    e = np.where(top == 0, -127, np.maximum(e - 1 - 2, -127)).astype(int)
    a = np.abs(full) / np.exp2(e.astype(np.float64))[:, :, None]
    # nearest, ties to the even code, saturated
    d = np.abs(a[..., None] - GRID)
    near = d.min(axis=-1)
    first = d.argmin(axis=-1)
    tie = (np.take_along_axis(d, np.minimum(first + 1, 7)[..., None], -1)[..., 0] == near) & (first < 7)
    code = np.where(tie & (first % 2 == 1), first + 1, first)
    code = code + 8 * np.signbit(full)
    code = np.where(bad[:, :, None], 0, code)
    return code.reshape(rows, kb * 32).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale, k):
    """float64 [rows, k]; NaN where the scale byte is 255."""
    v = VALUES[code].reshape(code.shape[0], -1, 32)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return (v * s[:, :, None]).reshape(code.shape[0], -1)[:, :k]


def rounded(x):
    code, scale = quantize(x)
    return values(code, scale, np.asarray(x).shape[1])


def unpack(codes):
    """uint8 [rows, 16 * ld] as the library holds them -> one code a value."""
    out = np.empty((codes.shape[0], codes.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = codes & 15, codes >> 4
    return out


def pack(code, ld=None):
    kb = code.shape[1] // 32
    full = np.zeros((code.shape[0], (ld or kb) * 32), np.uint8)
    full[:, :code.shape[1]] = code
    return full[:, 0::2] | (full[:, 1::2] << 4)


def activate(v, name):
    """activate() of the reference (src/additionally.h:66-165) in 64 bits."""
    return {
        "linear": lambda: v,
        "leaky": lambda: np.where(v > 0, v, 0.1 * v),
        "relu": lambda: np.where(v > 0, v, 0.0),
        "logistic": lambda: 1 / (1 + np.exp(-v)),
        "loggy": lambda: 2 / (1 + np.exp(-v)) - 1,
        "tanh": lambda: np.tanh(v),
        "elu": lambda: np.where(v >= 0, v, np.expm1(np.minimum(v, 0))),
        "relie": lambda: np.where(v > 0, v, 0.01 * v),
        "ramp": lambda: np.where(v > 0, v, 0.0) + 0.1 * v,
        "hardtan": lambda: np.clip(v, -1, 1),
        "lhtan": lambda: np.where(v < 0, .001 * v, np.where(v > 1, .001 * (v - 1) + 1, v)),
        "plse": lambda: np.where(v < -4, .01 * (v + 4), np.where(v > 4, .01 * (v - 4) + 1, .125 * v + .5)),
    }[name]()


def windows(x, batch, h, w, size, stride, pad):
    """rows [batch * h * w, c] of a map -> [batch * oh * ow, size * size * c]."""
    c = x.shape[1]
    m = np.zeros((batch, h + 2 * pad, w + 2 * pad, c))
    m[:, pad:pad + h, pad:pad + w] = x.reshape(batch, h, w, c)
    oh, ow = (h + 2 * pad - size) // stride + 1, (w + 2 * pad - size) // stride + 1
    out = np.empty((batch, oh, ow, size * size, c))
    for ky in range(size):
        for kx in range(size):
            out[:, :, :, ky * size + kx] = m[:, ky:ky + stride * (oh - 1) + 1:stride, kx:kx + stride * (ow - 1) + 1:stride]
    return out.reshape(batch * oh * ow, size * size * c), oh, ow


def filter_rows(w):
    """[n, c, size, size] -> [n, size * size * c'], c' = c padded by zeros to whole blocks."""
    n, c, size, _ = w.shape
    full = np.zeros((n, size, size, blocks(c) * 32))
    full[..., :c] = np.transpose(w, (0, 2, 3, 1))
    return full.reshape(n, -1)


# half a step of rounding to the type, relative to the value, and the smallest step's half (where values are subnormal)
HALF_STEP = {"float32": (2.0 ** -24, 2.0 ** -150), "float16": (2.0 ** -11, 2.0 ** -25), "bfloat16": (2.0 ** -8, 2.0 ** -134)}


def product_tolerance(a, b, bias, act, residual, dtype):
    """How far activation(a b^T + bias) + residual may be from its value in 64 bits.

    Products of two codes and two powers of two are exact.  The matrix instruction adds the 64 products of a step to the FP32
    accumulator; with S = sum |a_k b_k| every partial sum is at most S, and a step is counted with a whole step of FP32, 2^-23 S (twice
    a rounding: its addends are aligned to the largest of them and not all rounded one by one).  A split of the summed axis adds at most
    16 more additions.  The bias, the activation (slope at most 1.1; its own rounding) and the residual round once each, 2^-24 of
    what they hold; the result rounds once to its type."""
    s = np.abs(a) @ np.abs(b).T
    steps = (blocks(a.shape[1]) + 1) // 2 + 16
    tol = steps * 2.0 ** -23 * s
    v = a @ b.T
    if bias is not None:
        v = v + bias
        tol = tol + 2.0 ** -24 * (np.abs(v) + tol)
    y = activate(v, act)
    tol = 1.1 * tol + (2.0 ** -23 * np.abs(y) + 2.0 ** -24 if act != "linear" else 0)     # logistic and loggy round near 1
    if residual is not None:
        y = y + residual
        tol = tol + 2.0 ** -24 * (np.abs(y) + tol)
    half, least = HALF_STEP[dtype]
    return y, tol + half * (np.abs(y) + tol) + least
