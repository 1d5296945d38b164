"""MXFP4 operators on torch tensors of a GPU: the yl_mx_* entries of include/yolo2_hip.h (formats and formulas stand there).

    q = mx.quantize(x)                         # [..., k] FP32 / FP16 / BF16 -> Matrix (one row a k-vector)
    y = mx.matmul(q, w, bias=b, activation="leaky")
    y = mx.linear(x, w, bias=b)                # == matmul(quantize(x), w), in one call
    f = mx.quantize_filters(weights)           # [n, c, size, size] -> Matrix
    y = mx.conv2d(mx.quantize_nchw(x), f, batch, h, w, size, stride, pad, bias=b, activation="leaky", residual=r)

Every call runs on the current stream of its tensors' device and returns without waiting.  There are no derivatives: a call on a
tensor that requires a gradient, or that carries a tangent of forward mode, raises.  Plumbing only: all arithmetic happens in libyolo2hip.so."""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from ._lib import Dense, MxConv, MxEpilogue, MxMatrix, YoloHipError, lib, check

BLOCK = 32
ACTIVATIONS = {"logistic": 0, "relu": 1, "relie": 2, "linear": 3, "ramp": 4, "tanh": 5, "plse": 6, "leaky": 7, "elu": 8, "loggy": 9,
               "stair": 10, "hardtan": 11, "lhtan": 12}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ref = C.byref


def _fail(what: str):
    raise YoloHipError("mx: " + what)


def _tensor(t, name: str, device: Optional[int] = None) -> int:
    """The index of the GPU that t is on; -> raises unless t is a tensor on a GPU (on `device`, if given) that needs no gradient and
    whose memory holds its values."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail("%s is not a tensor on a GPU" % name)
    at = t.get_device()
    if device is not None and at != device:
        _fail("%s is on cuda:%d, not on cuda:%d" % (name, at, device))
    if t.requires_grad and torch.is_grad_enabled():
        _fail("%s requires a gradient, and there is no backward pass: detach it, or call under torch.no_grad()" % name)
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _fail("%s carries a tangent, and there is no forward-mode derivative: unpack it" % name)
    if t.is_neg():
        _fail("%s is a view that stands for the negatives of what its memory holds: call resolve_neg()" % name)
    return at


def _type(t, name: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        _fail("%s is %s: float32, float16 and bfloat16 are taken" % (name, t.dtype))
    return code


def _blocks(k: int) -> int:
    return (k + 4 * BLOCK - 1) // (4 * BLOCK) * 4          # yl_mx_blocks


@functools.lru_cache(maxsize=None)
def _gpu(index: int):
    return torch.device("cuda", index)                     # an index takes torch longer than the device itself


# the current stream of a device as a number; the public way makes an object of it first, which takes longer than a launch
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


class Matrix:
    """rows x k values in MXFP4: codes uint8 [rows, 16 * ld], scales uint8 [rows, ld], ld >= ceil(k / 32) blocks a row."""
    __slots__ = ("k", "rows", "index", "_both", "_codes", "_scales", "_c")

    def __init__(self, codes, scales, k: int):
        self.index = _tensor(codes, "codes")
        _tensor(scales, "scales", self.index)
        self.k = k = int(k)
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            _fail("codes and scales are two-dimensional uint8 tensors")
        rows, ld = scales.shape
        if codes.shape[0] != rows or codes.shape[1] != 16 * ld or not codes.is_contiguous() or not scales.is_contiguous():
            _fail("codes [rows, 16 * ld] and scales [rows, ld] are contiguous and of the same rows and blocks")
        if k < 0 or ld < (k + BLOCK - 1) // BLOCK:
            _fail("k = %d needs %d blocks, the matrix has %d" % (k, (k + BLOCK - 1) // BLOCK, ld))
        self.rows, self._both, self._codes, self._scales = rows, None, codes, scales
        self._c = MxMatrix(codes.data_ptr(), scales.data_ptr(), rows, k, ld)

    @classmethod
    def empty(cls, rows: int, k: int, device) -> "Matrix":
        """A matrix of yl_mx_blocks(k) blocks a row, nothing in it yet; codes and scales share an allocation."""
        ld = _blocks(k)
        self = cls.__new__(cls)
        both = torch.empty(rows * ld * 17, dtype=torch.uint8, device=device)
        at = both.data_ptr()
        self.k, self.rows, self.index, self._both, self._codes, self._scales = k, rows, both.get_device(), both, None, None
        self._c = MxMatrix(at, at + rows * ld * 16, rows, k, ld)
        return self

    # views of the allocation, made when they are asked for; each by itself, so that threads that ask at once get the same ones
    @property
    def codes(self):
        view = self._codes
        if view is None:
            view = self._codes = self._both[:16 * self.rows * self._c.ld].view(self.rows, 16 * self._c.ld)
        return view

    @property
    def scales(self):
        view = self._scales
        if view is None:
            view = self._scales = self._both[16 * self.rows * self._c.ld:].view(self.rows, self._c.ld)
        return view

    @property
    def device(self):
        return (self._codes if self._both is None else self._both).device


def _written(*tensors):
    """Results went into tensors of the caller's: autograd has to know, or a backward pass that saved one computes with what is there now."""
    for t in tensors:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def _matrix(m, name: str, device: Optional[int] = None) -> int:
    if not isinstance(m, Matrix):
        _fail("%s is not an mx.Matrix" % name)
    if device is not None and m.index != device:
        _fail("%s is on cuda:%d, not on cuda:%d" % (name, m.index, device))
    return m.index


def _rows_of(x, name: str) -> Dense:
    """[..., k] as rows of k: the leading axes have to be one run of equal steps."""
    kind, shape = _type(x, name), x.shape
    if len(shape) == 2:
        step, by = x.stride()
        return Dense(x.data_ptr(), kind, 1, shape[0], shape[1], 0, step, by)
    if len(shape) == 0:
        _fail("%s has no axis" % name)
    if len(shape) == 1:
        return Dense(x.data_ptr(), kind, 1, 1, shape[0], 0, 0, x.stride(0))
    try:
        flat = x.view(-1, shape[-1]) if x.numel() else x.reshape(math.prod(shape[:-1]), shape[-1])
    except RuntimeError:
        _fail("the leading axes of %s cannot be taken as one axis of rows: make it contiguous" % name)
    return Dense(x.data_ptr(), kind, 1, flat.shape[0], shape[-1], 0, flat.stride(0), x.stride(-1))


def _map_of(x, name: str) -> Dense:
    """[batch, c, h, w] as one row of channels a pixel."""
    kind = _type(x, name)
    if x.dim() != 4:
        _fail("%s is not [batch, channels, h, w]" % name)
    b, c, h, w = x.shape
    if h > 1 and w > 1 and x.stride(2) != w * x.stride(3):
        _fail("rows of the map %s do not follow one another: make it contiguous" % name)
    return Dense(x.data_ptr(), kind, b, h * w, c, x.stride(0), x.stride(3) if w > 1 else x.stride(2), x.stride(1))


def _quantize(src: Dense, device: int, out: Optional[Matrix]) -> Matrix:
    q = out
    if q is None:
        q = Matrix.empty(src.batch * src.rows, src.k, _gpu(device))
    else:
        _matrix(q, "out", device)
    check(lib.yl_mx_quantize(device, _stream(device), _ref(src), _ref(q._c)), "yl_mx_quantize")
    if out is not None:
        _written(out._both, *((out._codes, out._scales) if out._both is None else ()))
    return q


def quantize(x, out: Optional[Matrix] = None) -> Matrix:
    """x [..., k] -> Matrix of one row a k-vector.  k and the rows may have any strides; more than one leading axis has to be one run of
    equal steps (x.reshape(-1, k) without a copy)."""
    device = _tensor(x, "x")
    return _quantize(_rows_of(x, "x"), device, out)


def quantize_nchw(x, out: Optional[Matrix] = None) -> Matrix:
    """A map [batch, c, h, w] -> Matrix of batch * h * w rows of c values (conv2d's x)."""
    device = _tensor(x, "x")
    return _quantize(_map_of(x, "x"), device, out)


def quantize_filters(w) -> Matrix:
    """Filters [n, c, size, size] -> Matrix of n rows, tap after tap, the channels of each padded by zeros to whole blocks."""
    _tensor(w, "w")
    if w.dim() != 4 or w.shape[2] != w.shape[3]:
        _fail("w is not [filters, channels, size, size]")
    n, c, size, _ = w.shape
    rows = torch.zeros(n, size, size, (c + BLOCK - 1) // BLOCK * BLOCK, dtype=w.dtype, device=w.device)
    rows[..., :c] = w.permute(0, 2, 3, 1)
    return quantize(rows.view(n, rows.shape[1] * rows.shape[2] * rows.shape[3]))


def _dequantize(q: Matrix, out, dst: Dense, given: bool):
    check(lib.yl_mx_dequantize(q.index, _stream(q.index), _ref(q._c), _ref(dst)), "yl_mx_dequantize")
    if given:
        _written(out)
    return out


def dequantize(q: Matrix, dtype=torch.float32, out=None):
    """The values of q, [rows, k]."""
    device = _matrix(q, "q")
    given = out is not None
    if not given:
        out = torch.empty((q.rows, q.k), dtype=dtype, device=_gpu(device))
    else:
        _tensor(out, "out", device)
    return _dequantize(q, out, _rows_of(out, "out"), given)


def dequantize_nchw(q: Matrix, batch: int, h: int, w: int, dtype=torch.float32, out=None):
    """The values of a quantised map, [batch, q.k, h, w]."""
    device = _matrix(q, "q")
    given = out is not None
    if not given:
        out = torch.empty((batch, q.k, h, w), dtype=dtype, device=_gpu(device))
    else:
        _tensor(out, "out", device)
    return _dequantize(q, out, _map_of(out, "out"), given)


def _epilogue(n: int, device: int, bias, activation, residual) -> Optional[MxEpilogue]:
    act = ACTIVATIONS.get(activation, activation)
    if not isinstance(act, int):
        _fail("unknown activation %r" % (activation,))
    if bias is None and residual is None and act == 3:
        return None
    b = r = None
    if bias is not None:
        _tensor(bias, "bias", device)
        if bias.dtype is not torch.float32 or bias.shape != (n,) or not bias.is_contiguous():
            _fail("bias is a contiguous float32 tensor of %d values" % n)
        b = bias.data_ptr()
    if residual is not None:
        r = residual.data_ptr()
    return MxEpilogue(b, act, r, residual.stride(0) if r is not None else 0)


def _linear_args(lead, m: int, w: Matrix, device: int, bias, activation, residual, dtype, out):
    n = w.rows
    if out is None:
        kind = _TYPES.get(dtype)
        if kind is None:
            _fail("dtype is %s: float32, float16 and bfloat16 are made" % dtype)
        out = torch.empty((*lead, n), dtype=dtype, device=_gpu(device))
        y = Dense(out.data_ptr(), kind, 1, m, n, 0, n, 1)
    else:
        _tensor(out, "out", device)
        if tuple(out.shape) != (*lead, n):
            _fail("out is not %s" % ((*lead, n),))
        y = _rows_of(out, "out")
    if residual is not None:
        _tensor(residual, "residual", device)
        if residual.dtype is not out.dtype or residual.shape != out.shape:
            _fail("residual has not the result's type and shape")
        if residual.dim() != 2:
            try:
                residual = residual.view(-1, n) if residual.numel() else residual.reshape(m, n)
            except RuntimeError:
                _fail("the leading axes of residual cannot be taken as one axis of rows: make it contiguous")
        if n > 1 and m and residual.stride(1) != 1:
            _fail("residual's last axis is not contiguous")
    return out, y, _epilogue(n, device, bias, activation, residual)


def matmul(x: Matrix, w: Matrix, bias=None, activation="linear", residual=None, dtype=torch.float32, out=None):
    """activation(x w^T + bias) + residual, [x.rows, w.rows]."""
    device = _matrix(x, "x")
    _matrix(w, "w", device)
    given = out
    out, y, e = _linear_args((x.rows,), x.rows, w, device, bias, activation, residual, dtype, out)
    check(lib.yl_mx_matmul(device, _stream(device), _ref(x._c), _ref(w._c), None if e is None else _ref(e), _ref(y)), "yl_mx_matmul")
    _written(given)
    return out


def linear(x, w: Matrix, bias=None, activation="linear", residual=None, dtype=None, out=None):
    """matmul(quantize(x), w, ...) on x [..., k], the same bits; the result has x's leading axes and, unless `dtype` says otherwise,
    its type."""
    device = _tensor(x, "x")
    _matrix(w, "w", device)
    xd = _rows_of(x, "x")
    m, given = xd.rows, out
    out, y, e = _linear_args(x.shape[:-1], m, w, device, bias, activation, residual, dtype or x.dtype, out)
    need = lib.yl_mx_linear_workspace(m, xd.k)
    ws = torch.empty(need, dtype=torch.uint8, device=_gpu(device)) if need else None
    check(lib.yl_mx_linear(device, _stream(device), _ref(xd), _ref(w._c), None if e is None else _ref(e), _ref(y),
                           ws.data_ptr() if need else None, need), "yl_mx_linear")
    _written(given)
    return out


def conv2d(x: Matrix, filters: Matrix, batch: int, h: int, w: int, size: int, stride: int = 1, pad: int = 0, bias=None,
           activation="linear", residual=None, out=None, want: str = "float"):
    """The convolution of a quantised map with quantised filters.  `want`: "float" -> FP32 [batch, filters, oh, ow]; "mx" -> the next
    layer's Matrix of batch * oh * ow rows; "both" -> the pair."""
    device = _matrix(x, "x")
    _matrix(filters, "filters", device)
    if want not in ("float", "mx", "both"):
        _fail("want is \"float\", \"mx\" or \"both\"")
    if size < 1 or stride < 1 or pad < 0 or h + 2 * pad < size or w + 2 * pad < size:
        _fail("the filter is larger than the padded map, or size, stride or pad is not one")
    n, oh, ow = filters.rows, (h + 2 * pad - size) // stride + 1, (w + 2 * pad - size) // stride + 1
    if residual is not None:
        _tensor(residual, "residual", device)
        if residual.dtype is not torch.float32 or residual.shape != (batch, n, oh, ow) or not residual.is_contiguous():
            _fail("residual is a contiguous float32 tensor of the result's shape")
    given = out
    if want == "mx":
        if out is not None:
            _fail("out is given, but want is \"mx\"")
    elif out is None:
        out = torch.empty((batch, n, oh, ow), dtype=torch.float32, device=_gpu(device))
    else:
        _tensor(out, "out", device)
        if out.dtype is not torch.float32 or out.shape != (batch, n, oh, ow) or not out.is_contiguous():
            _fail("out is a contiguous float32 tensor of the result's shape")
    q = Matrix.empty(batch * oh * ow, n, _gpu(device)) if want != "float" else None
    e = _epilogue(n, device, bias, activation, residual)
    shape = MxConv(batch, h, w, size, stride, pad)
    check(lib.yl_mx_conv2d(device, _stream(device), _ref(x._c), _ref(filters._c), _ref(shape), None if e is None else _ref(e),
                           None if out is None else out.data_ptr(), None if q is None else _ref(q._c)), "yl_mx_conv2d")
    _written(given)
    return q if want == "mx" else (out, q) if want == "both" else out
