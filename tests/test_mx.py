"""The MXFP4 entries without a GPU: the 64-bit oracle against the format's own statements, and every refusal.  (A refused call has
launched nothing and touched no pointer, so the pointers here are numbers; accepted arguments end at the missing device.)"""
import ctypes as C

import numpy as np
import pytest

import mx_oracle as o
from yolo2_light_amd._lib import Dense, MxConv, MxEpilogue, MxMatrix, lib, last_error

ARG, DEVICE = -1, -4
F32, F16, BF16 = 0, 1, 2
HAVE_GPU = lib.yl_device_count() > 0
MB = 1 << 20


# ------------------------------------------------------------------ the oracle
def test_oracle_rounds_to_the_nearest_code_with_ties_to_even():
    x = np.array([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.26, 0.74, -0.25, -0.75, 7.9, -7.9, 5.01, 4.99] + [0.0] * 16])
    code, scale = o.quantize(x)
    assert scale[0, 0] == 127                                          # floor(log2 7.9) = 2
    assert o.values(code, scale, 16)[0].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, .5, .5, 0, -1, 6, -6, 6, 4]


def test_oracle_scales():
    for top, byte in ((1.0, 125), (1.999, 125), (2.0, 126), (4.0, 127), (2.0 ** -125, 0), (2.0 ** -149, 0), (2.0 ** 127, 252), (0.0, 0), (np.inf, 255), (np.nan, 255)):
        x = np.zeros((1, 32))
        x[0, 7] = top
        assert o.quantize(x)[1][0, 0] == byte, top


def test_oracle_pack_is_unpacked():
    code = np.arange(64, dtype=np.uint8).reshape(1, 64) % 16
    assert (o.unpack(o.pack(code))[0] == code[0]).all()
    assert o.pack(code)[0, 0] == 0x10


# ------------------------------------------------------------------ refusals
def matrix(rows=4, k=64, ld=4, codes=16 * MB, scales=32 * MB):
    return MxMatrix(codes, scales, rows, k, ld)


def dense(rows=4, k=64, type=F32, data=48 * MB, batch=1, bs=0, rs=None, ks=1):
    return Dense(data, type, batch, rows, k, bs, k if rs is None else rs, ks)


def r(x):
    return None if x is None else C.byref(x)


def quantize(src, dst, device=0):
    return lib.yl_mx_quantize(device, None, r(src), r(dst))


def dequantize(src, dst, device=0):
    return lib.yl_mx_dequantize(device, None, r(src), r(dst))


X, W, Y = dict(rows=4, k=64, ld=4), dict(rows=8, k=64, ld=4, codes=64 * MB, scales=80 * MB), dict(rows=4, k=8, data=96 * MB)


def matmul(x=X, w=W, y=Y, e=None, device=0):
    x, w, y = matrix(**x) if x else None, matrix(**w) if w else None, dense(**y) if y else None
    return lib.yl_mx_matmul(device, None, r(x), r(w), r(e), r(y))


def linear(x=None, w=W, y=Y, e=None, ws=112 * MB, ws_bytes=MB, device=0):
    x = dense() if x is None else x
    return lib.yl_mx_linear(device, None, r(x), r(matrix(**w)), r(e), r(dense(**y)), ws, ws_bytes)


def refused(rc, what):
    assert rc == ARG and what in last_error(), (rc, last_error())


def accepted(rc):
    assert rc == DEVICE and "no HIP device" in last_error(), (rc, last_error())


def test_blocks():
    assert [lib.yl_mx_blocks(k) for k in (0, 1, 32, 33, 128, 129, 4096)] == [0, 4, 4, 4, 4, 8, 128]
    assert lib.yl_mx_blocks(-1) == 0 and lib.yl_mx_blocks(1 << 60) == 0


def test_linear_workspace_is_whole_rows_or_nothing():
    for rows, k in ((1, 1), (1, 4096), (300, 33), (5000, 4096)):
        need = lib.yl_mx_linear_workspace(rows, k)
        assert need in (0, rows * lib.yl_mx_blocks(k) * 17)
    assert lib.yl_mx_linear_workspace(5000, 4096) > 0
    assert lib.yl_mx_linear_workspace(0, 64) == 0 and lib.yl_mx_linear_workspace(4, 0) == 0


@pytest.mark.parametrize("change, what", [
    (dict(rows=-1), "negative"), (dict(k=-1), "negative"), (dict(k=129), "ld"), (dict(ld=(1 << 20) + 1), "ld"), (dict(codes=None), "NULL"),
    (dict(scales=None), "NULL"), (dict(codes=16 * MB + 8), "16-byte"), (dict(rows=1 << 45), "too large")])
def test_refused_matrices(change, what):
    m = {**dict(rows=4, k=64, ld=4), **change}
    refused(quantize(dense(), matrix(**m)), what)
    refused(dequantize(matrix(**m), dense()), what)
    refused(matmul(x=m), what)
    refused(matmul(w={**W, **change}), what)


@pytest.mark.parametrize("change, what", [
    (dict(type=3), "type"), (dict(type=-1), "type"), (dict(rows=-1), "negative"), (dict(k=-2), "negative"), (dict(rs=-1), "negative"), (dict(ks=-1), "negative"),
    (dict(batch=-1), "negative"), (dict(data=None), "NULL"), (dict(data=48 * MB + 2), "aligned"), (dict(data=48 * MB + 1, type=F16), "aligned"),
    (dict(rs=1 << 50), "too large"), (dict(rows=1 << 30, rs=1 << 40), "too large")])
def test_refused_tensors(change, what):
    refused(quantize(dense(**change), matrix()), what)
    refused(dequantize(matrix(), dense(**change)), what)
    refused(linear(x=dense(**change)), what)


def test_refused_shapes_and_overlaps_of_rounding():
    refused(quantize(None, matrix()), "NULL")
    refused(quantize(dense(), None), "NULL")
    refused(quantize(dense(rows=5), matrix()), "batch * rows by k")
    refused(quantize(dense(k=63), matrix()), "batch * rows by k")
    refused(quantize(dense(batch=2, rows=4), matrix(rows=4)), "batch * rows by k")
    refused(quantize(dense(data=16 * MB), matrix()), "overlaps")
    refused(quantize(dense(data=32 * MB), matrix()), "overlaps")
    refused(quantize(dense(), matrix(scales=16 * MB + 16)), "overlap")
    refused(dequantize(matrix(), dense(data=16 * MB)), "overlaps")
    refused(dequantize(matrix(), dense(rs=63)), "overlap")             # two rows of the result share a place
    refused(dequantize(matrix(), dense(rs=0)), "overlap")
    refused(dequantize(matrix(rows=8), dense(batch=2, bs=64)), "overlap")
    if not HAVE_GPU:
        accepted(quantize(dense(rs=0), matrix()))                      # a broadcast input may
        accepted(quantize(dense(rows=4, k=64, rs=1, ks=4), matrix()))
        accepted(dequantize(matrix(), dense(rs=1, ks=4)))
        accepted(quantize(dense(rows=0), matrix(rows=0)))


def test_refused_products():
    refused(matmul(x=None), "NULL")
    refused(matmul(w=None), "NULL")
    refused(matmul(y=None), "NULL")
    refused(matmul(w={**W, "k": 65}), "k differ")
    refused(matmul(y={**Y, "rows": 5}), "rows")
    refused(matmul(y={**Y, "k": 9}), "rows")
    refused(matmul(y={**Y, "batch": 2}), "batch")
    refused(matmul(y={**Y, "ks": 2, "rs": 16}), "k_stride")
    refused(matmul(y={**Y, "rs": 7}), "overlap")
    refused(matmul(y={**Y, "data": 16 * MB}), "overlaps x")
    refused(matmul(y={**Y, "data": 80 * MB}), "overlaps w")
    for e, what in ((MxEpilogue(None, 13, None, 0), "activation"), (MxEpilogue(None, -1, None, 0), "activation"), (MxEpilogue(2, 3, None, 0), "bias"),
                    (MxEpilogue(96 * MB, 3, None, 0), "bias"), (MxEpilogue(None, 3, 96 * MB + 4, 8), "residual"), (MxEpilogue(None, 3, 96 * MB, 16), "residual"),
                    (MxEpilogue(None, 3, 200 * MB, -1), "residual"), (MxEpilogue(None, 3, 200 * MB + 2, 8), "residual")):
        refused(matmul(e=e), what)
    beside = {**Y, "rs": 16}
    refused(matmul(y=beside, e=MxEpilogue(None, 3, 96 * MB + 7 * 4, 16)), "residual")          # one column in common
    refused(matmul(y=beside, e=MxEpilogue(None, 3, 96 * MB + 9 * 4, 16)), "residual")          # and around the end of a row
    if not HAVE_GPU:
        accepted(matmul(y=beside, e=MxEpilogue(None, 3, 96 * MB + 8 * 4, 16)))                 # beside it in the same rows
        accepted(matmul(y={**beside, "data": 96 * MB + 8 * 4}, e=MxEpilogue(None, 3, 96 * MB, 16)))
        accepted(matmul(e=MxEpilogue(None, 3, 96 * MB, 8)))            # the residual may be y itself
        accepted(matmul(e=MxEpilogue(128 * MB, 7, 200 * MB, 8)))
        accepted(matmul(x={**X, "rows": 0, "codes": None, "scales": None}, y={**Y, "rows": 0, "data": None}))
        accepted(matmul(x={**X, "k": 0, "ld": 0, "codes": None, "scales": None}, w={**W, "k": 0, "ld": 0}))


def test_refused_linear_layers():
    big, wide = dict(rows=5000, k=64), {**Y, "rows": 5000}
    refused(linear(x=dense(batch=2, bs=256)), "batch")
    refused(linear(x=dense(k=63)), "k differ")
    refused(linear(x=dense(data=96 * MB)), "overlaps x")
    refused(linear(x=dense(**big), y=wide, ws=None), "workspace")
    refused(linear(x=dense(**big), y=wide, ws_bytes=100), "workspace")
    refused(linear(x=dense(**big), y=wide, ws=112 * MB + 8), "aligned")
    for at in (48, 64, 80, 96):
        refused(linear(x=dense(**big), y=wide, ws=at * MB), "overlaps")
    refused(linear(x=dense(**big), y=wide, e=MxEpilogue(112 * MB, 3, None, 0)), "overlaps")
    refused(linear(x=dense(**big), y=wide, e=MxEpilogue(None, 3, 112 * MB, 8)), "overlaps")
    refused(linear(x=dense(rs=80), y={**Y, "data": 48 * MB + 63 * 4, "rs": 80}), "overlaps x")
    if not HAVE_GPU:
        accepted(linear(x=dense(rs=80), y={**Y, "data": 48 * MB + 64 * 4, "rs": 80}))          # behind x in the same rows
        accepted(linear())
        accepted(linear(x=dense(**big), y=wide))


def test_refused_inputs_that_no_workspace_holds():
    """A broadcast row has any number of rows; the workspace of 0 bytes of such an x is not the one of an x that is rounded in the product."""
    for rows, k in ((1 << 29, 1 << 23), (2 ** 31 - 300, 1 << 21), (1 << 31 >> 1, 1 << 22)):
        assert lib.yl_mx_linear_workspace(rows, k) == 0
        w, y = dict(rows=1, k=k, ld=k // 32, codes=1 << 40, scales=1 << 41), dict(rows=rows, k=1, data=1 << 42)
        for ws, ws_bytes in ((None, 0), (1 << 44, 1 << 43)):
            refused(linear(x=dense(rows=rows, k=k, rs=0), w=w, y=y, ws=ws, ws_bytes=ws_bytes), "too large")


def conv(x=None, f=None, shape=(1, 4, 4, 3, 1, 1), e=None, out=96 * MB, q=None, device=0):
    x = matrix(rows=16, k=32, ld=1) if x is None else x
    f = matrix(rows=8, k=9 * 32, ld=12, codes=64 * MB, scales=80 * MB) if f is None else f
    return lib.yl_mx_conv2d(device, None, r(x), r(f), r(MxConv(*shape)) if shape else None, r(e), out, r(q))


def test_refused_convolutions():
    refused(conv(shape=None), "NULL")
    for shape in ((1, 4, 4, 0, 1, 0), (1, 4, 4, 6, 1, 1), (1, 4, 4, 3, 0, 1), (1, 4, 4, 3, 1, -1), (1, 4, 4, 3, 1, 3), (-1, 4, 4, 3, 1, 1), (1, 0, 4, 3, 1, 1)):
        refused(conv(shape=shape), "shape")
    refused(conv(shape=(1, 4, 5, 3, 1, 1)), "batch * h * w")
    refused(conv(x=matrix(rows=16, k=33, ld=4)), "filters' k")
    refused(conv(x=matrix(rows=16, k=0, ld=0)), "no channels")
    refused(conv(x=matrix(rows=4, k=32, ld=1), shape=(1, 2, 2, 3, 1, 0)), "larger")
    refused(conv(out=96 * MB + 2), "aligned")
    for at in (16, 32, 64, 80):
        refused(conv(out=at * MB), "overlaps")
    refused(conv(e=MxEpilogue(96 * MB, 3, None, 0)), "bias")
    refused(conv(e=MxEpilogue(None, 3, 96 * MB + 4, 0)), "residual")
    q = dict(rows=16, k=8, ld=1, codes=112 * MB, scales=128 * MB)
    refused(conv(q=matrix(**{**q, "rows": 15})), "q_out")
    refused(conv(q=matrix(**{**q, "k": 9})), "q_out")
    for at in (16, 32, 64, 80, 96):
        refused(conv(q=matrix(**{**q, "codes": at * MB})), "q_out overlaps")
    if not HAVE_GPU:
        accepted(conv())
        accepted(conv(q=matrix(**q)))
        accepted(conv(out=None, q=matrix(**q)))
        accepted(conv(e=MxEpilogue(None, 3, 96 * MB, 0)))
        accepted(conv(x=matrix(rows=0, k=32, ld=1), shape=(0, 4, 4, 3, 1, 1)))


def conv_taken(batch, h, w, c, n, size, stride, pad):
    """yl_mx_conv2d takes these sizes (all pointers far from one another); None: refused."""
    rows, taps, oh, ow = batch * h * w, size * size, (h + 2 * pad - size) // stride + 1, (w + 2 * pad - size) // stride + 1
    x = matrix(rows=rows, k=c, ld=c // 32, codes=1 << 50, scales=1 << 52)
    f = matrix(rows=n, k=taps * c, ld=lib.yl_mx_blocks(taps * c), codes=1 << 54, scales=1 << 55)
    assert n * batch * oh * ow < 1 << 46
    rc = conv(x=x, f=f, shape=(batch, h, w, size, stride, pad), out=1 << 57, q=matrix(rows=batch * oh * ow, k=n, ld=(n + 31) // 32, codes=1 << 59, scales=1 << 61))
    assert rc in (ARG, DEVICE)
    return rc == DEVICE


@pytest.mark.skipif(HAVE_GPU, reason="asks the entry for sizes without memory behind them: ends at the missing device")
@pytest.mark.parametrize("batch, h, w, c, n, size, stride, pad, takes", [
    (1, 608, 608, 32, 64, 3, 2, 1, True), (64, 608, 608, 32, 64, 3, 2, 1, True), (1, 8224, 8224, 32, 64, 3, 2, 1, False),     # planes above 2^32 bytes
    (1, 4096, 4096, 32, 31, 1, 1, 0, True), (1, 4096, 4096, 32, 32, 1, 1, 0, False), (1, 4096, 4096, 32, 33, 1, 1, 0, False),  # around 2 GB
    (1, 20000, 20000, 32, 1, 3, 1, 1, False), (3, 20000, 20000, 32, 1, 3, 1, 1, False),                                        # an image's pixels above 2^28
    (8, 16000, 16000, 32, 1, 3, 1, 1, True), (9, 16000, 16000, 32, 1, 3, 1, 1, False),                                         # positions around 2^31
    (1, 1 << 20, 32, 32, 2, 3, 1, 1, True), (1, (1 << 20) + 1, 32, 32, 2, 3, 1, 1, False), (2, 13, 1 << 20, 64, 1, 3, 2, 1, True),
    (1, 60, 1 << 20, 512, 1, 3, 1, 1, False), (4, 13, 13, 1 << 14, 64, 3, 1, 1, True), (4, 5, 5, (1 << 18) + 32, 8, 1, 1, 0, False)])
def test_a_network_takes_the_sizes_that_the_operator_takes(batch, h, w, c, n, size, stride, pad, takes):
    """A layer beyond the kernel's 32-bit offsets stays in FP32; in MXFP4 its last filters once wrapped onto the first, without an error."""
    from yolo2_light_amd import Network
    import descs as D
    assert conv_taken(batch, h, w, c, n, size, stride, pad) == takes
    zeros = np.zeros(max(c, n * c * size * size), np.float32)
    first = D.conv(batch, w, h, 1, c, 1, 1, 0, D.LEAKY, zeros[:c], zeros[:c])
    net = Network.from_desc([first, D.conv(batch, w, h, c, n, size, stride, pad, D.LEAKY, zeros[:n * c * size * size], zeros[:n])], batch, w, h, 1)
    net.set_precision(3)
    assert [li["conv_mode"] for li in net.layers()] == [0, 4 if takes else 0]
    net.close()


def test_as_many_rows_as_32_bits_count():
    most = 0x7fffffff - 256
    for x, y in ((dict(rows=most + 1, k=32, ld=1), dict(rows=most + 1, k=1, data=1 << 50)), (dict(rows=1, k=32, ld=1), dict(rows=1, k=most + 1, data=1 << 50))):
        w = dict(rows=y["k"], k=32, ld=1, codes=1 << 45, scales=1 << 47)
        refused(matmul(x={**x, "codes": 1 << 40, "scales": 1 << 43}, w=w, y=y), "2^31 - 257")


FAR = dict(codes=1 << 45, scales=1 << 50)


@pytest.mark.skipif(HAVE_GPU, reason="asks the entries for sizes without memory behind them: ends at the missing device")
def test_launches_of_more_than_32_bits_of_threads():
    """Every form at the largest size it launches, and one workgroup above it."""
    def both(call, most):
        accepted(call(most))
        refused(call(most + 1), "2^32 threads")
    # rounding tensors whose k is not contiguous: 64 rows by up to 8 blocks a workgroup of 256
    for k, groups in ((2, 1), (256, 1), (257, 2), (4096, 16)):
        most = (2 ** 24 - 1) // groups * 64
        both(lambda rows: quantize(dense(rows=rows, k=k, rs=1, ks=1 << 31, data=1 << 54), matrix(rows=rows, k=k, ld=(k + 31) // 32, **FAR)), most)
        both(lambda rows: dequantize(matrix(rows=rows, k=k, ld=(k + 31) // 32, **FAR), dense(rows=rows, k=k, rs=1, ks=1 << 31, data=1 << 54)), most)
        accepted(quantize(dense(rows=1 << 31, k=k, data=1 << 54), matrix(rows=1 << 31, k=k, ld=(k + 31) // 32, **FAR)))         # contiguous k: a loop
    w = lambda rows: dict(rows=rows, k=32, ld=1, **FAR)  # noqa: E731
    y = lambda m, n: dict(rows=m, k=n, data=1 << 53)  # noqa: E731
    for m, most in ((1, (2 ** 23 - 1) * 16), (16, (2 ** 23 - 1) * 16), (17, (2 ** 23 - 1) * 32), (32, (2 ** 23 - 1) * 32)):      # 512 threads a workgroup
        both(lambda n: matmul(x=dict(rows=m, k=32, ld=1), w=w(n), y=y(m, n)), most)
        both(lambda n: linear(x=dense(rows=m, k=32), w=w(n), y=y(m, n)), most)
    accepted(matmul(x=dict(rows=33, k=32, ld=1), w=w(2 ** 31 - 257), y=y(33, 2 ** 31 - 257)))
    rare = MxEpilogue(None, 0, None, 0)                           # 64 x 64 tiles alone
    both(lambda n: matmul(x=dict(rows=64, k=32, ld=1), w=w(n), y=y(64, n), e=rare), (2 ** 24 - 1) * 64)
    most = (2 ** 24 - 1) * 64                                     # x in columns of a workspace
    both(lambda m: linear(x=dense(rows=m, k=32, rs=1, ks=1 << 31, data=1 << 40), w=dict(rows=1, k=32, ld=1), y=y(m, 1), ws=1 << 57, ws_bytes=1 << 40), most)
    most = (2 ** 24 - 1) * 64 // 2 ** 12                          # images of 64 x 64
    x = lambda b: matrix(rows=b * 4096, k=32, ld=1, **FAR)  # noqa: E731
    f = matrix(rows=8, k=32, ld=1)
    both(lambda b: conv(x=x(b), f=f, shape=(b, 64, 64, 1, 1, 0), e=rare, out=1 << 57), most)


def test_no_such_device():
    for device in (-1, 4096):
        rc = quantize(dense(), matrix(), device=device)
        assert rc == (ARG if HAVE_GPU else DEVICE), last_error()


def test_python_refuses_what_is_not_on_a_gpu():
    torch = pytest.importorskip("torch")
    from yolo2_light_amd import YoloHipError, mx
    x = torch.zeros(4, 64)
    for call in (lambda: mx.quantize(x), lambda: mx.quantize_nchw(x), lambda: mx.quantize_filters(x), lambda: mx.linear(x, None),
                 lambda: mx.Matrix(x, x, 64), lambda: mx.matmul(x, x), lambda: mx.conv2d(x, x, 1, 2, 2, 1), lambda: mx.dequantize(x)):
        with pytest.raises(YoloHipError):
            call()


def test_python_counts_the_rows_of_empty_tensors():
    torch = pytest.importorskip("torch")
    from yolo2_light_amd import mx
    for shape in ((2, 3, 0), (2, 0, 3), (0, 3, 5), (3, 0), (0, 3), (2, 3, 4, 0), (2, 3, 4)):
        d = mx._rows_of(torch.zeros(shape), "x")
        assert (d.rows, d.k) == (int(np.prod(shape[:-1])), shape[-1]), shape


def test_python_views_of_a_matrix_from_two_threads():
    """codes and scales of Matrix.empty are made when they are asked for: a thread that asks while another is between the two finds them right."""
    torch = pytest.importorskip("torch")
    from yolo2_light_amd import mx

    class Between(mx.Matrix):                                      # reads scales the moment the first of the two is set
        __slots__ = ("seen",)

        def __setattr__(self, name, value):
            first = name in ("_codes", "_scales") and value is not None and not hasattr(self, "seen")
            super().__setattr__(name, value)
            if first and hasattr(self, "_c"):
                object.__setattr__(self, "seen", None)
                object.__setattr__(self, "seen", (self.codes, self.scales))

    for ask in ("codes", "scales"):
        m = Between.empty(3, 200, "cpu")
        got = getattr(m, ask)
        for codes, scales in ((m.codes, m.scales), m.seen):
            assert codes.shape == (3, 128) and scales.shape == (3, 8)
            assert codes.data_ptr() == m._c.codes and scales.data_ptr() == m._c.scales
        assert got.data_ptr() == getattr(m._c, ask) and m.device == torch.device("cpu")
