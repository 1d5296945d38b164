"""The MXFP4 operators on the GPU against their definition in 64 bits (mx_oracle.py), at the sizes, strides, types and values where
they can go wrong; tolerances are mx_oracle.product_tolerance's, everything that is only rounded is compared bit for bit."""
import numpy as np
import pytest

import mx_oracle as o

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


@pytest.fixture(scope="module")
def mx():
    from yolo2_light_amd import mx
    return mx


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(*shape, seed=0, dtype="float32", spread=1.0):
    """Normal values whose columns differ in magnitude, on the CPU."""
    g = gen(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(TYPES[dtype])


def f64(t):
    return t.detach().cpu().double().numpy()


def check_matrix(q, x64):
    """q holds exactly the oracle's rounding of x64, and zero codes behind its end."""
    code, scale = o.quantize(x64)
    kb = scale.shape[1]
    got = o.unpack(q.codes.cpu().numpy())[:, :kb * 32]
    assert (q.scales.cpu().numpy()[:, :kb] == scale).all()
    bad = got != code
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], code[bad][:4])


def make(mx, rows, k, seed, spread=1.0, ld=None):
    """A matrix from the oracle's codes (not the kernel's), and its values."""
    x = f64(rand(rows, k, seed=seed, spread=spread))
    code, scale = o.quantize(x)
    ld = ld or max(4, (o.blocks(k) + 3) // 4 * 4)
    s = np.full((rows, ld), 77, np.uint8)                  # blocks behind the last one hold anything
    s[:, :scale.shape[1]] = scale
    c = o.pack(code, ld)
    c[:, scale.shape[1] * 16:] = 0x5A
    return mx.Matrix(torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), k), o.values(code, scale, k)


def close(y, want, tol):
    y = f64(y)
    assert y.shape == want.shape
    off = np.abs(y - want) - tol
    assert np.isfinite(y).all() and (off <= 0).all(), "worst %.3g over, at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))


# ------------------------------------------------------------------ rounding
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, k", [(1, 1), (1, 31), (1, 32), (1, 33), (3, 64), (2, 127), (5, 128), (1, 4096), (257, 160), (33, 1005), (1000, 40), (7, 2049)])
def test_rows(mx, rows, k, dtype):
    x = rand(rows, k, seed=rows + k, dtype=dtype, spread=1.5).cuda()
    q = mx.quantize(x)
    check_matrix(q, f64(x))
    v = mx.dequantize(q, TYPES[dtype])
    assert (f64(v) == o.rounded(f64(x))).all()            # E2M1 times a power of two that FP16's own values gave: all exact


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 32, 3, 5), (2, 64, 8, 8), (3, 33, 7, 9), (1, 255, 13, 13), (2, 3, 17, 5), (1, 96, 1, 70), (1, 257, 70, 1), (4, 128, 19, 19), (1, 1024, 5, 5)])
def test_maps(mx, shape, dtype):
    b, c, h, w = shape
    x = rand(b, h, w, c, seed=c + h, dtype=dtype).permute(0, 3, 1, 2).contiguous().cuda()
    q = mx.quantize_nchw(x)
    rows = f64(x).transpose(0, 2, 3, 1).reshape(-1, c)
    check_matrix(q, rows)
    v = mx.dequantize_nchw(q, b, h, w, TYPES[dtype])
    assert (f64(v).transpose(0, 2, 3, 1).reshape(-1, c) == o.rounded(rows)).all()


def test_strides(mx):
    base = rand(40, 300, seed=1).cuda()
    for x in (base[:, :257], base[:, 3:260], base[::2, 1:200], base.t()[:257], base.t()[5:260:3], base[:, ::3], base[3], base[3:4, :7].expand(5, 7), base[:, :0], base[:0]):
        q = mx.quantize(x)
        x2 = f64(x)[None] if x.dim() == 1 else f64(x)
        assert q.rows == x2.shape[0]
        if x2.size:
            check_matrix(q, x2)
        v = mx.dequantize(q)
        assert v.shape == x2.shape and (f64(v) == (o.rounded(x2) if x2.size else x2)).all()
    x = rand(2, 3, 5, 96, seed=2, dtype="bfloat16").cuda()
    check_matrix(mx.quantize(x), f64(x).reshape(-1, 96))
    m = rand(2, 9, 11, 48, seed=3).permute(0, 3, 1, 2).cuda()                       # channels last
    check_matrix(mx.quantize_nchw(m), f64(m).transpose(0, 2, 3, 1).reshape(-1, 48))
    check_matrix(mx.quantize_nchw(m[:, 5:40]), f64(m)[:, 5:40].transpose(0, 2, 3, 1).reshape(-1, 35))
    q = mx.quantize(x)
    out = torch.full((30, 200), 7.0, device="cuda")
    mx.dequantize(q, out=out[:, 100:196])
    assert (f64(out)[:, 100:196] == o.rounded(f64(x).reshape(-1, 96))).all() and (out[:, :100] == 7).all() and (out[:, 196:] == 7).all()
    out = torch.full((96, 33), 7.0, device="cuda")
    mx.dequantize(q, out=out.t()[:30])
    assert (f64(out)[:, :30].T == o.rounded(f64(x).reshape(-1, 96))).all() and (out[:, 30:] == 7).all()


def test_every_tie_and_every_scale(mx):
    """All borders between codes, one FP32 step to either side of them, under every scale that FP32 has."""
    grid = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0]
    rows = []
    for e in range(-149, 126):
        s = np.float64(2.0) ** e
        for step in (-1, 0, 1):
            with np.errstate(over="ignore", under="ignore"):
                v = np.array(grid, np.float64).astype(np.float32) * np.float32(s)
                v = np.nextafter(v, np.float32(np.inf) * np.float32(step)) if step else v
                top = np.float32(min(7.5 * s, 3.4e38))
            rows.append(np.concatenate([v, -v, [top, 0.0, -0.0, top / 2]]).astype(np.float32))
    x = torch.from_numpy(np.stack(rows)).cuda()
    check_matrix(mx.quantize(x), f64(x))
    assert (f64(mx.dequantize(mx.quantize(x))) == o.rounded(f64(x))).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_blocks_that_are_not_numbers(mx, dtype):
    x = rand(6, 100, seed=5, dtype=dtype)
    x[0, 3], x[1, 40], x[2, 99], x[3, 64], x[4, 31] = float("inf"), float("-inf"), float("nan"), float("nan"), float("inf")
    x[4, 30] = float("nan")
    x = x.cuda()
    q = mx.quantize(x)
    check_matrix(q, f64(x))
    v, want = f64(mx.dequantize(q, TYPES[dtype])), o.rounded(f64(x))
    assert (np.isnan(v) == np.isnan(want)).all() and (v[~np.isnan(v)] == want[~np.isnan(v)]).all()
    w, wv = make(mx, 40, 100, 6)
    for y in (mx.matmul(q, w), mx.linear(x, w, dtype=torch.float32), mx.linear(x.repeat(100, 1), w, dtype=torch.float32)[:6]):
        y = f64(y)
        assert np.isnan(y[:5]).all() and np.isfinite(y[5]).all()


def test_dequantize_codes_that_no_rounding_makes(mx):
    code = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scale = np.arange(256, dtype=np.uint8).reshape(256, 1)
    m = mx.Matrix(torch.from_numpy(o.pack(code, 4)).cuda(), torch.from_numpy(np.repeat(scale, 4, 1)).cuda(), 32)
    want = o.values(code, scale, 32)
    for name, t in TYPES.items():
        with np.errstate(over="ignore"):
            w = torch.from_numpy(want.astype(np.float32)).to(t) if name != "float16" else torch.from_numpy(want.astype(np.float16))
        v = mx.dequantize(m, t).cpu()
        ok = (v == w) | (v.isnan() & w.isnan())
        assert ok.all(), (name, v[~ok][:4], w[~ok][:4])


def test_rounding_leaves_what_it_does_not_own(mx):
    x = rand(5, 70, seed=8).cuda()
    c = torch.full((7, 8 * 16), 0xAB, dtype=torch.uint8, device="cuda")
    s = torch.full((7, 8), 0xCD, dtype=torch.uint8, device="cuda")
    mx.quantize(x, out=mx.Matrix(c[:5], s[:5], 70))
    check_matrix(mx.Matrix(c[:5], s[:5], 70), f64(x))
    assert (c[:5, 3 * 16:] == 0xAB).all() and (c[5:] == 0xAB).all() and (s[:5, 3:] == 0xCD).all() and (s[5:] == 0xCD).all()


# ------------------------------------------------------------------ products
SIZES = [(1, 1, 1), (1, 16, 32), (1, 17, 33), (2, 64, 64), (3, 33, 96), (1, 512, 1024), (1, 100, 4097), (5, 257, 1000), (8, 64, 2048), (9, 96, 513),
         (16, 128, 256), (17, 1000, 300), (31, 48, 6000), (32, 256, 512), (33, 130, 65), (40, 520, 1000), (64, 64, 64), (65, 63, 129), (100, 1, 640), (127, 257, 31),
         (128, 128, 128), (129, 127, 2000), (200, 300, 400), (256, 256, 256), (257, 255, 257), (300, 1100, 96), (512, 40, 1111), (1000, 72, 288), (515, 517, 519)]


@pytest.mark.parametrize("m, n, k", SIZES)
def test_products(mx, m, n, k):
    x, xv = make(mx, m, k, m + n)
    w, wv = make(mx, n, k, n + k)
    for dtype in TYPES:
        want, tol = o.product_tolerance(xv, wv, None, "linear", None, dtype) if dtype != "float16" else o.product_tolerance(xv / 64, wv / 64, None, "linear", None, dtype)
        if dtype == "float16":                                    # keep FP16 in range: x and w 64 times smaller
            x16, w16 = (mx.Matrix(q.codes, q.scales - 6, k) for q in (x, w))
            close(mx.matmul(x16, w16, dtype=TYPES[dtype]), want, tol)
        else:
            close(mx.matmul(x, w, dtype=TYPES[dtype]), want, tol)


def gpu_values(mx, q):
    """The values of a matrix of finite blocks, float64 on the GPU (dequantize is compared with the oracle above)."""
    return mx.dequantize(q).double()


@pytest.mark.parametrize("m, n, k", [(1024, 1024, 96), (2000, 2050, 300), (4100, 4099, 130), (4096, 4096, 512), (257, 33_000, 64), (20_000, 900, 33), (1500, 260, 2100)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_products_that_fill_the_chip(mx, m, n, k, dtype):
    """The same tolerance as mx_oracle.product_tolerance, computed on the GPU."""
    x, w = mx.quantize(rand(m, k, seed=m, spread=0.5).cuda()), mx.quantize(rand(n, k, seed=n, spread=0.5).cuda())
    res, b = rand(m, n, seed=3, dtype=dtype).cuda(), rand(n, seed=4).cuda()
    y = mx.matmul(x, w, bias=b, activation="leaky", residual=res, dtype=TYPES[dtype]).double()
    xv, wv = gpu_values(mx, x), gpu_values(mx, w)
    v = xv @ wv.t() + b.double()
    want = torch.where(v > 0, v, 0.1 * v) + res.double()
    tol = ((o.blocks(k) + 1) // 2 + 16) * 2.0 ** -23 * (xv.abs() @ wv.abs().t())
    tol = tol + 2.0 ** -22 * (v.abs() + want.abs() + tol) + 2.0 ** -24
    tol = tol + o.HALF_STEP[dtype][0] * (want.abs() + tol)
    assert ((y - want).abs() <= tol).all(), ((y - want).abs() - tol).max()


def whole_product_tolerance(x, w, bias, act, res, dtype, steps_of):
    """mx_oracle.product_tolerance in FP64 on the GPU: activation(x w^T + bias) + res and how far a result may be from it."""
    v = x @ w.t()
    tol = ((o.blocks(steps_of) + 1) // 2 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().t())
    v = v + bias.double()
    tol = tol + 2.0 ** -24 * (v.abs() + tol)
    y = {"linear": lambda: v, "leaky": lambda: torch.where(v > 0, v, 0.1 * v), "relu": lambda: v.clamp(min=0), "logistic": lambda: torch.sigmoid(v)}[act]()
    tol = 1.1 * tol + (2.0 ** -23 * y.abs() + 2.0 ** -24 if act != "linear" else 0)
    if res is not None:
        y = y + res.double()
        tol = tol + 2.0 ** -24 * (y.abs() + tol)
    half, least = o.HALF_STEP[dtype]
    return y, tol + half * (y.abs() + tol) + least


def random_matrix(mx, rows, k, seed, ld=None):
    """Rows of every block different: random codes and scales over 2^5, what lies behind k's last block anything."""
    g, kb = torch.Generator(device="cuda").manual_seed(seed), (k + 31) // 32
    ld = ld or (kb + 3) // 4 * 4
    codes = torch.randint(0, 256, (rows, 16 * ld), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(120, 125, (rows, ld), dtype=torch.uint8, device="cuda", generator=g)
    if k % 32:                                                    # the codes behind k in the last block are zero
        last = codes[:, 16 * (kb - 1):16 * kb]
        last[:, (k % 32 + 1) // 2:] = 0
        if k % 2:
            last[:, k % 32 // 2] &= 15
    scales[:, kb:] = 255
    return mx.Matrix(codes, scales, k)


# (form, m, n, k, ld of x, ld of w): 256 x 256, 128 x 128, 64 x 128 and 64 x 64 tiles with scales by words and by bytes; k ends inside a panel of 256,
# inside a word of four blocks and inside a block; rows and columns end inside a tile, in one and in both halves of it
FORMS = [("256", 4100, 4099, 2100, 68, 68), ("256", 4096, 4352, 2048, 64, 64), ("256", 3841, 4330, 2177, 72, 72), ("256 bytes", 4100, 4099, 2100, 67, 69), ("256 bytes", 4000, 4200, 2321, 73, 76),
         ("128", 3001, 2900, 1025, 36, 36), ("128 bytes", 3001, 2900, 1025, 33, 35), ("128, k >= 2048", 2000, 2100, 2100, 68, 68), ("128 bytes, k >= 2048", 2000, 2100, 2100, 66, 67),
         ("64 x 128", 1000, 2500, 700, 24, 24), ("64 x 128 bytes", 1000, 2500, 700, 22, 25), ("64", 650, 700, 300, 12, 12), ("64 bytes", 650, 700, 300, 10, 11)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("form, m, n, k, x_ld, w_ld", FORMS, ids=["-".join(str(v) for v in f) for f in FORMS])
def test_every_tile_with_the_whole_epilogue(mx, form, m, n, k, x_ld, w_ld, dtype):
    """Every element of products that fill the chip: bias, activation, a residual and a result in rows of other lengths."""
    x, w = random_matrix(mx, m, k, m, x_ld), random_matrix(mx, n, k, n + 1, w_ld)
    bias = rand(n, seed=4).cuda()
    res = rand(m, n + 5, seed=3, dtype=dtype).cuda()[:, 2:n + 2]
    act = {"float32": "leaky", "float16": "relu", "bfloat16": "leaky"}[dtype]
    whole = torch.full((m + 2, n + 9), 3.0, dtype=TYPES[dtype], device="cuda")
    mx.matmul(x, w, bias=bias, activation=act, residual=res, out=whole[1:m + 1, 4:n + 4])
    want, tol = whole_product_tolerance(gpu_values(mx, x), gpu_values(mx, w), bias, act, res, dtype, k)
    off = (whole[1:m + 1, 4:n + 4].double() - want).abs() - tol
    assert (off <= 0).all(), (off.max(), (off > 0).nonzero()[:4])
    assert (whole[0] == 3).all() and (whole[m + 1] == 3).all() and (whole[:, :4] == 3).all() and (whole[:, n + 4:] == 3).all()
    if dtype == "float32":                                        # the same sums without anything behind them
        y = mx.matmul(x, w)
        want, tol = whole_product_tolerance(gpu_values(mx, x), gpu_values(mx, w), torch.zeros_like(bias), "linear", None, dtype, k)
        assert ((y.double() - want).abs() <= tol).all()
        y = mx.matmul(x, w, bias=bias, activation="logistic", residual=res)        # 64 x 64 tiles, single values
        want, tol = whole_product_tolerance(gpu_values(mx, x), gpu_values(mx, w), bias, "logistic", res, dtype, k)
        assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m", [1, 20, 40, 300])
def test_stair(mx, m):
    """The one activation with jumps: sums, bias and result are small multiples of 1/4, exact in FP32 and on whole numbers often."""
    n, k = 70, 96
    g = gen(m)
    x, w = torch.randint(-3, 4, (m, k), generator=g).float() / 2, torch.randint(-1, 2, (n, k), generator=g).float() / 2
    x[:, ::32], w[:, ::32] = 6.0, 4.0                             # scales of 1: every block holds the values as they are
    bias = torch.randint(-20, 21, (n,), generator=g).float() / 4 - 60.0
    xq, wq = mx.quantize(x.cuda()), mx.quantize(w.cuda())
    assert (f64(mx.dequantize(xq)) == f64(x)).all() and (f64(mx.dequantize(wq)) == f64(w)).all()
    v = f64(x) @ f64(w).T + f64(bias)
    whole = np.floor(v)                                           # stair_activate: even steps are flat, odd ones rise
    want = np.where(whole % 2 == 0, np.floor(v / 2), v - whole + np.floor(v / 2))
    assert (v == whole).sum() > 10 and (v < 0).any() and (v > 0).any()
    got = mx.matmul(xq, wq, bias=bias.cuda(), activation="stair")
    assert (f64(got) == want).all()


@pytest.mark.parametrize("m", [1, 16, 20, 40, 200])
def test_activations_of_infinities(mx, m):
    """RELU is x * (x > 0), here as in every path of this library: NaN of -Inf.  The others as their formulas say."""
    n, k = 48, 64
    big = mx.Matrix(torch.full((m, 64), 0x77, dtype=torch.uint8, device="cuda"), torch.full((m, 4), 254, dtype=torch.uint8, device="cuda"), k)
    wc = torch.full((n, 64), 0x77, dtype=torch.uint8, device="cuda")
    wc[n // 2:] = 0xFF                                            # -6: the sums of the upper half are -Inf
    w = mx.Matrix(wc, torch.full((n, 4), 254, dtype=torch.uint8, device="cuda"), k)
    inf, nan = float("inf"), float("nan")
    for act, up, down in (("linear", inf, -inf), ("leaky", inf, -inf), ("relu", inf, nan), ("logistic", 1.0, 0.0), ("relie", inf, -inf), ("hardtan", 1.0, -1.0), ("lhtan", inf, -inf)):
        want = torch.tensor([up] * (n // 2) + [down] * (n - n // 2), device="cuda").expand(m, n)
        assert torch.equal(mx.matmul(big, w, activation=act).nan_to_num(12.5), want.nan_to_num(12.5)), act


@pytest.mark.parametrize("m, n, k", [(1, 100, 200), (7, 33, 64), (40, 129, 300), (130, 260, 96), (300, 300, 300)])
@pytest.mark.parametrize("act", ["leaky", "relu", "logistic", "tanh", "elu", "relie", "ramp", "hardtan", "lhtan", "plse", "loggy"])
def test_epilogues(mx, m, n, k, act):
    x, xv = make(mx, m, k, 1, spread=0.3)
    w, wv = make(mx, n, k, 2, spread=0.3)
    w, wv = mx.Matrix(w.codes, w.scales - 4, k), wv / 16
    bias, res = rand(n, seed=3, spread=0.2), rand(m, n, seed=4, dtype="bfloat16")
    want, tol = o.product_tolerance(xv, wv, f64(bias), act, f64(res), "bfloat16")
    close(mx.matmul(x, w, bias=bias.cuda(), activation=act, residual=res.cuda(), dtype=torch.bfloat16), want, tol)
    want, tol = o.product_tolerance(xv, wv, f64(bias), act, None, "float32")
    close(mx.matmul(x, w, bias=bias.cuda(), activation=act), want, tol)


@pytest.mark.parametrize("m, n, k", [(3, 70, 100), (40, 140, 260), (300, 260, 300)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_results_and_residuals(mx, m, n, k, dtype):
    x, xv = make(mx, m, k, 5, spread=0.3)
    w, wv = make(mx, n, k, 6, spread=0.3)
    res = rand(m, n + 5, seed=7, dtype=dtype)
    want, tol = o.product_tolerance(xv, wv, None, "linear", f64(res)[:, 2:n + 2], dtype)
    out = torch.full((m + 1, n + 9), 3.0, dtype=TYPES[dtype], device="cuda")
    y = mx.matmul(x, w, residual=res.cuda()[:, 2:n + 2], out=out[:m, 4:n + 4])
    assert y.data_ptr() == out[:, 4:].data_ptr()
    close(out[:m, 4:n + 4], want, tol)
    assert (out[:m, :4] == 3).all() and (out[:m, n + 4:] == 3).all() and (out[m:] == 3).all()
    out[:m, 4:n + 4] = res.cuda()[:, 2:n + 2]                     # the residual is the result's own place
    mx.matmul(x, w, residual=out[:m, 4:n + 4], out=out[:m, 4:n + 4])
    close(out[:m, 4:n + 4], want, tol)
    assert (out[:m, :4] == 3).all() and (out[:m, n + 4:] == 3).all()
    one = rand(1, n, seed=9, dtype=dtype).cuda().expand(m, n)     # one row for all
    want, tol = o.product_tolerance(xv, wv, None, "linear", f64(one), dtype)
    close(mx.matmul(x, w, residual=one, dtype=TYPES[dtype]), want, tol)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_operands_and_results_side_by_side(mx, m):
    """x, the residual and the result as columns of one buffer."""
    n, k = 72, 96
    w, _ = make(mx, n, k, 1)
    x, res = rand(m, k, seed=2), rand(m, n, seed=3)
    want = mx.linear(x.cuda(), w, residual=res.cuda())
    buf = torch.full((m, k + 2 * n + 8), 5.0, device="cuda")
    buf[:, :k], buf[:, k:k + n] = x.cuda(), res.cuda()
    mx.linear(buf[:, :k], w, residual=buf[:, k:k + n], out=buf[:, k + n:k + 2 * n])
    assert torch.equal(buf[:, k + n:k + 2 * n], want) and (buf[:, k + 2 * n:] == 5).all()
    assert torch.equal(buf[:, :k].cpu(), x) and torch.equal(buf[:, k:k + n].cpu(), res)


@pytest.mark.parametrize("ld", [3, 5, 6, 7, 9])
@pytest.mark.parametrize("m", [1, 20, 150])
def test_rows_of_any_stride(mx, ld, m):
    k = 32 * ld - 3
    x, xv = make(mx, m, k, 1, ld=ld)
    w, wv = make(mx, 150, k, 2, ld=ld + 2)
    want, tol = o.product_tolerance(xv, wv, None, "linear", None, "float32")
    close(mx.matmul(x, w), want, tol)
    s = torch.empty(m * ld + 3, dtype=torch.uint8, device="cuda")[3:].view(m, ld)       # scales at an odd address
    s.copy_(x.scales)
    close(mx.matmul(mx.Matrix(x.codes, s, k), w), want, tol)


def test_empty_products(mx):
    w, wv = make(mx, 40, 64, 1)
    assert mx.linear(torch.empty(0, 64, device="cuda"), w).shape == (0, 40)
    assert mx.matmul(mx.Matrix.empty(0, 64, "cuda"), w).shape == (0, 40)
    assert mx.matmul(mx.Matrix.empty(5, 64, "cuda"), mx.Matrix.empty(0, 64, "cuda")).shape == (5, 0)
    b = rand(40, seed=1).cuda()
    y = mx.linear(torch.empty(3, 0, device="cuda"), mx.Matrix.empty(40, 0, "cuda"), bias=b, activation="relu")
    assert (y == b.clamp(min=0).expand(3, 40)).all()              # nothing to sum
    y = mx.matmul(mx.Matrix.empty(300, 0, "cuda"), mx.Matrix.empty(40, 0, "cuda"), bias=b)
    assert (y == b.expand(300, 40)).all()


@pytest.mark.parametrize("lead", [(2, 3), (1, 2, 2), (7,), ()])
def test_nothing_to_sum_under_any_leading_axes(mx, lead):
    """x [..., 0]: every row of the result is activation(bias) + residual."""
    m, n = int(np.prod(lead)), 40
    b, res = rand(n, seed=1).cuda(), rand(m, n, seed=2).reshape(*lead, n).cuda()
    w = mx.Matrix.empty(n, 0, "cuda")
    out = torch.full((*lead, n), float("nan"), device="cuda")
    y = mx.linear(torch.empty(*lead, 0, device="cuda"), w, bias=b, activation="relu", residual=res, out=out)
    assert torch.equal(y, b.clamp(min=0) + res)
    q = mx.quantize(torch.empty(*lead, 0, device="cuda"))
    assert (q.rows, q.k) == (m, 0) and mx.dequantize(q).shape == (m, 0)
    assert mx.linear(torch.ones(*lead, 64, device="cuda"), mx.Matrix.empty(0, 64, "cuda")).shape == (*lead, 0)


def test_no_filters_or_no_channels(mx):
    for shape in ((0, 64, 3, 3), (5, 0, 3, 3), (0, 0, 1, 1)):
        f = mx.quantize_filters(torch.zeros(shape, device="cuda"))
        assert (f.rows, f.k) == (shape[0], shape[2] * shape[3] * ((shape[1] + 31) // 32 * 32))


def test_extreme_scales(mx):
    """2^100 against 2^-100, and sums that leave FP32."""
    x, xv = make(mx, 70, 256, 1, spread=0.2)
    w, wv = make(mx, 70, 256, 2, spread=0.2)
    want, tol = o.product_tolerance(xv, wv, None, "linear", None, "float32")
    close(mx.matmul(mx.Matrix(x.codes, x.scales + 100, 256), mx.Matrix(w.codes, w.scales - 100, 256)), want, tol)
    big = mx.Matrix(torch.full_like(x.codes, 0x77), torch.full_like(x.scales, 254), 256)
    assert torch.isposinf(mx.matmul(big, big)).all()
    assert torch.isposinf(mx.matmul(mx.Matrix(big.codes[:1], big.scales[:1], 256), big)).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m, n, k", [s for s in SIZES if s[0] * s[1] * s[2] < 40_000_000] + [(1, 4096, 4096), (4, 2050, 4100), (48, 512, 2048), (600, 130, 200),
                         (1, 33, 76_800), (1, 33, 76_801), (2, 40, 16_384), (2, 40, 16_385), (16, 40, 2048), (16, 40, 2049), (17, 8200, 96), (5, 8200, 100)])      # borders of the forms
def test_linear_is_matmul_of_the_rounded_rows(mx, m, n, k, dtype):
    x = rand(m, k + 3, seed=m + k, dtype=dtype).cuda()[:, 1:k + 1]
    w, _ = make(mx, n, k, n)
    b, res = rand(n, seed=1).cuda(), rand(m, n, seed=2, dtype=dtype).cuda()
    y = mx.linear(x, w, bias=b, activation="leaky", residual=res)
    z = mx.matmul(mx.quantize(x), w, bias=b, activation="leaky", residual=res, dtype=TYPES[dtype])
    assert y.dtype == TYPES[dtype] and torch.equal(y, z)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 70, 300])
def test_linear(mx, m):
    n, k = 200, 520
    x, b = rand(m, k, seed=m), rand(n, seed=1)
    w, wv = make(mx, n, k, 3)
    want, tol = o.product_tolerance(o.rounded(f64(x)), wv, f64(b), "relu", None, "float32")
    close(mx.linear(x.cuda(), w, bias=b.cuda(), activation="relu"), want, tol)
    assert torch.equal(mx.linear(x.t().contiguous().t().cuda(), w, bias=b.cuda(), activation="relu"),            # columns in memory
                       mx.linear(x.cuda(), w, bias=b.cuda(), activation="relu"))


def test_a_row_does_not_depend_on_the_rows_beside_it(mx):
    """A token of a padded batch is what it is: rows of a call are independent, also of a row of NaN."""
    w, _ = make(mx, 300, 512, 1)
    for m in (2, 16, 40, 300):
        x = rand(m, 512, seed=m).cuda()
        y = mx.linear(x, w)
        x2 = x.clone()
        x2[m // 2:] = float("nan")
        y2 = mx.linear(x2, w)
        assert torch.equal(y[:m // 2], y2[:m // 2]) and y2[m // 2:].isnan().all()
        assert torch.equal(y, mx.linear(x, w))                    # and the same again


# ------------------------------------------------------------------ convolutions
CONVS = [(1, 1, 1, 1, 1, 1, 1, 0), (1, 32, 8, 4, 4, 3, 1, 1), (2, 32, 32, 7, 5, 3, 1, 1), (1, 33, 17, 6, 6, 3, 2, 1), (2, 64, 40, 13, 13, 1, 1, 0), (1, 96, 255, 13, 13, 1, 1, 0),
         (3, 128, 64, 9, 9, 3, 1, 1), (1, 160, 33, 8, 8, 5, 1, 2), (2, 256, 100, 7, 7, 3, 2, 1), (1, 512, 128, 10, 10, 3, 1, 1), (2, 40, 128, 16, 16, 3, 1, 1), (1, 64, 64, 1, 1, 3, 1, 1),
         (1, 64, 64, 1, 40, 3, 1, 1), (2, 48, 96, 12, 9, 2, 2, 0), (1, 128, 256, 20, 20, 3, 3, 0), (5, 32, 64, 31, 17, 3, 2, 1), (1, 256, 512, 12, 12, 1, 2, 0), (2, 64, 32, 26, 26, 3, 1, 2)]


def conv_case(mx, batch, c, n, h, w, size, seed=0):
    x = rand(batch, h, w, c, seed=seed, spread=0.4).permute(0, 3, 1, 2).contiguous()
    f = rand(n, size, size, c, seed=seed + 1, spread=0.3).permute(0, 3, 1, 2).contiguous() / (c * size * size) ** 0.5
    xv = o.rounded(f64(x).transpose(0, 2, 3, 1).reshape(-1, c))
    rows = o.filter_rows(f64(f))
    fv = o.rounded(rows).reshape(n, size * size, -1)[:, :, :c].reshape(n, -1)
    return x.cuda(), f.cuda(), xv, fv, rows


@pytest.mark.parametrize("batch, c, n, h, w, size, stride, pad", CONVS)
def test_convolutions(mx, batch, c, n, h, w, size, stride, pad):
    x, f, xv, fv, rows = conv_case(mx, batch, c, n, h, w, size, seed=c + n)
    win, oh, ow = o.windows(xv, batch, h, w, size, stride, pad)
    bias, res = rand(n, seed=1, spread=0.2), rand(batch, n, oh, ow, seed=2)
    fq, q = mx.quantize_filters(f), mx.quantize_nchw(x)
    check_matrix(fq, rows)
    lay = lambda a: a.reshape(batch, oh, ow, n).transpose(0, 3, 1, 2)  # noqa: E731
    want, tol = o.product_tolerance(win, fv, f64(bias), "leaky", f64(res).transpose(0, 2, 3, 1).reshape(-1, n), "float32")
    y, yq = mx.conv2d(q, fq, batch, h, w, size, stride, pad, bias=bias.cuda(), activation="leaky", residual=res.cuda(), want="both")
    close(y, lay(want), lay(tol))
    again = mx.quantize_nchw(y)                                   # the side output: the result's own rounding
    kb = o.blocks(n)
    assert torch.equal(yq.codes[:, :kb * 16], again.codes[:, :kb * 16]) and torch.equal(yq.scales[:, :kb], again.scales[:, :kb])
    only = mx.conv2d(q, fq, batch, h, w, size, stride, pad, bias=bias.cuda(), activation="leaky", residual=res.cuda(), want="mx")
    assert torch.equal(only.codes[:, :kb * 16], yq.codes[:, :kb * 16]) and torch.equal(only.scales[:, :kb], yq.scales[:, :kb])
    want, tol = o.product_tolerance(win, fv, None, "linear", None, "float32")
    close(mx.conv2d(q, fq, batch, h, w, size, stride, pad), lay(want), lay(tol))
    r2 = res.cuda()
    z = mx.conv2d(q, fq, batch, h, w, size, stride, pad, bias=bias.cuda(), activation="leaky", residual=r2, out=r2)      # in place
    assert torch.equal(z, y)


@pytest.mark.parametrize("act", ["relu", "logistic", "tanh", "elu", "relie", "ramp", "hardtan", "lhtan", "plse", "loggy"])
@pytest.mark.parametrize("batch, c, n, h, w, size, stride, pad", [(2, 64, 70, 9, 7, 3, 1, 1), (1, 33, 17, 6, 6, 3, 2, 1), (3, 128, 130, 13, 13, 1, 1, 0)])
def test_convolutions_with_every_activation(mx, batch, c, n, h, w, size, stride, pad, act):
    """... and their MXFP4 output, where filters end inside a block: what is behind them is zero, whatever the activation makes of zero."""
    x, f, xv, fv, _ = conv_case(mx, batch, c, n, h, w, size, seed=c + n)
    win, oh, ow = o.windows(xv, batch, h, w, size, stride, pad)
    bias, res = rand(n, seed=1, spread=0.2), rand(batch, n, oh, ow, seed=2)
    want, tol = o.product_tolerance(win, fv, f64(bias), act, f64(res).transpose(0, 2, 3, 1).reshape(-1, n), "float32")
    lay = lambda a: a.reshape(batch, oh, ow, n).transpose(0, 3, 1, 2)  # noqa: E731
    args = (mx.quantize_nchw(x), mx.quantize_filters(f), batch, h, w, size, stride, pad)
    y, side = mx.conv2d(*args, bias=bias.cuda(), activation=act, residual=res.cuda(), want="both")
    close(y, lay(want), lay(tol))
    only = mx.conv2d(*args, bias=bias.cuda(), activation=act, residual=res.cuda(), want="mx")
    for q in (side, only):
        check_matrix(q, f64(y).transpose(0, 2, 3, 1).reshape(-1, n))


@pytest.mark.parametrize("batch, c, n, h, w, size, stride, pad", [(8, 32, 300, 50, 51, 3, 1, 1), (4, 160, 512, 61, 40, 3, 1, 1), (16, 128, 256, 64, 70, 3, 2, 1),
                                                                  (30, 96, 513, 26, 26, 1, 1, 0), (3, 256, 2000, 70, 60, 1, 1, 0)])
def test_convolutions_that_fill_the_chip(mx, batch, c, n, h, w, size, stride, pad):
    x, f, *_ = conv_case(mx, 1, c, n, h, w, size, seed=c)
    x = torch.cat([x * s for s in torch.linspace(0.5, 1.5, batch).tolist()])
    q, fq = mx.quantize_nchw(x), mx.quantize_filters(f)
    y, side = mx.conv2d(q, fq, batch, h, w, size, stride, pad, activation="leaky", want="both")
    xv = gpu_values(mx, q).view(batch, h, w, c).permute(0, 3, 1, 2)
    fv = gpu_values(mx, fq).view(n, size, size, -1)[..., :c].permute(0, 3, 1, 2)
    xv, fv = xv.cpu(), fv.cpu()
    some = [0, batch // 2, batch - 1]                             # the sums of three images on the CPU
    v = torch.nn.functional.conv2d(xv[some], fv, stride=stride, padding=pad)
    absum = torch.nn.functional.conv2d(xv[some].abs(), fv.abs(), stride=stride, padding=pad)
    want = torch.where(v > 0, v, 0.1 * v)
    tol = ((o.blocks(c) * size * size + 1) // 2 + 16) * 2.0 ** -23 * absum + 2.0 ** -22 * want.abs() + 2.0 ** -24
    off = (y[some].cpu().double() - want).abs() - tol
    assert (off <= 0).all(), off.max()
    again = mx.quantize_nchw(y)
    kb = o.blocks(n)
    assert torch.equal(side.codes[:, :kb * 16], again.codes[:, :kb * 16]) and torch.equal(side.scales[:, :kb], again.scales[:, :kb])


def test_a_convolution_of_size_one_is_the_product(mx):
    x, f, *_ = conv_case(mx, 2, 96, 70, 9, 11, 1)
    fq, q = mx.quantize_filters(f), mx.quantize_nchw(x)
    y = mx.conv2d(q, fq, 2, 9, 11, 1).permute(0, 2, 3, 1).reshape(-1, 70)
    z = mx.matmul(q, fq)
    # the same products of codes; the order of the sum may differ between the two forms
    tol = 2.0 ** -23 * 20 * (mx.dequantize(q).abs() @ mx.dequantize(fq).abs().t())
    assert ((y - z).abs() <= tol).all()


def test_images_of_a_batch_do_not_meet(mx):
    x, f, *_ = conv_case(mx, 3, 64, 64, 11, 7, 3)
    fq = mx.quantize_filters(f)
    y = mx.conv2d(mx.quantize_nchw(x), fq, 3, 11, 7, 3, 1, 1)
    x2 = x.clone()
    x2[1] = float("nan")
    y2 = mx.conv2d(mx.quantize_nchw(x2), fq, 3, 11, 7, 3, 1, 1)
    assert torch.equal(y[0], y2[0]) and torch.equal(y[2], y2[2]) and y2[1].isnan().all()
    x2 = x.clone()
    x2[1, 5, 5, 3] = float("inf")                                 # one block of one pixel
    y2 = mx.conv2d(mx.quantize_nchw(x2), fq, 3, 11, 7, 3, 1, 1)
    hit = torch.zeros(3, 64, 11, 7, dtype=torch.bool)
    hit[1, :, 4:7, 2:5] = True
    assert (y2.isnan().cpu() == hit).all() and torch.equal(y2.cpu()[~hit], y.cpu()[~hit])


def test_side_output_of_results_that_are_not_numbers(mx):
    x, f, *_ = conv_case(mx, 1, 32, 70, 6, 6, 1)
    res = torch.zeros(1, 70, 6, 6, device="cuda")
    res[0, 40, 2, 3], res[0, 69, 0, 0] = float("inf"), float("nan")
    y, q = mx.conv2d(mx.quantize_nchw(x), mx.quantize_filters(f), 1, 6, 6, 1, residual=res, want="both")
    again = mx.quantize_nchw(y)
    assert torch.equal(q.codes[:, :48], again.codes[:, :48]) and torch.equal(q.scales[:, :3], again.scales[:, :3])
    assert (q.scales[2 * 6 + 3, 1] == 255) and (q.scales[0, 2] == 255) and (q.scales[:, :3] == 255).sum() == 2


# ------------------------------------------------------------------ a run of them, streams, graphs, large sizes
def test_a_chain_of_layers(mx):
    """Two convolutions with a [shortcut], then a linear head on the pooled pixels, side outputs against separate rounding."""
    x, f1, *_ = conv_case(mx, 2, 64, 32, 10, 10, 1)
    f2 = conv_case(mx, 2, 32, 64, 10, 10, 3, seed=5)[1]
    q1, q2 = mx.quantize_filters(f1), mx.quantize_filters(f2)
    w = mx.quantize(rand(50, 64, seed=3).cuda())
    a = mx.conv2d(mx.quantize_nchw(x), q1, 2, 10, 10, 1, activation="leaky", want="mx")
    y = mx.conv2d(a, q2, 2, 10, 10, 3, 1, 1, activation="leaky", residual=x)
    a2 = mx.quantize_nchw(mx.conv2d(mx.quantize_nchw(x), q1, 2, 10, 10, 1, activation="leaky"))
    assert torch.equal(y, mx.conv2d(a2, q2, 2, 10, 10, 3, 1, 1, activation="leaky", residual=x))
    pooled = y.amax(dim=(2, 3))
    head = mx.linear(pooled, w, activation="logistic")
    want, tol = o.product_tolerance(o.rounded(f64(pooled)), o.rounded(f64(rand(50, 64, seed=3))), None, "logistic", None, "float32")
    close(head, want, tol)


def test_another_stream(mx):
    w, _ = make(mx, 256, 512, 1)
    x = rand(200, 512, seed=2).cuda()
    want = mx.linear(x, w)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            z = torch.full((200, 512), float("nan"), device="cuda")
            for _ in range(20):
                z = z * 1.0
            z = torch.where(z.isnan(), x, z)                      # only work queued on this stream makes z the input
            got = mx.linear(z, w)
        side.synchronize()
        assert torch.equal(got, want)


def test_two_streams_at_once(mx):
    w, _ = make(mx, 512, 1024, 1)
    xs = [rand(400, 1024, seed=i).cuda() for i in range(2)]
    want = [mx.linear(x, w, activation="leaky") for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(mx.linear(xs[i], w, activation="leaky"))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_captured_and_replayed(mx):
    """Two graphs of the same operators, replayed in turn with new inputs and eager work between them."""
    w, _ = make(mx, 300, 256, 1)
    f = mx.quantize_filters(rand(40, 3, 3, 64, seed=3).permute(0, 3, 1, 2).contiguous().cuda())
    graphs = []
    for m in (1, 150):
        x, img = torch.zeros(m, 256, device="cuda"), torch.zeros(1, 64, 9, 9, device="cuda")
        step = lambda x=x, img=img: (mx.linear(x, w, activation="leaky"), mx.dequantize(mx.quantize(x)), mx.conv2d(mx.quantize_nchw(img), f, 1, 9, 9, 3, 1, 1))  # noqa: E731
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys = step()
        graphs.append((g, x, img, ys, step))
    for turn in range(4):
        for i, (g, x, img, ys, step) in enumerate(graphs):
            x.copy_(rand(*x.shape, seed=10 * turn + i))
            img.copy_(rand(*img.shape, seed=20 * turn + i))
            g.replay()
            torch.cuda.synchronize()
            got = [y.clone() for y in ys]
            want = step()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
            torch.randn(100, 100, device="cuda").sum().item()


def test_the_current_device_stays(mx):
    before = torch.cuda.current_device()
    mx.quantize(torch.zeros(3, 40, device="cuda"))
    assert torch.cuda.current_device() == before


def test_an_error_that_another_call_left_is_not_this_calls(mx):
    """A HIP call of the thread fails and nobody has asked for its error yet: the operators work, report nothing, and leave it there."""
    from yolo2_light_amd._lib import lib
    w, _ = make(mx, 300, 64, 1)
    x = rand(200, 64, seed=2).cuda()
    f, img = mx.quantize_filters(rand(8, 64, 1, 1, seed=3).cuda()), rand(1, 64, 5, 5, seed=4).cuda()
    q, qi, y, y1 = mx.quantize(x), mx.quantize_nchw(img), mx.linear(x, w), mx.linear(x[:1], w)
    v, c = mx.dequantize(q), mx.conv2d(qi, f, 1, 5, 5, 1)
    got = [torch.zeros_like(t) for t in (y, y1, v, c)]
    spare, q2 = torch.empty(200 * 4 * 17, dtype=torch.uint8, device="cuda"), mx.Matrix.empty(200, 64, "cuda")
    del spare                                                     # the allocator holds linear's workspace
    torch.cuda.synchronize()
    lib.hipGetLastError()
    try:
        assert lib.hipSetDevice(4096) != 0                        # no such device: refused, and kept as the thread's last error
        kept = lib.hipPeekAtLastError()
        mx.quantize(x, out=q2)
        mx.linear(x, w, out=got[0])
        mx.linear(x[:1], w, out=got[1])
        mx.dequantize(q2, out=got[2])
        mx.conv2d(qi, f, 1, 5, 5, 1, out=got[3])
        assert lib.hipPeekAtLastError() == kept
    finally:
        lib.hipGetLastError()
    assert all(torch.equal(a, b) for a, b in zip(got, (y, y1, v, c)))


def test_offsets_beyond_32_bits(mx):
    """Inputs, codes and results whose byte offsets pass 2^32: the last rows are as right as the first."""
    rows, k = 66_000, 33_000
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")                  # 4.4 GB
    tail = rand(3, k, seed=1, dtype="bfloat16")
    x[:3], x[-3:] = tail.cuda(), tail.cuda()
    q = mx.quantize(x)
    v = mx.dequantize(q, torch.bfloat16)
    want = o.rounded(f64(tail))
    assert (f64(v[:3]) == want).all() and (f64(v[-3:]) == want).all() and not v[3:-3].any()
    del x, v
    w, wv = make(mx, 7, k, 2)
    want, tol = o.product_tolerance(want, wv, None, "linear", None, "float32")
    y = mx.matmul(q, w)
    close(y[:3], want, tol)
    close(y[-3:], want, tol)
    assert not y[3:-3].any()
    del q, y
    a, av = make(mx, 70_000, 32, 3)
    b, bv = make(mx, 32_768, 32, 4)
    y = mx.matmul(a, b, dtype=torch.bfloat16)                                      # 4.6 GB
    for rows in (slice(0, 3), slice(-3, None)):
        want, tol = o.product_tolerance(av[rows], bv, None, "linear", None, "bfloat16")
        close(y[rows], want, tol)


def test_a_large_map(mx):
    """A result above 2^32 bytes: 40 images of 128 filters at 480 x 480."""
    batch, n, h = 40, 128, 480
    f, q = mx.quantize_filters(rand(n, 1, 1, 32, seed=1).permute(0, 3, 1, 2).contiguous().cuda()), None
    x = torch.zeros(batch, 32, h, h, device="cuda")
    last = rand(h, h, 32, seed=2).permute(2, 0, 1).contiguous()
    x[0], x[-1] = last.cuda(), last.cuda()
    q = mx.quantize_nchw(x)
    y = mx.conv2d(q, f, batch, h, h, 1)
    assert torch.equal(y[0], y[-1]) and not y[1:-1].any()
    rows = f64(last).transpose(1, 2, 0).reshape(-1, 32)[-500:]
    want, tol = o.product_tolerance(o.rounded(rows), o.rounded(f64(mx.dequantize(f))), None, "linear", None, "float32")
    got = y[-1].reshape(n, -1).t()[-500:]
    close(got, want, tol)


def at_the_end(t):
    """t's values in the last bytes of an allocation of its own (32 MB: a segment of the allocator's, nothing behind it)."""
    whole = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    end = whole[(32 << 20) - t.numel() * t.element_size():].view(t.dtype).view(t.shape)
    end.copy_(t)
    return end


@pytest.mark.parametrize("m, n, k", [(1, 48, 96), (5, 72, 160), (33, 64, 64), (40, 256, 160), (41, 261, 100), (129, 136, 96), (257, 1000, 64)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_behind_the_last_are_not_read(mx, m, n, k, dtype):
    """A strip of 32 rows with fewer than a step's rows in it once read the residual of the rows behind them."""
    x, w, b = at_the_end(rand(m, k, seed=1, dtype=dtype)), mx.quantize(rand(n, k, seed=2).cuda()), at_the_end(rand(n, seed=3))
    w = mx.Matrix(at_the_end(w.codes), at_the_end(w.scales), k)
    res = at_the_end(rand(m, n, seed=4, dtype=dtype))
    y = mx.linear(x, w, bias=b, activation="leaky", residual=res, out=at_the_end(torch.zeros(m, n, dtype=TYPES[dtype])))
    q = mx.quantize(x)
    q = mx.Matrix(at_the_end(q.codes), at_the_end(q.scales), k)
    assert torch.equal(y, mx.matmul(q, w, bias=b, activation="leaky", residual=res, dtype=TYPES[dtype]))
    want, tol = o.product_tolerance(o.rounded(f64(x)), o.rounded(f64(rand(n, k, seed=2))), f64(b), "leaky", f64(res), dtype)
    close(y, want, tol)


@pytest.mark.parametrize("batch, c, n, h, w, size, stride, pad", [(1, 32, 33, 9, 9, 3, 1, 1), (2, 64, 70, 7, 5, 1, 1, 0), (1, 128, 100, 13, 13, 3, 2, 1), (3, 40, 255, 6, 6, 1, 1, 0), (8, 32, 41, 70, 70, 3, 1, 1)])
def test_a_convolution_stays_inside_its_tensors(mx, batch, c, n, h, w, size, stride, pad):
    x, f, *_ = conv_case(mx, batch, c, n, h, w, size, seed=c + n)
    oh, ow = (h + 2 * pad - size) // stride + 1, (w + 2 * pad - size) // stride + 1
    bias, res = rand(n, seed=1).cuda(), rand(batch, n, oh, ow, seed=2).cuda()
    q, fq = mx.quantize_nchw(x), mx.quantize_filters(f)
    want, side = mx.conv2d(q, fq, batch, h, w, size, stride, pad, bias=bias, activation="leaky", residual=res, want="both")
    ends = [mx.Matrix(at_the_end(m.codes), at_the_end(m.scales), m.k) for m in (q, fq)]
    got, side2 = mx.conv2d(*ends, batch, h, w, size, stride, pad, bias=at_the_end(bias), activation="leaky", residual=at_the_end(res), out=at_the_end(res), want="both")
    kb = o.blocks(n)
    assert torch.equal(got, want) and torch.equal(side.codes[:, :16 * kb], side2.codes[:, :16 * kb]) and torch.equal(side.scales[:, :kb], side2.scales[:, :kb])
    plain = mx.conv2d(q, fq, batch, h, w, size, stride, pad)
    assert torch.equal(mx.conv2d(*ends, batch, h, w, size, stride, pad, out=at_the_end(plain * 0)), plain)


def test_gradients_are_refused(mx):
    from yolo2_light_amd import YoloHipError
    w, _ = make(mx, 8, 32, 1)
    x = torch.zeros(2, 32, device="cuda", requires_grad=True)
    with pytest.raises(YoloHipError, match="no backward"):
        mx.linear(x, w)
    with torch.no_grad():
        assert mx.linear(x, w).shape == (2, 8)


def test_tangents_are_refused(mx):
    """A dual tensor of forward mode does not require a gradient; its result would have lost the tangent."""
    from torch.autograd import forward_ad
    from yolo2_light_amd import YoloHipError
    w, _ = make(mx, 8, 64, 1)
    x, b = torch.ones(2, 64, device="cuda"), torch.ones(8, device="cuda")
    want = mx.linear(x, w, bias=b)
    with forward_ad.dual_level():
        d, db, m = forward_ad.make_dual(x, x), forward_ad.make_dual(b, b), forward_ad.make_dual(x.view(1, 32, 2, 2), x.view(1, 32, 2, 2))
        for call in (lambda: mx.quantize(d), lambda: mx.linear(d[:1], w), lambda: mx.linear(x, w, bias=db), lambda: mx.quantize_nchw(m), lambda: mx.quantize_filters(m),
                     lambda: mx.linear(x, w, residual=db.expand(2, 8)), lambda: mx.linear(x, w, out=db.expand(2, 8).contiguous())):
            with pytest.raises(YoloHipError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(YoloHipError, match="tangent"):
                call()
        assert torch.equal(mx.linear(x, w, bias=b), want) and torch.equal(mx.linear(forward_ad.unpack_dual(d).primal, w, bias=b), want)
    assert torch.equal(mx.linear(x, w, bias=b), want)


def test_autograd_knows_of_results_written_into_given_tensors(mx):
    """y = a * buffer keeps the buffer for its backward pass; a call that writes the buffer in between must not go unseen."""
    w, _ = make(mx, 8, 64, 1)
    x, img = rand(2, 64, seed=2).cuda(), rand(1, 64, 3, 3, seed=3).cuda()
    q, qi, f = mx.quantize(x), mx.quantize_nchw(img), mx.quantize_filters(rand(8, 64, 1, 1, seed=4).cuda())
    for shape, write in (((2, 8), lambda out: mx.linear(x, w, out=out)), ((2, 8), lambda out: mx.matmul(q, w, out=out)), ((2, 64), lambda out: mx.dequantize(q, out=out)),
                         ((1, 64, 3, 3), lambda out: mx.dequantize_nchw(qi, 1, 3, 3, out=out)), ((1, 8, 3, 3), lambda out: mx.conv2d(qi, f, 1, 3, 3, 1, out=out))):
        a, buffer = torch.ones(shape, device="cuda", requires_grad=True), torch.ones(shape, device="cuda")
        y = (a * buffer).sum()
        write(buffer)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        (a * buffer).sum().backward()                             # with what is there now
        assert torch.equal(a.grad, buffer)
        with torch.inference_mode():
            write(torch.empty(shape, device="cuda"))
    before = q.codes._version, q.scales._version
    mx.quantize(x, out=q)
    assert q.codes._version > before[0] and q.scales._version > before[1]


def test_negated_views_are_refused(mx):
    """z.conj().imag shares z's memory, which holds the negatives of its values."""
    from yolo2_light_amd import YoloHipError
    w, _ = make(mx, 8, 64, 1)
    z = torch.complex(rand(8, 64, seed=1), rand(8, 64, seed=2)).cuda().conj()
    x, one = z.imag, torch.complex(torch.zeros(1), torch.ones(1)).cuda().conj().imag
    assert x.is_neg() and one.is_neg() and one.is_contiguous()
    plain = x.resolve_neg()
    check_matrix(mx.quantize(plain), f64(plain))
    m = z.view(1, 8, 8, 8).imag
    for call in (lambda: mx.quantize(x), lambda: mx.linear(x, w), lambda: mx.quantize_nchw(m), lambda: mx.quantize_filters(m), lambda: mx.dequantize(w, out=x),
                 lambda: mx.linear(plain, w, residual=x[:, :8]), lambda: mx.linear(plain, w, out=x[:, :8]), lambda: mx.linear(plain, w, bias=one.expand(8)),
                 lambda: mx.linear(plain[:, :64], mx.Matrix(w.codes[:1], w.scales[:1], 64), bias=one)):
        with pytest.raises(YoloHipError, match="resolve_neg"):
            call()


def test_python_refusals(mx):
    from yolo2_light_amd import YoloHipError
    w, _ = make(mx, 8, 64, 1)
    x = torch.zeros(2, 64, device="cuda")
    for call in (lambda: mx.linear(x.double(), w), lambda: mx.linear(x[:, :63], w), lambda: mx.linear(x, w, activation="gelu"), lambda: mx.linear(x, w, bias=torch.zeros(7, device="cuda")),
                 lambda: mx.linear(x, w, residual=torch.zeros(2, 9, device="cuda")), lambda: mx.linear(x, w, out=torch.zeros(3, 8, device="cuda")),
                 lambda: mx.linear(x, w, residual=torch.zeros(8, 2, device="cuda").t()), lambda: mx.quantize(torch.zeros(2, 3, 4, device="cuda").transpose(0, 1)),
                 lambda: mx.Matrix(w.codes, w.scales, 200), lambda: mx.Matrix(w.codes[:, :16], w.scales, 64), lambda: mx.conv2d(w, w, 3, 2, 2, 1),
                 lambda: mx.conv2d(mx.quantize(torch.zeros(4, 64, device="cuda")), w, 1, 2, 2, 3), lambda: mx.quantize_nchw(x)):
        with pytest.raises(YoloHipError):
            call()
