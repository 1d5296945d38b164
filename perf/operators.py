"""The MXFP4 operators, measured: rounding to microscaled 4-bit floating point and back, the product of two such matrices, the
linear layer that rounds its input on the way, and the convolution layer over a map.

An MXFP4 matrix holds, for every row, blocks of 32 consecutive values: 32 E2M1 codes (16 bytes, the even element in the low half of
a byte) and one E8M0 scale byte.  A block's scale is 2^(floor(log2 max|x|) - 2); its codes are x / scale, rounded to the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code) and saturated at 6.

`run` computes an operator in elementary torch operations where `own` is false and with yolo2_light_amd.mx where it is true."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32


def listed():
    return [
        # rounding to MXFP4 and back: the row of one decoding step; a batch of feature maps of the 76 x 76 stage of a 608 x 608
        # detector; a padded batch of rows whose length is no multiple of the block
        {"name": "round_token", "op": "round", "layout": "rows", "rows": 1, "k": 4096, "pad": 0, "type": "bf16"},
        {"name": "round_map", "op": "round", "layout": "nchw", "batch": 16, "c": 256, "h": 76, "w": 76, "type": "f32"},
        {"name": "round_ragged", "op": "round", "layout": "rows", "rows": 3001, "k": 1005, "pad": 11, "type": "f16"},
        # the product of two quantised matrices: the largest square one; a few hundred rows against a layer's weights; odd sizes with
        # the whole epilogue
        {"name": "matmul_large", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False, "act": "linear", "residual": False},
        {"name": "matmul_rows", "op": "matmul", "m": 512, "n": 4096, "k": 4096, "type": "f16", "bias": True, "act": "relu", "residual": False},
        {"name": "matmul_ragged", "op": "matmul", "m": 1001, "n": 1237, "k": 1511, "type": "f32", "bias": True, "act": "leaky", "residual": True},
        # the linear layer on values that it rounds itself: a single token, the tokens of a batch that decodes, a prompt
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "pad": 0, "type": "bf16", "bias": True, "act": "linear", "residual": False},
        {"name": "linear_batch", "op": "linear", "m": 40, "n": 8192, "k": 8192, "pad": 0, "type": "bf16", "bias": True, "act": "linear", "residual": True},
        {"name": "linear_prompt", "op": "linear", "m": 4096, "n": 16384, "k": 4096, "pad": 64, "type": "bf16", "bias": True, "act": "relu", "residual": False},
        # convolution layers of a 608 x 608 detector on eight images: the deepest 3 x 3 layer, a 1 x 1 layer of the 76 x 76 stage,
        # a 3 x 3 layer of stride 2
        {"name": "conv3_deep", "op": "conv", "batch": 8, "c": 512, "n": 1024, "h": 19, "w": 19, "size": 3, "stride": 1, "act": "leaky", "residual": True},
        {"name": "conv1_wide", "op": "conv", "batch": 8, "c": 256, "n": 128, "h": 76, "w": 76, "size": 1, "stride": 1, "act": "leaky", "residual": False},
        {"name": "conv3_down", "op": "conv", "batch": 8, "c": 64, "n": 128, "h": 152, "w": 152, "size": 3, "stride": 2, "act": "leaky", "residual": False},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _fits(case):
    w = work(case)
    if case["op"] == "round":  # no more than the listed map
        return w["bytes"] <= 8 * 16 * 256 * 76 * 76
    return w["flops"] <= 2 * 8192 ** 3 and w["bytes"] <= 1 << 28


def draw(rng):
    while True:
        op = rng.choice(("round", "round", "matmul", "matmul", "linear", "linear", "linear", "conv", "conv"))
        act = rng.choice(("linear", "linear", "leaky", "relu", "logistic"))
        flags = {"bias": rng.random() < 0.6, "act": act, "residual": rng.random() < 0.4}
        kind = rng.choice(("bf16", "bf16", "f16", "f32"))
        if op == "round" and rng.random() < 0.5:
            case = {"op": op, "layout": "nchw", "batch": _log(rng, 1, 16), "c": _log(rng, 3, 1024), "h": _log(rng, 1, 152), "w": _log(rng, 1, 152), "type": kind}
        elif op == "round":
            case = {"op": op, "layout": "rows", "rows": _log(rng, 1, 65536), "k": _log(rng, 1, 16384), "pad": rng.choice((0, 0, 3, 64)), "type": kind}
        elif op == "matmul":
            case = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 16, 16384), "k": _log(rng, 32, 16384), "type": kind, **flags}
        elif op == "linear":
            m = _log(rng, 1, 64) if rng.random() < 0.6 else _log(rng, 64, 8192)
            case = {"op": op, "m": m, "n": _log(rng, 16, 16384), "k": _log(rng, 32, 16384), "pad": rng.choice((0, 0, 3, 64)), "type": kind, **flags}
        else:
            case = {"op": op, "batch": _log(rng, 1, 16), "c": _log(rng, 16, 1024), "n": _log(rng, 16, 1024), "h": _log(rng, 7, 152), "w": _log(rng, 7, 152),
                    "size": rng.choice((1, 3)), "stride": rng.choice((1, 1, 2)), "act": rng.choice(("leaky", "linear", "relu")), "residual": rng.random() < 0.3}
        if _fits(case):
            return case


def _out_hw(case):
    pad = case["size"] // 2
    return tuple((case[d] + 2 * pad - case["size"]) // case["stride"] + 1 for d in ("h", "w"))


def work(case):
    packed = 17.0 / 32.0  # bytes of a value in MXFP4, its share of the scale included
    if case["op"] == "round":
        n = case["rows"] * case["k"] if case["layout"] == "rows" else case["batch"] * case["c"] * case["h"] * case["w"]
        return {"bytes": 2.0 * n * BYTES[case["type"]], "flops": 2.0 * n}
    if case["op"] == "conv":
        oh, ow = _out_hw(case)
        taps, outs = case["size"] ** 2, case["batch"] * case["n"] * oh * ow
        read = 4.0 * case["batch"] * case["c"] * case["h"] * case["w"] + packed * case["n"] * case["c"] * taps + 4.0 * case["n"]
        return {"bytes": read + 4.0 * outs * (2 if case["residual"] else 1), "flops": 2.0 * outs * case["c"] * taps}
    m, n, k, size = case["m"], case["n"], case["k"], BYTES[case["type"]]
    x = packed * m * k if case["op"] == "matmul" else size * m * k
    return {"bytes": x + packed * n * k + size * m * n * (2 if case["residual"] else 1) + (4.0 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------- inputs


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, k):
    """Rows of a layer's input: channels of different magnitude, a few of them far above the others."""
    size = torch.exp(0.5 * _normal(gen, k))
    size[torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 100)]] *= 12.0
    return _normal(gen, rows, k) * size


def _map(gen, case):
    """A feature map behind a leaky activation."""
    x = _normal(gen, case["batch"], case["c"], case["h"], case["w"]) * torch.exp(0.5 * _normal(gen, 1, case["c"], 1, 1))
    return torch.where(x > 0, x, 0.1 * x)


def _pack(x):
    """[rows, k] in FP32 -> codes uint8 [rows, 16 * blocks] and scales uint8 [rows, blocks], blocks a multiple of four."""
    rows, k = x.shape
    blocks = (k + 4 * BLOCK - 1) // (4 * BLOCK) * 4
    code, exponent = _code_and_exponent(x)
    codes = torch.zeros(rows, blocks * BLOCK, dtype=torch.uint8, device=x.device)
    codes[:, : code.shape[1]] = code
    scales = torch.zeros(rows, blocks, dtype=torch.uint8, device=x.device)
    scales[:, : exponent.shape[1]] = (exponent + 127).to(torch.uint8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales


def _filters(w):
    """[n, c, size, size] -> [n, size * size * c'] with c' = c padded by zeros to whole blocks: the order in which filters are kept."""
    n, c, size, _ = w.shape
    w = torch.nn.functional.pad(w.permute(0, 2, 3, 1), (0, -c % BLOCK))
    return w.reshape(n, -1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case)}
    if case["op"] == "round":
        kind = DTYPES[case["type"]]
        if case["layout"] == "nchw":
            s["x"] = _map(gen, case).to(kind)
        else:
            s["x"] = _activations(gen, case["rows"], case["k"] + case["pad"]).to(kind)[:, : case["k"]]
        return s
    if case["op"] == "conv":
        c, n, size = case["c"], case["n"], case["size"]
        s["x"] = _map(gen, case)
        w = _normal(gen, n, c, size, size) / math.sqrt(c * size * size)
        s["w_codes"], s["w_scales"] = _pack(_filters(w))
        s["bias"] = 0.2 * _normal(gen, n)
        oh, ow = _out_hw(case)
        s["residual"] = _normal(gen, case["batch"], n, oh, ow) if case["residual"] else None
        return s
    m, n, k, kind = case["m"], case["n"], case["k"], DTYPES[case["type"]]
    if case["op"] == "matmul":
        s["x_codes"], s["x_scales"] = _pack(_activations(gen, m, k))
    else:
        s["x"] = _activations(gen, m, k + case["pad"]).to(kind)[:, :k]
    s["w_codes"], s["w_scales"] = _pack(_normal(gen, n, k) / math.sqrt(k))
    s["bias"] = 0.2 * _normal(gen, n) if case["bias"] else None
    s["residual"] = _normal(gen, m, n).to(kind) if case["residual"] else None
    return s


# ---------------------------------------------------------------- the plain form


def _code_and_exponent(x):
    """FP32 [rows, k] -> E2M1 codes uint8 [rows, 32 * blocks] and the blocks' exponents [rows, blocks]."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    exponent = (torch.frexp(x.abs().amax(dim=2)).exponent - 3).clamp(min=-127)
    a = torch.ldexp(x.abs(), -exponent.unsqueeze(2).to(torch.int32))
    code = torch.bucketize(a, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)).to(torch.uint8)  # ties down
    for tie, up in ((0.75, 2), (1.75, 4), (3.5, 6)):  # ... but to the even code
        code = torch.where(a == tie, up, code)
    code = code | (torch.signbit(x).to(torch.uint8) << 3)
    exponent = torch.where(x.abs().amax(dim=2) == 0, -127, exponent)
    return code.reshape(rows, -1), exponent


def _values(code, exponent, k):
    """The values that codes [rows, 32 * blocks] and exponents [rows, blocks] stand for, FP32 [rows, k]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=code.device)
    v = table[code.int()].reshape(code.shape[0], -1, BLOCK)
    return torch.ldexp(v, exponent.unsqueeze(2).to(torch.int32)).reshape(code.shape[0], -1)[:, :k]


def _rounded(x):
    code, exponent = _code_and_exponent(x)
    return _values(code, exponent, x.shape[1])


def _unpacked(codes, scales, k):
    code = torch.stack((codes & 15, codes >> 4), dim=2).reshape(codes.shape[0], -1)
    return _values(code, scales.int() - 127, k)


def _activate(y, act):
    if act == "leaky":
        return torch.where(y > 0, y, 0.1 * y)
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "logistic":
        return 1.0 / (1.0 + torch.exp(-y))
    return y


def _as_rows(x):
    return x.permute(0, 2, 3, 1).reshape(-1, x.shape[1])


def _as_map(rows, b, h, w):
    return rows.reshape(b, h, w, -1).permute(0, 3, 1, 2)


def _windows(x, size, stride):
    """[b, c, h, w] -> [b * oh * ow, size * size * c]: the values under every position of a filter."""
    pad = size // 2
    oh, ow = ((d + 2 * pad - size) // stride + 1 for d in x.shape[2:])
    x = torch.nn.functional.pad(x, (pad, pad, pad, pad))
    taps = [x[:, :, i: i + stride * (oh - 1) + 1: stride, j: j + stride * (ow - 1) + 1: stride] for i in range(size) for j in range(size)]
    return torch.cat([_as_rows(t) for t in taps], dim=1)


def _plain(s):
    case = s["case"]
    if case["op"] == "round":
        x = s["x"]
        if case["layout"] == "rows":
            return _rounded(x.float()).to(x.dtype)
        b, _, h, w = x.shape
        return _as_map(_rounded(_as_rows(x.float())), b, h, w).to(x.dtype).contiguous()
    if case["op"] == "conv":
        b, c, h, w = s["x"].shape
        x = _as_map(_rounded(_as_rows(s["x"])), b, h, w)
        taps = case["size"] ** 2
        blocks = (c + BLOCK - 1) // BLOCK
        f = _unpacked(s["w_codes"], s["w_scales"], taps * blocks * BLOCK).reshape(case["n"], taps, -1)[:, :, :c].reshape(case["n"], -1)
        y = _activate(_windows(x, case["size"], case["stride"]) @ f.t() + s["bias"], case["act"])
        y = _as_map(y, b, *_out_hw(case))
        return (y + s["residual"] if case["residual"] else y).contiguous()
    k = case["k"]
    x = _unpacked(s["x_codes"], s["x_scales"], k) if case["op"] == "matmul" else _rounded(s["x"].float())
    y = x @ _unpacked(s["w_codes"], s["w_scales"], k).t()
    if case["bias"]:
        y = y + s["bias"]
    y = _activate(y, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    return y.to(DTYPES[case["type"]])


def run(s):
    if not own:
        return _plain(s)
    from yolo2_light_amd import mx

    case = s["case"]
    if case["op"] == "round":
        x = s["x"]
        if case["layout"] == "rows":
            return mx.dequantize(mx.quantize(x), x.dtype)
        return mx.dequantize_nchw(mx.quantize_nchw(x), x.shape[0], x.shape[2], x.shape[3], x.dtype)
    if case["op"] == "conv":
        b, c, h, w = s["x"].shape
        taps = case["size"] ** 2
        filters = mx.Matrix(s["w_codes"], s["w_scales"], taps * ((c + BLOCK - 1) // BLOCK) * BLOCK)
        return mx.conv2d(mx.quantize_nchw(s["x"]), filters, b, h, w, case["size"], case["stride"], case["size"] // 2,
                         bias=s["bias"], activation=case["act"], residual=s["residual"])
    w = mx.Matrix(s["w_codes"], s["w_scales"], case["k"])
    more = {"bias": s["bias"], "activation": case["act"], "residual": s["residual"], "dtype": DTYPES[case["type"]]}
    if case["op"] == "matmul":
        return mx.matmul(mx.Matrix(s["x_codes"], s["x_scales"], case["k"]), w, **more)
    return mx.linear(s["x"], w, **more)


# ---------------------------------------------------------------- the definition in 64 bits


def _exact_rounded(x):
    x = x.double()
    rows, k = x.shape
    blocks = (k + BLOCK - 1) // BLOCK
    full = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :k] = x
    full = full.view(rows, blocks, BLOCK)
    top = full.abs().max(dim=2, keepdim=True).values
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2)
    a = full.abs() / scale
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = (torch.round(a / step) * step).clamp(max=6)  # a whole number of steps, halves to the even one
    return (torch.sign(full) * a * scale).view(rows, -1)[:, :k]


def _exact_unpacked(codes, scales, k):
    rows = codes.shape[0]
    c = torch.empty(rows, codes.shape[1] * 2, dtype=torch.int32, device=codes.device)
    c[:, 0::2] = codes.int() % 16
    c[:, 1::2] = codes.int() // 16
    field, low = (c // 2) % 4, (c % 2).double()
    v = torch.where(field == 0, 0.5 * low, (1 + 0.5 * low) * torch.exp2(field.double() - 1))
    v = torch.where(c >= 8, -v, v).view(rows, -1, BLOCK) * torch.exp2(scales.double() - 127).unsqueeze(2)
    return v.view(rows, -1)[:, :k]


def _exact_activate(y, act):
    return {"linear": lambda: y, "leaky": lambda: torch.maximum(y, 0.1 * y), "relu": lambda: y.clamp(min=0), "logistic": lambda: torch.sigmoid(y)}[act]()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "round":
        x = s["x"]
        if case["layout"] == "rows":
            return _exact_rounded(x)
        b, c, h, w = x.shape
        return _exact_rounded(x.movedim(1, 3).reshape(-1, c)).view(b, h, w, c).movedim(3, 1).contiguous()
    if case["op"] == "conv":
        b, c, h, w = s["x"].shape
        n, size, stride, pad = case["n"], case["size"], case["stride"], case["size"] // 2
        oh, ow = _out_hw(case)
        whole = (c + BLOCK - 1) // BLOCK * BLOCK
        x = torch.zeros(b, h + 2 * pad, w + 2 * pad, c, dtype=torch.float64, device="cuda")
        x[:, pad: pad + h, pad: pad + w] = _exact_rounded(s["x"].movedim(1, 3).reshape(-1, c)).view(b, h, w, c)
        f = _exact_unpacked(s["w_codes"], s["w_scales"], size * size * whole).view(n, size, size, whole)
        y = s["bias"].double().expand(b, oh, ow, n).clone()
        for i in range(size):
            for j in range(size):
                under = x[:, i: i + stride * (oh - 1) + 1: stride, j: j + stride * (ow - 1) + 1: stride]
                y += (under.reshape(-1, c) @ f[:, i, j, :c].t().contiguous()).view(b, oh, ow, n)
        y = _exact_activate(y.movedim(3, 1), case["act"])
        return (y + s["residual"].double() if case["residual"] else y).contiguous()
    k = case["k"]
    x = _exact_unpacked(s["x_codes"], s["x_scales"], k) if case["op"] == "matmul" else _exact_rounded(s["x"])
    y = torch.mm(x, _exact_unpacked(s["w_codes"], s["w_scales"], k).t())
    if case["bias"]:
        y += s["bias"].double()
    y = _exact_activate(y, case["act"])
    return y + s["residual"].double() if case["residual"] else y
