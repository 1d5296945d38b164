"""Networks whose convolutions run in MXFP4 (yl_network_set_precision(net, YL_PRECISION_MXFP4)): every such layer against the 64-bit
convolution of the rounded operands (mx_oracle.py), fused == unfused bit for bit, batch items independent."""
import numpy as np
import pytest

import common
import descs as D
import mx_oracle as o
from common import Network

pytestmark = pytest.mark.gpu
MXFP4 = 3


def layer_want(x, wts, bias, li, batch):
    """activation(conv(rounded x, rounded w) + bias) of a layer in 64 bits, with its tolerance, as [batch][n][oh][ow]."""
    c, n, size = li["c"], li["n"], li["size"]
    rows = o.rounded(x.reshape(batch, c, li["h"] * li["w"]).transpose(0, 2, 1).reshape(-1, c))
    f = o.rounded(o.filter_rows(np.asarray(wts, np.float64).reshape(n, c, size, size)))
    win, oh, ow = o.windows(rows, batch, li["h"], li["w"], size, li["stride"], li["pad"])
    act = {D.LEAKY: "leaky", D.LINEAR: "linear", 1: "relu"}[li["activation"]]
    want, tol = o.product_tolerance(win, f, np.asarray(bias, np.float64), act, None, "float32")
    lay = lambda a: a.reshape(batch, oh * ow, n).transpose(0, 2, 1).reshape(-1)  # noqa: E731
    return lay(want), lay(tol)


@pytest.mark.parametrize("shape", [(2, 32, 13, 13, 33, 3, 1, 1), (1, 64, 26, 26, 64, 3, 2, 1), (3, 96, 7, 9, 255, 1, 1, 0), (2, 128, 13, 13, 128, 1, 1, 0), (1, 32, 12, 12, 24, 5, 1, 2)])
def test_one_layer(shape):
    B, C, H, W, M, size, stride, pad = shape
    rng = np.random.default_rng(M + size)
    w0, b0 = rng.normal(0, 0.3, C * C).astype(np.float32), rng.normal(0, 0.1, C).astype(np.float32)
    wts, bias = rng.normal(0, (2.0 / (C * size * size)) ** 0.5, M * C * size * size).astype(np.float32), rng.normal(0, 0.5, M).astype(np.float32)
    x = rng.standard_normal((B, C, H, W)).astype(np.float32)
    layers = [D.conv(B, W, H, C, C, 1, 1, 0, D.LEAKY, w0, b0), D.conv(B, W, H, C, M, size, stride, pad, D.LEAKY, wts, bias)]
    net = Network.from_desc(layers, B, W, H, C)
    net.set_precision(MXFP4)
    net.to_device(0)
    got = net.predict(x)
    assert "mx_product" not in net.layer_kernel(0) and "mx_product" in net.layer_kernel(1)
    want, tol = layer_want(net.layer_output(0), wts, bias, net.layers()[1], B)
    assert (np.abs(got - want) <= tol).all()
    net.close()


@pytest.mark.parametrize("name, width, height, batch", [("yolov3", 96, 96, 2), ("yolov3", 160, 96, 3), ("yolov3-tiny", 96, 96, 2)])
def test_networks_teacher_forced_and_fused(name, width, height, batch):
    cfg, wts = common.model_files(name, width, height)
    x = common.seeded_input(batch, 3, height, width)
    plain = Network.load(cfg, wts, batch, 0, device=0, mxfp4=True)
    fused = Network.load(cfg, wts, batch, 0, device=0, fuse=True, mxfp4=True)
    plain.predict(x)
    fused.predict(x)
    infos, n = plain.layers(), 0
    for i, li in enumerate(infos):
        if li["type"] != common.CONV or "mx_product" not in plain.layer_kernel(i):
            assert li["int8"] == 0
            continue
        n += 1
        assert li["int8"] == 3 and li["conv_mode"] == 4
        want, tol = layer_want(plain.layer_output(i - 1), plain.layer_weights(i), plain.layer_biases(i), li, batch)
        assert (np.abs(plain.layer_output(i) - want) <= tol).all(), "layer %d" % i
    assert n == (9 if name == "yolov3-tiny" else 71)              # all but the first layer, the linear heads and (tiny) 16 channels
    checked = 0
    for i, li in enumerate(infos):
        if fused.layer_materialised(i):
            assert np.array_equal(plain.layer_output(i).view(np.uint32), fused.layer_output(i).view(np.uint32)), "layer %d" % i
            checked += 1
    assert checked > 10 and any(not fused.layer_materialised(i) for i in range(len(infos)))
    for b in range(batch):
        assert np.array_equal(plain.get_boxes(b, width, height, 0.24, nms=0.4), fused.get_boxes(b, width, height, 0.24, nms=0.4))
    again = fused.predict(x).copy()
    assert np.array_equal(again, plain.predict(x))
    plain.close(); fused.close()


@pytest.mark.parametrize("act", ["logistic", "relu", "relie", "ramp", "tanh", "plse", "elu", "loggy", "hardtan", "lhtan"])
def test_a_layer_of_any_activation(act):
    """The rare ones are a pass of their own behind the product, RELU too."""
    from yolo2_light_amd.mx import ACTIVATIONS
    B, C, H, W, M = 2, 64, 9, 11, 70
    rng = np.random.default_rng(ACTIVATIONS[act])
    w0, b0 = rng.normal(0, 0.3, C * C).astype(np.float32), rng.normal(0, 0.1, C).astype(np.float32)
    wts, bias = rng.normal(0, (2.0 / (C * 9)) ** 0.5, M * C * 9).astype(np.float32), rng.normal(0, 0.5, M).astype(np.float32)
    net = Network.from_desc([D.conv(B, W, H, C, C, 1, 1, 0, D.LEAKY, w0, b0), D.conv(B, W, H, C, M, 3, 1, 1, ACTIVATIONS[act], wts, bias)], B, W, H, C)
    net.set_precision(MXFP4)
    net.to_device(0)
    got = net.predict(rng.standard_normal((B, C, H, W)).astype(np.float32))
    assert "mx_product" in net.layer_kernel(1)
    rows = o.rounded(net.layer_output(0).reshape(B, C, H * W).transpose(0, 2, 1).reshape(-1, C))
    win, oh, ow = o.windows(rows, B, H, W, 3, 1, 1)
    want, tol = o.product_tolerance(win, o.rounded(o.filter_rows(wts.astype(np.float64).reshape(M, C, 3, 3))), bias.astype(np.float64), act, None, "float32")
    lay = lambda a: a.reshape(B, oh * ow, M).transpose(0, 2, 1).reshape(-1)  # noqa: E731
    assert (np.abs(got - lay(want)) <= lay(tol)).all()
    net.close()


def test_a_network_at_its_own_size():
    """yolov3 at 608 x 608: its layers fill the chip in other tiles than the small maps above; some of every stage in 64 bits, fused == unfused."""
    torch = pytest.importorskip("torch")
    from yolo2_light_amd import mx
    cfg, wts = common.model_files("yolov3", 608, 608)
    batch = 2
    x = common.seeded_input(batch, 3, 608, 608)
    plain = Network.load(cfg, wts, batch, 0, device=0, mxfp4=True)
    plain.predict(x)
    infos, kernels = plain.layers(), set()
    for i in (1, 2, 5, 7, 12, 13, 38, 63, 75, 87):
        li = infos[i]
        assert li["int8"] == 3
        kernels.add(plain.layer_kernel(i))
        c, n, size, h, w = li["c"], li["n"], li["size"], li["h"], li["w"]
        src = torch.from_numpy(np.ascontiguousarray(plain.layer_output(i - 1).reshape(batch, c, h, w))).cuda()
        f = torch.from_numpy(np.ascontiguousarray(plain.layer_weights(i).reshape(n, c, size, size))).cuda()
        xv = mx.dequantize_nchw(mx.quantize_nchw(src), batch, h, w).double().cpu()            # compared with mx_oracle.py in test_gpu_mx.py
        fv = mx.dequantize(mx.quantize_filters(f)).double().view(n, size, size, c).permute(0, 3, 1, 2).cpu()
        del src, f
        step = max(1, n // 32)                                    # every step-th filter, the last one too
        some = sorted(set(range(0, n, step)) | {n - 1})
        v = torch.nn.functional.conv2d(xv, fv[some], stride=li["stride"], padding=li["pad"])
        tol = ((c // 32 * size * size + 1) // 2 + 16) * 2.0 ** -23 * torch.nn.functional.conv2d(xv.abs(), fv[some].abs(), stride=li["stride"], padding=li["pad"])
        v = v + torch.from_numpy(plain.layer_biases(i).astype(np.float64))[some][None, :, None, None]
        want = torch.where(v > 0, v, 0.1 * v)
        tol = tol + 2.0 ** -22 * (v.abs() + tol) + 2.0 ** -24
        got = torch.from_numpy(plain.layer_output(i).reshape(batch, n, li["out_h"], li["out_w"])[:, some].astype(np.float64))
        assert ((got - want).abs() <= tol).all(), "layer %d" % i
        print("layer %d" % i, flush=True)
    assert any("64x128" in k for k in kernels) and any("64x64" in k for k in kernels), kernels
    heads = {i: plain.layer_output(i).copy() for i, li in enumerate(infos) if li["type"] == common.YOLO}
    plain.close()
    fused = Network.load(cfg, wts, batch, 0, device=0, fuse=True, mxfp4=True)
    fused.predict(x)
    assert len(heads) == 3 and all(np.array_equal(fused.layer_output(i).view(np.uint32), h.view(np.uint32)) for i, h in heads.items())
    fused.close()


def test_batch_items_are_independent():
    cfg, wts = common.model_files("yolov3", 96, 96)
    x = common.seeded_input(3, 3, 96, 96)
    net = Network.load(cfg, wts, 3, 0, device=0, fuse=True, mxfp4=True)
    one = Network.load(cfg, wts, 1, 0, device=0, fuse=True, mxfp4=True)
    net.predict(x)
    heads = [i for i, li in enumerate(net.layers()) if li["type"] == common.YOLO]
    whole = {i: net.layer_output(i).reshape(3, -1).copy() for i in heads}
    for b in range(3):
        one.predict(x[b:b + 1])
        for i in heads:
            close = np.abs(one.layer_output(i) - whole[i][b])
            assert np.array_equal(one.layer_output(i), whole[i][b]), (i, b, close.max())
    net.close(); one.close()


def test_precision_is_set_before_the_device():
    cfg, wts = common.model_files("yolov3-tiny", 96, 96)
    net = Network.load(cfg, wts, 1, 0, device=0)
    with pytest.raises(Exception, match="precede"):
        net.set_precision(MXFP4)
    net.close()


def test_the_price_of_four_bits_is_reported_and_bounded():
    """Head tensors of an MXFP4 run against the FP32 run of the same images (synthetic weights): no parity claim, a bound that catches a
    broken path (an unrelated tensor correlates near 0)."""
    cfg, wts = common.model_files("yolov3", 160, 160)
    x = common.seeded_input(2, 3, 160, 160)
    f32 = Network.load(cfg, wts, 2, 0, device=0, fuse=True)
    mx4 = Network.load(cfg, wts, 2, 0, device=0, fuse=True, mxfp4=True)
    f32.predict(x)
    mx4.predict(x)
    for i, li in enumerate(f32.layers()):
        if li["type"] == common.YOLO:
            corr = float(np.corrcoef(f32.layer_output(i), mx4.layer_output(i))[0, 1])
            print("head %d: correlation %.4f" % (i, corr))
            assert corr > 0.5
    f32.close(); mx4.close()
