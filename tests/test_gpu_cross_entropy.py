"""GPU: softmax cross entropy of a pointwise classifier against the same formulas in 64 bits."""
import math

import pytest
import torch

import step_reference as R
from mappedconvolutions_b200 import host, ops as twin
from mappedconvolutions_b200 import nn as mnn

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def image(g, shape, dtype, layout, scale=1.0):
    t = (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


def classifier(g, classes, cin, dtype, scale=4.0):
    s = scale / math.sqrt(cin)
    u = lambda *shape: ((torch.rand(shape, generator=g, device="cuda") * 2 - 1) * s).to(dtype)  # noqa: E731
    return u(classes, cin, 1), u(classes)


def labels(g, shape, classes, ignored, ignore=-100):
    t = torch.randint(0, classes, shape, generator=g, device="cuda")
    t[torch.rand(shape, generator=g, device="cuda") < ignored] = ignore
    return t


def layout_kept(t, layout):
    return t.is_contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t.is_contiguous()


# (batch, height, width, channels, classes): single values, one class, odd counts, tile edges and one past them, many classes
SHAPES = [(1, 1, 1, 1, 1), (1, 1, 3, 5, 2), (2, 3, 5, 3, 7), (1, 1, 642, 64, 642), (3, 11, 13, 50, 99), (2, 8, 16, 128, 128),
          (1, 9, 57, 200, 257), (2, 1, 129, 256, 129), (1, 16, 16, 8, 1000), (4, 12, 11, 24, 13), (1, 1, 127, 65, 2562),
          (1, 2, 64, 320, 130), (2, 25, 21, 72, 511), (9, 2, 3, 17, 40)]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_forward_and_backward(ops, i, dtype, layout):
    b, h, w, cin, classes = SHAPES[i]
    g = torch.Generator("cuda").manual_seed(i)
    x = image(g, (b, cin, h, w), dtype, layout)
    weight, bias = classifier(g, classes, cin, dtype)
    target = labels(g, (b, h, w), classes, (0.0, 0.3)[i % 2])
    mean = i % 3 != 0
    grad = torch.tensor(1.7, device="cuda", dtype=F64 if dtype == F64 else F32)
    if mean and not (target != -100).any():
        target[0, 0, 0] = 0
    want = R.cross_entropy(x, weight, bias, target, -100, mean, grad)
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean)
    assert loss.dtype == grad.dtype and loss.dim() == 0 and layout_kept(gx, layout)
    R.check(dict(loss=loss, gx=gx, gw=gw, gb=gb), want, str(SHAPES[i]))
    loss2, saved2 = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
    again = ops.cross_entropy_backward(grad, saved2, x, weight, bias, target, -100, mean)
    assert torch.equal(loss, loss2) and all(torch.equal(p, q) for p, q in zip((gx, gw, gb), again))
    only_x = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean, True, False)
    only_w = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean, False, True)
    assert torch.equal(only_x[0], gx) and only_x[1] is None and only_w[0] is None and torch.equal(only_w[1], gw)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("pixels,classes", [(40_000, 700), (300, 20_000), (9000, 2562)])
def test_several_pieces(ops, pixels, classes, dtype):
    """scores of more than one piece, shares of the pixels, parts of the classes"""
    g = torch.Generator("cuda").manual_seed(21)
    x = image(g, (2, 40, 1, pixels // 2), dtype, "nchw")
    weight, bias = classifier(g, classes, 40, dtype)
    target = labels(g, (2, 1, pixels // 2), classes, 0.1)
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    got = dict(zip(("gx", "gw", "gb"), ops.cross_entropy_backward(grad, saved, x, weight, bias, target)))
    R.check(dict(loss=loss, **got), R.cross_entropy(x, weight, bias, target, -100, True, grad), "pieces")


# float32 layers of 10^7 products and more (from 2048 weights on: tensor cores, three bf16 parts of every value): odd counts, one block of channels or
# classes and one more, one image or several
MANY = [(2, 1, 3, 1 << 20, 20), (3, 67, 101, 77, 99), (1, 1, 40962, 64, 64), (2, 1, 10242, 65, 129), (1, 130, 129, 128, 257), (5, 33, 40, 10, 2562), (1, 1, 600, 200, 1000),
        (1, 300, 400, 1, 1000), (7, 1, 2562, 130, 63)]


# bf16: tiles of 64, 128 and 256 classes whose weights stay in shared memory, or travel beside several tiles of classes
WIDE = [(1, 1, 60_001, 40, 13), (3, 100, 203, 64, 99), (1, 1, 45_000, 256, 250), (2, 1, 30_001, 320, 70), (1, 150, 400, 24, 300), (5, 1, 10_242, 96, 129)]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("i", range(len(WIDE)))
def test_many_pixels(ops, i, layout):
    b, h, w, cin, classes = WIDE[i]
    g = torch.Generator("cuda").manual_seed(70 + i)
    x = image(g, (b, cin, h, w), BF, layout)
    weight, bias = classifier(g, classes, cin, BF)
    target = labels(g, (b, h, w), classes, 0.2)
    grad = torch.tensor(2.5, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    got = dict(zip(("gx", "gw", "gb"), ops.cross_entropy_backward(grad, saved, x, weight, bias, target)))
    R.check(dict(loss=loss, **got), R.cross_entropy(x, weight, bias, target, -100, True, grad), str(WIDE[i]))


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("i", range(len(MANY)))
def test_float32_of_many_products(ops, i, layout):
    b, h, w, cin, classes = MANY[i]
    g = torch.Generator("cuda").manual_seed(50 + i)
    x = image(g, (b, cin, h, w), F32, layout)
    weight, bias = classifier(g, classes, cin, F32)
    target = labels(g, (b, h, w), classes, 0.2)
    off = (target == -100)[:, None].expand_as(x)
    grad = torch.tensor(-0.6, device="cuda")
    mean = i % 2 == 0
    want = R.cross_entropy(x, weight, bias, target, -100, mean, grad)
    results = []
    for value in (0.0, float("nan"), float("inf")):  # whatever the pixels without a label hold
        x = torch.where(off, torch.full_like(x, value), x)
        x = x.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else x.contiguous()
        loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
        results.append([loss] + ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean))
        assert layout_kept(results[-1][1], layout)
        assert all(torch.equal(p, q) for p, q in zip(results[0], results[-1]))
    R.check(dict(zip(("loss", "gx", "gw", "gb"), results[0])), want, str(MANY[i]))
    # as near as float32 sums are: relative errors of whole tensors.  (A float32 sum of n channels is a random walk of n roundings:
    # sqrt(n) 2^-24 of the scores, which exponentials pass on as relative errors; below 5e-6 for all but 2^20 channels.)
    near = max(5e-6, cin ** 0.5 * 2.0 ** -24)
    for got, name in zip(results[0], ("loss", "gx", "gw", "gb")):
        assert (got.double() - want[name][0]).norm() <= near * want[name][0].norm(), name
    only_x = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean, True, False)
    only_w = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean, False, True)
    assert torch.equal(only_x[0], results[0][1]) and torch.equal(only_w[1], results[0][2])
    few = bias.clone()
    few[classes // 2:] = -float("inf")  # classes ruled out, and a label that is none
    target = target.clamp(max=classes // 2 - 1)
    x = torch.where(off, torch.zeros_like(x), x)
    loss, saved = ops.cross_entropy_forward(x, weight, few, target, -100, mean)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, few, target, -100, mean)
    half = R.cross_entropy(x, weight[:classes // 2], bias[:classes // 2], target, -100, mean, grad)
    R.check(dict(loss=loss, gx=gx, gw=gw[:classes // 2], gb=gb[:classes // 2]), half, "ruled out")
    assert not gw[classes // 2:].any() and not gb[classes // 2:].any()
    target[0, 0, 0] = classes
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean)
    assert loss.isnan() and gw.isnan().all() and gb.isnan().all() and gx[0, :, 0, 0].isnan().all() and gx[-1, :, -1, -1].isfinite().all()


# float32 layers of few classes on both sides of the rule for the tensor cores (768 weights of 48 channels or more, 2.5e6 products), one
# class among them, odd counts, fewer pixels than a tile in the last image's planes
FEW = [(1, 1, 3300, 1000, 1), (2, 41, 43, 1024, 1), (1, 1, 1700, 770, 2), (3, 37, 31, 256, 3), (1, 60, 71, 48, 16), (1, 60, 71, 47, 17),
       (5, 1, 1301, 64, 13), (1, 1, 977, 64, 40), (1, 1, 976, 64, 40), (2, 1, 131, 100, 99)]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("i", range(len(FEW)))
def test_float32_of_few_classes(ops, i, layout):
    b, h, w, cin, classes = FEW[i]
    g = torch.Generator("cuda").manual_seed(90 + i)
    x = image(g, (b, cin, h, w), F32, layout)
    weight, bias = classifier(g, classes, cin, F32)
    target = labels(g, (b, h, w), classes, 0.2)
    x = torch.where((target == -100)[:, None], torch.full_like(x, float("nan")), x)
    x = x.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else x.contiguous()
    grad = torch.tensor(1.3, device="cuda")
    for mean in (True, False):
        loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
        got = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean)
        assert layout_kept(got[0], layout)
        R.check(dict(zip(("loss", "gx", "gw", "gb"), [loss] + got)), R.cross_entropy(x, weight, bias, target, -100, mean, grad), str(FEW[i]))
        again = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, mean)
        assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("batch,height,width,classes,dtype", [
    (3, 1, 90_000, 2562, BF),   # bf16: score gradients of more than one piece, whole images and part of one
    (1, 1, 250_000, 2562, BF),
    (2, 1, 300_000, 130, F32),  # float32: scores of more than one piece
    (3, 1, 200_000, 100, F32),
    (2, 1, 300_000, 640, F32),  # and on the tensor cores
    (3, 1, 100_000, 640, F32)])
@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
def test_more_than_the_workspace_holds(ops, layout, batch, height, width, classes, dtype):
    """bf16: a gigabyte of score gradients at a time; float32: a quarter of one.  Checked against the same call in parts."""
    g = torch.Generator("cuda").manual_seed(31)
    x = image(g, (batch, 8, height, width), dtype, layout)
    weight, bias = classifier(g, classes, 8, dtype)
    target = labels(g, (batch, height, width), classes, 0.1)
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, False)
    total, w_sum, b_sum, u = 0.0, 0.0, 0.0, torch.finfo(dtype).eps / 2
    # float32: the whole takes the tensor cores, its parts may not; the exponentials and logarithms of either are within 2^-19
    # (step_reference), and so are a pixel's loss, its probabilities and what is made of them
    apart = 2 * 2.0 ** -19 if dtype == F32 else 0.0
    for i in range(batch):
        for k in range(0, width, 30_000):
            part = x[i:i + 1, :, :, k:k + 30_000]
            part = part.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else part.contiguous()
            some = target[i:i + 1, :, k:k + 30_000].contiguous()
            one, kept = ops.cross_entropy_forward(part, weight, bias, some, -100, False)
            px, pw, pb = ops.cross_entropy_backward(grad, kept, part, weight, bias, some, -100, False)
            # (tiles of another width: other orders of the sums)
            assert (gx[i:i + 1, :, :, k:k + 30_000].double() - px).norm() <= (2 * u + apart) * px.double().norm()
            total, w_sum, b_sum = total + one.double(), w_sum + pw.double(), b_sum + pb.double()
    n = batch * ((width + 29_999) // 30_000)
    assert abs(loss.item() - total.item()) <= ((n + 1) * 2.0 ** -24 + apart) * total.item()
    # the parts' sums are rounded n times, the whole once; their elements do not cancel more than the parts' sizes say
    for whole, parts in ((gw, w_sum), (gb, b_sum)):
        assert (whole.double() - parts).norm() <= (n ** 0.5 + 1) * 2 * u * parts.norm() + 2.0 ** -18 * parts.norm()


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("cin", [40, 64, 300])
def test_ignored_pixels_count_nothing_whatever_they_hold(ops, dtype, layout, cin):
    g = torch.Generator("cuda").manual_seed(22)
    x = image(g, (2, cin, 13, 17), dtype, layout)
    weight, bias = classifier(g, 90, cin, dtype)
    target = labels(g, (2, 13, 17), 90, 0.4, 7)
    off = (target == 7)[:, None].expand_as(x)
    grad = torch.tensor(1.0, device="cuda", dtype=F64 if dtype == F64 else F32)
    want = None
    for value in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max):
        x = torch.where(off, torch.full_like(x, value), x)
        x = x.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else x.contiguous()
        loss, saved = ops.cross_entropy_forward(x, weight, bias, target, 7)
        got = [loss] + ops.cross_entropy_backward(grad, saved, x, weight, bias, target, 7)
        assert not got[1][off].any() and all(t.isfinite().all() for t in got)
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
def test_no_label_at_all(ops, dtype):
    g = torch.Generator("cuda").manual_seed(23)
    x = image(g, (2, 24, 5, 7), dtype, "nhwc")
    weight, bias = classifier(g, 30, 24, dtype)
    target = torch.full((2, 5, 7), -100, device="cuda")
    for mean in (True, False):
        loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
        assert loss.isnan() if mean else loss.item() == 0
        for t in ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target, -100, mean):
            assert not t.any()
    empty = torch.empty(0, 24, 5, 7, device="cuda", dtype=dtype)
    for mean in (True, False):
        loss, saved = ops.cross_entropy_forward(empty, weight, bias, target[:0], -100, mean)
        assert saved is None and (loss.isnan() if mean else loss.item() == 0)
        gx, gw, gb = ops.cross_entropy_backward(torch.ones_like(loss), None, empty, weight, bias, target[:0], -100, mean)
        assert gx.shape == empty.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("label", [-1, 30, 1 << 40, -(1 << 40)])
def test_labels_that_are_no_class(ops, dtype, label):
    g = torch.Generator("cuda").manual_seed(24)
    x = image(g, (2, 24, 5, 7), dtype, "nhwc")
    weight, bias = classifier(g, 30, 24, dtype)
    target = labels(g, (2, 5, 7), 30, 0.0)
    target[1, 2, 3] = label
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    gx, gw, gb = ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target)
    assert loss.isnan() and gw.isnan().all() and gb.isnan().all()
    at = torch.zeros_like(gx, dtype=torch.bool)
    at[1, :, 2, 3] = True
    assert gx[at].isnan().all() and gx[~at].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_large_scores_and_classes_ruled_out(ops, dtype):
    """scores of hundreds neither overflow nor underflow; a bias of -infinity, or of the type's lowest value, takes a class out"""
    g = torch.Generator("cuda").manual_seed(25)
    x = image(g, (1, 32, 9, 20), dtype, "nhwc", 10.0)
    weight, bias = classifier(g, 150, 32, dtype, 30.0)
    target = labels(g, (1, 9, 20), 140, 0.0)
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    got = dict(zip(("gx", "gw", "gb"), ops.cross_entropy_backward(grad, saved, x, weight, bias, target)))
    R.check(dict(loss=loss, **got), R.cross_entropy(x, weight, bias, target, -100, True, grad), "large")
    for low in (-float("inf"), torch.finfo(dtype).min):
        few = bias.clone()
        few[140:] = low
        loss, saved = ops.cross_entropy_forward(x, weight, few, target)
        gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, few, target)
        want = R.cross_entropy(x, weight[:140], bias[:140], target, -100, True, grad)
        R.check(dict(loss=loss, gx=gx, gw=gw[:140], gb=gb[:140]), want, "ruled out")
        assert not gw[140:].any() and not gb[140:].any()
    bias[3] = float("nan")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    assert loss.isnan()


def test_largest_weights_in_parts(ops):
    """float32 values that bf16 would round to infinity"""
    g = torch.Generator("cuda").manual_seed(27)
    x = image(g, (2, 40, 50, 60), F32, "nchw")
    x[:, 5] = 2.0 ** -120
    weight, bias = classifier(g, 130, 40, F32)
    weight[:, 5] = 0
    weight[::7, 5], weight[3::7, 5] = torch.finfo(F32).max, -torch.finfo(F32).max
    target = labels(g, (2, 50, 60), 130, 0.2)
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target)
    want = R.cross_entropy(x, weight, bias, target, -100, True, grad)
    rest = torch.arange(40, device="cuda") != 5  # (that channel's weight gradients are below what float32 holds)
    want["gw"] = tuple(v[:, rest] for v in want["gw"])
    R.check(dict(loss=loss, gx=gx, gw=gw[:, rest], gb=gb), want, "largest")


def test_refusals(ops):
    x = torch.zeros(2, 6, 4, 5, device="cuda")
    w, b, t = torch.zeros(9, 6, 1, device="cuda"), torch.zeros(9, device="cuda"), torch.zeros(2, 4, 5, dtype=torch.int64, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, w, b, t)
    for call, text in [(lambda: ops.cross_entropy_forward(x, w, b, t.int()), "int64"), (lambda: ops.cross_entropy_forward(x, w, b, t[:1]), "shape"),
                       (lambda: ops.cross_entropy_forward(x, w, b[:8], t), "shape"), (lambda: ops.cross_entropy_forward(x, w[:, :5], b, t), "shape"),
                       (lambda: ops.cross_entropy_forward(x, w[:, :, 0], b, t), "3-D"), (lambda: ops.cross_entropy_forward(x, w.double(), b, t), "dtype"),
                       (lambda: ops.cross_entropy_forward(x, w, b, t.cpu()), "CUDA only"),
                       (lambda: ops.cross_entropy_forward(x[:, :, ::2], w, b, t[:, ::2]), "contiguous"),
                       (lambda: ops.cross_entropy_forward(x, w[:0], b[:0], t), "class"),
                       (lambda: ops.cross_entropy_backward(loss.double(), saved, x, w, b, t), "grad_loss"),
                       (lambda: ops.cross_entropy_backward(loss, None, x, w, b, t), "saved"),
                       (lambda: ops.cross_entropy_backward(loss, saved[:64], x, w, b, t), "saved")]:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_layer(dtype):
    g = torch.Generator("cuda").manual_seed(26)
    layer = mnn.PointwiseCrossEntropy(24, 50, ignore_index=3).to("cuda").to(dtype)
    scores = mnn.PointwiseConvolution(24, 50).to("cuda").to(dtype)
    scores.load_state_dict(layer.state_dict())  # the layer that gives the scores themselves
    x = image(g, (3, 24, 10, 11), dtype, "nhwc").requires_grad_(True)
    target = labels(g, (3, 10, 11), 50, 0.2, 3)
    loss = layer(x, target)
    (loss * 2).backward()
    want = R.cross_entropy(x.detach(), layer.weight.detach(), layer.bias.detach(), target, 3, True, torch.tensor(2.0))
    R.check(dict(loss=loss.detach(), gx=x.grad, gw=layer.weight.grad, gb=layer.bias.grad), want, "layer")
    other = torch.nn.functional.cross_entropy(scores(x).double(), target, ignore_index=3)
    assert abs(other.item() - loss.item()) < 2e-2
    with torch.no_grad():
        assert torch.equal(layer(x, target), loss)
    (only,) = torch.autograd.grad(layer(x, target), layer.bias, torch.tensor(2.0, device="cuda"))
    assert torch.equal(only, layer.bias.grad)
    (gx,) = torch.autograd.grad(layer(x, target), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        gx.sum().backward()


def test_gradients_against_differences():
    torch.manual_seed(0)
    layer = mnn.PointwiseCrossEntropy(5, 7, reduction="sum").to("cuda").double()
    x = torch.randn(2, 5, 3, 4, device="cuda", dtype=F64, requires_grad=True)
    target = torch.randint(0, 7, (2, 3, 4), device="cuda")
    target[0, 1] = -100
    assert torch.autograd.gradcheck(lambda t, w, b: torch.func.functional_call(layer, dict(weight=w, bias=b), (t, target)),
                                    (x, layer.weight, layer.bias))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_captured_calls_and_streams(dtype):
    g = torch.Generator("cuda").manual_seed(27)
    layer = mnn.PointwiseCrossEntropy(64, 300).to("cuda").to(dtype)
    x, target = image(g, (2, 64, 20, 30), dtype, "nhwc").requires_grad_(True), labels(g, (2, 20, 30), 300, 0.1)

    def step():
        loss = layer(x, target)
        return [loss.detach()] + list(torch.autograd.grad(loss, [x, layer.weight, layer.bias]))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        x.copy_(image(g, x.shape, dtype, "nhwc"))
        target.copy_(labels(g, (2, 20, 30), 300, 0.3))
    for graph, _ in graphs * 2:
        graph.replay()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
