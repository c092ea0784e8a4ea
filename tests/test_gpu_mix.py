"""GPU: pointwise layer and gated feed-forward block against the same formulas in 64 bits."""
import math

import pytest
import torch

import mix_reference as R
from mappedconvolutions_b200 import host, ops as twin
from mappedconvolutions_b200 import nn as mnn

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def image(g, shape, dtype, layout, scale=1.0):
    t = (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


def params(g, n_out, n_in, dtype):
    s = 1 / math.sqrt(n_in)
    u = lambda *shape: ((torch.rand(shape, generator=g, device="cuda") * 2 - 1) * s).to(dtype)
    return u(n_out, n_in, 1), u(n_out)


def layout_kept(t, layout):
    return t.is_contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t.is_contiguous()


# (batch, height, width, channels in, hidden, channels out): single values, odd counts, tile edges and one past them,
# more than one tile in every direction
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 3, 5, 3, 5, 7), (1, 1, 642, 64, 64, 64), (3, 11, 13, 50, 43, 99), (2, 8, 16, 128, 128, 256),
          (1, 9, 57, 200, 264, 136), (2, 1, 129, 257, 131, 65), (1, 1, 3, 24, 520, 8), (5, 16, 24, 8, 16, 40),
          (1, 25, 41, 512, 96, 24), (2, 40, 52, 72, 320, 328)]
ACT_OF = [None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_pointwise(ops, i, dtype, layout):
    b, h, w, cin, _, cout = SHAPES[i]
    g = torch.Generator("cuda").manual_seed(i)
    x, gy = image(g, (b, cin, h, w), dtype, layout), image(g, (b, cout, h, w), dtype, layout, 0.01)
    r = image(g, (b, cout, h, w), dtype, layout) if i % 2 else None
    weight, bias = params(g, cout, cin, dtype)
    for name in {ACT_OF[i % 6], ACT_OF[(i + 3) % 6]}:
        want = R.pointwise(x, weight, bias, r, name, gy)
        y, saved = ops.pointwise_forward(x, weight, bias, r, R.ACTS[name], True)
        y2, none = ops.pointwise_forward(x, weight, bias, r, R.ACTS[name], False)
        assert none is None and torch.equal(y, y2) and layout_kept(y, layout)
        gx, gw, gb = ops.pointwise_backward(gy, saved, x, weight, bias, R.ACTS[name])
        assert layout_kept(gx, layout)
        R.check(dict(y=y, gx=gx, gw=gw, gb=gb), want, str((SHAPES[i], name)))
        again = ops.pointwise_backward(gy, saved, x, weight, bias, R.ACTS[name])
        assert all(torch.equal(p, q) for p, q in zip((gx, gw, gb), again))  # fixed order of every sum
        only_x = ops.pointwise_backward(gy, saved, x, weight, bias, R.ACTS[name], True, False)
        only_w = ops.pointwise_backward(gy, saved, x, weight, bias, R.ACTS[name], False, True)
        assert torch.equal(only_x[0], gx) and only_x[1] is None and only_w[0] is None and torch.equal(only_w[1], gw)


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_gated(ops, i, dtype, layout):
    b, h, w, cin, hidden, cout = SHAPES[i]
    g = torch.Generator("cuda").manual_seed(100 + i)
    x, gy = image(g, (b, cin, h, w), dtype, layout), image(g, (b, cout, h, w), dtype, layout, 0.01)
    r = image(g, (b, cout, h, w), dtype, layout) if i % 2 == 0 else None
    wi, bi = params(g, 2 * hidden, cin, dtype)
    wo, bo = params(g, cout, hidden, dtype)
    for name in {ACT_OF[(i + 4) % 6], ACT_OF[(i + 1) % 6]}:
        want = R.gated(x, wi, bi, wo, bo, r, name, gy)
        y, saved = ops.gated_forward(x, wi, bi, wo, bo, r, R.ACTS[name], True)
        y2, none = ops.gated_forward(x, wi, bi, wo, bo, r, R.ACTS[name], False)
        assert none is None and torch.equal(y, y2) and layout_kept(y, layout)
        grads = ops.gated_backward(gy, saved, x, wi, bi, wo, R.ACTS[name])
        assert layout_kept(grads[0], layout)
        names = ("gx", "gw_in", "gb_in", "gw_out", "gb_out")
        R.check(dict(zip(names, grads), y=y), want, str((SHAPES[i], name)))
        again = ops.gated_backward(gy, saved, x, wi, bi, wo, R.ACTS[name])
        assert all(torch.equal(p, q) for p, q in zip(grads, again))
        only_x = ops.gated_backward(gy, saved, x, wi, bi, wo, R.ACTS[name], True, False)
        only_w = ops.gated_backward(gy, saved, x, wi, bi, wo, R.ACTS[name], False, True)
        assert torch.equal(only_x[0], grads[0]) and only_x[1:] == [None] * 4 and only_w[0] is None
        assert all(torch.equal(p, q) for p, q in zip(grads[1:], only_w[1:]))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_many_pixels(dtype):
    """more tiles than a wave of blocks holds, and shares of the parameter gradients that end inside a tile"""
    b, h, w, cin, hidden, cout = 3, 200, 301, 16, 24, 8
    g = torch.Generator("cuda").manual_seed(7)
    x, gy = image(g, (b, cin, h, w), dtype, "nhwc"), image(g, (b, cout, h, w), dtype, "nhwc", 0.01)
    wi, bi = params(g, 2 * hidden, cin, dtype)
    wo, bo = params(g, cout, hidden, dtype)
    y, saved = host.impl.gated_forward(x, wi, bi, wo, bo, None, 4, True)
    grads = host.impl.gated_backward(gy, saved, x, wi, bi, wo, 4)
    R.check(dict(zip(("gx", "gw_in", "gb_in", "gw_out", "gb_out"), grads), y=y), R.gated(x, wi, bi, wo, bo, None, "silu", gy))


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
def test_many_channels(layout):
    """rows longer than a block's shared memory, odd in length, and more channel tiles than pairs of blocks"""
    g = torch.Generator("cuda").manual_seed(9)
    cin, cout = 1501, 9003
    x, gy = image(g, (2, cin, 3, 5), BF, layout), image(g, (2, cout, 3, 5), BF, layout, 0.01)
    weight, bias = params(g, cout, cin, BF)
    y, saved = host.impl.pointwise_forward(x, weight, bias, None, 4, True)
    g3 = host.impl.pointwise_backward(gy, saved, x, weight, bias, 4)
    R.check(dict(zip(("gx", "gw", "gb"), g3), y=y), R.pointwise(x, weight, bias, None, "silu", gy))


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("shape", [(3000, 2, 3), (70_000, 1, 2), (5, 1, 1), (2, 40, 64)])
def test_many_small_images(shape, layout, dtype):
    """more images than a grid's last dimension, images smaller than a tile, single pixels"""
    b, h, w = shape
    g = torch.Generator("cuda").manual_seed(8)
    x, gy = image(g, (b, 6, h, w), dtype, layout), image(g, (b, 5, h, w), dtype, layout, 0.01)
    r = image(g, (b, 5, h, w), dtype, layout)
    weight, bias = params(g, 5, 6, dtype)
    y, saved = host.impl.pointwise_forward(x, weight, bias, r, 4, True)
    g3 = host.impl.pointwise_backward(gy, saved, x, weight, bias, 4)
    R.check(dict(zip(("gx", "gw", "gb"), g3), y=y), R.pointwise(x, weight, bias, r, "silu", gy))
    wi, bi = params(g, 16, 6, dtype)
    wo, bo = params(g, 5, 8, dtype)
    y, saved = host.impl.gated_forward(x, wi, bi, wo, bo, r, 4, True)
    g5 = host.impl.gated_backward(gy, saved, x, wi, bi, wo, 4)
    R.check(dict(zip(("gx", "gw_in", "gb_in", "gw_out", "gb_out"), g5), y=y), R.gated(x, wi, bi, wo, bo, r, "silu", gy))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_layers_and_their_gradients(dtype):
    """two layers as a block would chain them, through autograd, against the chained formulas"""
    g = torch.Generator("cuda").manual_seed(3)
    p = mnn.PointwiseConvolution(24, 40, activation="gelu").cuda().to(dtype)
    f = mnn.GatedFeedForward(40, 72, activation="silu").cuda().to(dtype)
    x = image(g, (2, 24, 9, 17), dtype, "nhwc").requires_grad_(True)
    y1 = p(x)
    y1.retain_grad()
    y2 = f(y1, y1)  # the block's input is its residual
    gy = image(g, y2.shape, dtype, "nhwc", 0.01)
    y2.backward(gy)
    R.check(dict(y=y1), R.pointwise(x, p.weight, p.bias, None, "gelu"))
    want = R.gated(y1, f.weight_in, f.bias_in, f.weight_out, f.bias_out, y1, "silu", gy)
    R.check(dict(y=y2, gw_in=f.weight_in.grad, gb_in=f.bias_in.grad, gw_out=f.weight_out.grad, gb_out=f.bias_out.grad), want)
    value, bound = want["gx"]  # autograd adds the residual's gradient in the tensors' type
    total = value + gy.double()
    R.check(dict(g1=y1.grad), dict(g1=(total, bound + torch.finfo(dtype).eps / 2 * (total.abs() + bound))))
    want = R.pointwise(x, p.weight, p.bias, None, "gelu", y1.grad)
    R.check(dict(gx=x.grad, gw=p.weight.grad, gb=p.bias.grad), want)


@pytest.mark.parametrize("layer", ["pointwise", "gated"])
def test_gradients_are_differences(layer):
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(2, 3, 4, 5, generator=g, device="cuda", dtype=F64).requires_grad_(True)
    r = torch.randn(2, 6, 4, 5, generator=g, device="cuda", dtype=F64).requires_grad_(True)
    for name in ("gelu", "gelu_tanh", "silu", "sigmoid", None):
        m = mnn.PointwiseConvolution(3, 6, activation=name) if layer == "pointwise" else \
            mnn.GatedFeedForward(3, 4, 6, activation=name)
        m = m.cuda().double()
        names = [n for n, _ in m.named_parameters()]
        call = lambda x, r, *ps: torch.func.functional_call(m, dict(zip(names, ps)), (x, r))
        assert torch.autograd.gradcheck(call, (x, r, *m.parameters()))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_only_what_is_needed_is_computed(dtype):
    m = mnn.GatedFeedForward(16, 32).cuda().to(dtype)
    x = torch.randn(2, 16, 5, 7, device="cuda").to(dtype)
    m.bias_out.requires_grad_(False)
    m(x).sum().backward()
    assert m.weight_in.grad is not None and m.bias_out.grad is None
    m.requires_grad_(False)
    r = torch.zeros(2, 16, 5, 7, device="cuda", dtype=dtype, requires_grad=True)
    m(x, r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))
    with torch.no_grad():
        assert not m(x, r).requires_grad


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("shape", [(0, 16, 4, 4), (2, 16, 0, 4)])
def test_no_pixels(ops, shape, dtype):
    x = torch.empty(shape, device="cuda", dtype=dtype)
    w, b = torch.ones(8, 16, 1, device="cuda", dtype=dtype), torch.ones(8, device="cuda", dtype=dtype)
    y, saved = ops.pointwise_forward(x, w, b, None, 1, True)
    assert y.shape == (shape[0], 8, *shape[2:])
    gx, gw, gb = ops.pointwise_backward(y, saved, x, w, b, 1)
    assert gx.shape == x.shape and not gw.any() and not gb.any()
    wi, bi = torch.ones(8, 16, 1, device="cuda", dtype=dtype), torch.ones(8, device="cuda", dtype=dtype)
    wo, bo = torch.ones(16, 4, 1, device="cuda", dtype=dtype), torch.ones(16, device="cuda", dtype=dtype)
    y, saved = ops.gated_forward(x, wi, bi, wo, bo, None, 4, True)
    assert y.shape == shape
    assert not any(t.any() for t in ops.gated_backward(y, saved, x, wi, bi, wo, 4)[1:])


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
def test_infinities_and_nan_stay_in_their_pixel(ops, dtype, layout):
    """and the channels behind them are what the formulas give for such values"""
    g = torch.Generator("cuda").manual_seed(11)
    x = image(g, (2, 20, 6, 50), dtype, layout)
    clean = x.clone(memory_format=torch.preserve_format)
    x[0, 3, 2, 7], x[1, 19, 5, 49] = float("nan"), float("inf")
    w, b = params(g, 33, 20, dtype)
    wi, bi = params(g, 2 * 24, 20, dtype)
    wo, bo = params(g, 33, 24, dtype)
    for run in (lambda t: ops.pointwise_forward(t, w, b, None, 1)[0], lambda t: ops.gated_forward(t, wi, bi, wo, bo, None, 1)[0]):
        y, y0 = run(x), run(clean)
        touched = torch.zeros(2, 1, 6, 50, dtype=torch.bool, device="cuda")
        touched[0, 0, 2, 7] = touched[1, 0, 5, 49] = True
        assert torch.equal(torch.where(touched, 0, y), torch.where(touched, 0, y0))
        assert y[0, :, 2, 7].isnan().all()
    z = (x.double()[1, :, 5, 49][None] * w.double()[:, :, 0]).sum(1) + b.double()
    y = ops.pointwise_forward(x, w, b, None, 1)[0][1, :, 5, 49].double()
    assert torch.equal(y.isinf(), z == float("inf")) and torch.equal(y == 0, z == -float("inf"))


def test_views_that_start_anywhere(ops):
    """batch slices of tensors whose images are not whole 16-byte groups, and parameters cut out of one buffer"""
    g = torch.Generator("cuda").manual_seed(12)
    for dtype in (BF, F32):
        for layout in ("nhwc", "nchw"):
            x = image(g, (3, 5, 3, 7), dtype, layout)[1:]
            gy = image(g, (3, 9, 3, 7), dtype, layout)[1:]
            r = image(g, (3, 9, 3, 7), dtype, layout)[1:]
            flat = torch.randn(1 + 45 + 9 + 60 + 12 + 54 + 9, generator=g, device="cuda").to(dtype)
            w, b = flat[1:46].view(9, 5, 1), flat[46:55]
            wi, bi = flat[55:115].view(12, 5, 1), flat[115:127]
            wo, bo = flat[127:181].view(9, 6, 1), flat[181:190]
            y, saved = ops.pointwise_forward(x, w, b, r, 2, True)
            g3 = ops.pointwise_backward(gy, saved, x, w, b, 2)
            R.check(dict(zip(("gx", "gw", "gb"), g3), y=y), R.pointwise(x, w, b, r, "gelu", gy))
            y, saved = ops.gated_forward(x, wi, bi, wo, bo, r, 2, True)
            g5 = ops.gated_backward(gy, saved, x, wi, bi, wo, 2)
            R.check(dict(zip(("gx", "gw_in", "gb_in", "gw_out", "gb_out"), g5), y=y), R.gated(x, wi, bi, wo, bo, r, "gelu", gy))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_gradients_in_any_layout(dtype):
    """what stands behind the layer hands back expanded, transposed or otherwise strided gradients and residuals"""
    g = torch.Generator("cuda").manual_seed(13)
    m = mnn.PointwiseConvolution(8, 16, activation="silu").cuda().to(dtype)
    for layout in ("nhwc", "nchw"):
        x = image(g, (2, 8, 4, 6), dtype, layout).requires_grad_(True)
        for gy in (torch.ones((), device="cuda", dtype=dtype).expand(2, 16, 4, 6),
                   image(g, (2, 16, 6, 4), dtype, "nchw").transpose(2, 3), image(g, (2, 16, 4, 6), dtype, "nhwc"),
                   image(g, (2, 16, 4, 12), dtype, "nchw")[..., ::2]):
            r = image(g, (2, 16, 6, 4), dtype, "nchw").transpose(2, 3)
            m.zero_grad()
            x.grad = None
            y = m(x, r)
            y.backward(gy)
            R.check(dict(y=y, gx=x.grad, gw=m.weight.grad, gb=m.bias.grad), R.pointwise(x, m.weight, m.bias, r, "silu", gy))


def test_refusals(ops):
    x = torch.randn(2, 8, 4, 6, device="cuda")
    w, b = torch.randn(16, 8, 1, device="cuda"), torch.randn(16, device="cuda")
    r = torch.randn(2, 16, 4, 6, device="cuda")
    ops.pointwise_forward(x, w, b, r, 1)
    for args in [(x[0], w, b, r), (x, w[:, :4], b, r), (x, w, b[:8], r), (x, w.double(), b, r), (x, w, b.double(), r),
                 (x, w, b, r[:1]), (x, w, b, r.double()), (x.cpu(), w, b, r), (x, w.cpu(), b, r), (x, w[:, :, 0], b, r),
                 (x.transpose(2, 3), w, b, r.transpose(2, 3)), (x.half(), w.half(), b.half(), r.half()),
                 (x, w.expand(16, 8, 1).transpose(0, 1), b, r), (x, w, torch.ones(1, device="cuda").expand(16), r)]:
        with pytest.raises(RuntimeError):
            ops.pointwise_forward(*args, 1)
    for act in (-1, 6):
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.pointwise_forward(x, w, b, r, act)
    with pytest.raises(RuntimeError):  # needs what the forward call kept
        ops.pointwise_backward(r, None, x, w, b, 1)
    with pytest.raises(RuntimeError):
        ops.pointwise_backward(r[:, :8], None, x, w, b, 0)
    wi, bi = torch.randn(24, 8, 1, device="cuda"), torch.randn(24, device="cuda")
    wo, bo = torch.randn(16, 12, 1, device="cuda"), torch.randn(16, device="cuda")
    ops.gated_forward(x, wi, bi, wo, bo, r)
    for args in [(x, wi[:12], bi[:12], wo, bo, r), (x, wi, bi[:12], wo, bo, r), (x, wi, bi, wo[:, :6], bo, r),
                 (x, wi, bi, wo, bo[:3], r), (x, wi.double(), bi, wo, bo, r), (x, wi, bi, wo, bo, r[..., :3])]:
        with pytest.raises(RuntimeError):
            ops.gated_forward(*args)
    with pytest.raises(RuntimeError):
        ops.gated_backward(r, None, x, wi, bi, wo)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_backward_refuses_what_another_forward_call_kept(ops, dtype):
    t = lambda *shape: torch.randn(*shape, device="cuda").to(dtype)
    x, w, b, gy = t(2, 7, 4, 6), t(16, 7, 1), t(16), t(2, 16, 4, 6)
    wi, bi, wo, bo = t(24, 7, 1), t(24), t(16, 12, 1), t(16)
    one = ops.pointwise_forward(x, w, b, None, 1, True)[1]
    two = ops.gated_forward(x, wi, bi, wo, bo, None, 4, True)[1]
    few = ops.pointwise_forward(x[:1], w, b, None, 1, True)[1]
    for bad in (None, few, one[:-1], one.float(), one.view(-1, 2)[:, 0]):
        with pytest.raises(RuntimeError, match="saved must be"):
            ops.pointwise_backward(gy, bad, x, w, b, 1)
    for bad in (None, one, two[:-1], two.double()):
        with pytest.raises(RuntimeError, match="saved must be"):
            ops.gated_backward(gy, bad, x, wi, bi, wo, 4)
    ops.pointwise_backward(gy, one, x, w, b, 1)
    ops.gated_backward(gy, two, x, wi, bi, wo, 4)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_captured_step(dtype):
    """forward and backward in a graph, replayed on other data.  (No eager graph of the same leaves is alive: torch's
    AccumulateGrad nodes would then belong to the default stream, which a capture must not touch, whatever the layer.)"""
    g = torch.Generator("cuda").manual_seed(17)
    p = mnn.PointwiseConvolution(12, 32, activation="relu").cuda().to(dtype)
    f = mnn.GatedFeedForward(32, 48).cuda().to(dtype)
    x, gy = image(g, (2, 12, 8, 24), dtype, "nhwc"), image(g, (2, 32, 8, 24), dtype, "nhwc", 0.1)
    leaves = list(p.parameters()) + list(f.parameters())
    x.requires_grad_(True)

    def step():
        h = p(x)
        y = f(h, h)
        return [y] + list(torch.autograd.grad(y, [x] + leaves, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        gg = torch.Generator("cuda").manual_seed(seed)
        with torch.no_grad():
            x.copy_(image(gg, x.shape, dtype, "nhwc"))
            gy.copy_(image(gg, gy.shape, dtype, "nhwc", 0.1))
        graph.replay()
        captured = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_other_streams():
    """two calls at once on two streams, each with scratch memory of its own"""
    g = torch.Generator("cuda").manual_seed(19)
    m = mnn.GatedFeedForward(64, 128).cuda().to(BF)
    xs = [image(g, (4, 64, 60, 64), BF, "nhwc") for _ in range(2)]
    want = [m(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = m(xs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_first_cuda_call_of_a_thread():
    """with all memory cached, the tensor maps of a call are the first thing that its thread asks the driver for"""
    import threading
    g = torch.Generator("cuda").manual_seed(20)
    x, (w, b) = image(g, (2, 64, 8, 16), BF, "nhwc"), params(g, 64, 64, BF)
    want = host.impl.pointwise_forward(x, w, b, None, 1)[0].clone()
    got = []
    torch.cuda.synchronize()

    def call():
        try:
            got.append(host.impl.pointwise_forward(x, w, b, None, 1)[0])
        except RuntimeError as e:
            got.append(e)
    for _ in range(2):
        t = threading.Thread(target=call)
        t.start()
        t.join()
    assert all(isinstance(y, torch.Tensor) and torch.equal(y, want) for y in got), got


def test_offsets_beyond_32_bits():
    """an activation of more than 2^32 bytes and 2^31 elements: its last pixels"""
    n, cin, cout = 35_000_001, 64, 8
    x = torch.zeros(1, cin, 1, n, device="cuda", dtype=BF, ).contiguous(memory_format=torch.channels_last)
    g = torch.Generator("cuda").manual_seed(23)
    x[..., -300:] = torch.randn(1, cin, 1, 300, generator=g, device="cuda").to(BF)
    w, b = params(g, cout, cin, BF)
    y, saved = host.impl.pointwise_forward(x, w, b, None, 1, True)
    tail = x[..., -300:].contiguous(memory_format=torch.channels_last)
    R.check(dict(y=y[..., -300:]), R.pointwise(tail, w, b, None, "relu"))
    gy = torch.zeros_like(y)
    gy[..., -300:] = torch.randn(1, cout, 1, 300, generator=g, device="cuda").to(BF)
    gx, gw, gb = host.impl.pointwise_backward(gy, saved, x, w, b, 1)
    want = R.pointwise(tail, w, b, None, "relu", gy[..., -300:])
    R.check(dict(gx=gx[..., -300:], gw=gw, gb=gb), want)
    assert not gx[..., :-300].any()
