"""GPU: group normalisation with an activation against the same formulas in 64 bits."""
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


def image(g, shape, dtype, layout, scale=1.0, offset=0.0):
    t = (torch.randn(shape, generator=g, device="cuda") * scale + offset).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


def layout_kept(t, layout):
    return t.is_contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t.is_contiguous()


# (batch, height, width, channels, groups): one value to a group, odd counts, groups that end inside a vector, images that do
# not start on 16 bytes, more vectors than threads, several tiles and segments to an image
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 1, 6, 3), (2, 3, 5, 7, 7), (3, 5, 7, 12, 4), (1, 1, 642, 64, 8), (2, 11, 13, 50, 10),
          (2, 16, 24, 96, 8), (1, 9, 57, 200, 25), (5, 7, 9, 13, 13), (2, 3, 3, 2056, 8), (1, 2, 3, 257, 1), (2, 70, 70, 24, 3),
          (1, 125, 251, 32, 4), (65, 2, 4, 16, 2), (1, 1, 40962, 8, 2)]
ACT_OF = [None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_forward_and_backward(ops, i, dtype, layout):
    b, h, w, c, groups = SHAPES[i]
    g = torch.Generator("cuda").manual_seed(i)
    x, gy = image(g, (b, c, h, w), dtype, layout, 2.0, 0.5), image(g, (b, c, h, w), dtype, layout, 0.01)
    weight, bias = (torch.randn(c, generator=g, device="cuda").to(dtype) for _ in range(2))
    for name in {ACT_OF[i % 6], ACT_OF[(i + 3) % 6]}:
        want = R.group_norm(x, weight, bias, groups, 1e-5, name, gy)
        y, stats = ops.group_norm_forward(x, weight, bias, groups, 1e-5, R.ACTS[name])
        gx, gw, gb = ops.group_norm_backward(gy, stats, x, weight, bias, groups, 1e-5, R.ACTS[name])
        assert layout_kept(y, layout) and layout_kept(gx, layout)
        R.check(dict(y=y, gx=gx, gw=gw, gb=gb), want, str((SHAPES[i], name)))
        y2, stats2 = ops.group_norm_forward(x, weight, bias, groups, 1e-5, R.ACTS[name])
        again = ops.group_norm_backward(gy, stats2, x, weight, bias, groups, 1e-5, R.ACTS[name])
        assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip((gx, gw, gb), again))  # fixed order of every sum
        only_x = ops.group_norm_backward(gy, stats, x, weight, bias, groups, 1e-5, R.ACTS[name], True, False)
        only_w = ops.group_norm_backward(gy, stats, x, weight, bias, groups, 1e-5, R.ACTS[name], False, True)
        assert torch.equal(only_x[0], gx) and only_x[1] is None and only_w[0] is None and torch.equal(only_w[1], gw)
    plain = R.group_norm(x, None, None, groups, 1e-5, None, gy)
    y, stats = ops.group_norm_forward(x, None, None, groups)
    gx, gw, gb = ops.group_norm_backward(gy, stats, x, None, None, groups)
    assert gw is None and gb is None
    R.check(dict(y=y, gx=gx), plain, "without parameters")


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("offset", [1e3, -1e4])
def test_values_far_from_zero(ops, layout, offset):
    """mean >> deviation: differences, not squares of values, are summed"""
    g = torch.Generator("cuda").manual_seed(3)
    x, gy = image(g, (2, 24, 33, 41), F32, layout, 1.0, offset), image(g, (2, 24, 33, 41), F32, layout)
    w, b = (torch.randn(24, generator=g, device="cuda") for _ in range(2))
    y, stats = ops.group_norm_forward(x, w, b, 4, 1e-5, R.ACTS["silu"])
    got = dict(zip(("gx", "gw", "gb"), ops.group_norm_backward(gy, stats, x, w, b, 4, 1e-5, R.ACTS["silu"])))
    R.check(dict(y=y, **got), R.group_norm(x, w, b, 4, 1e-5, "silu", gy), str(offset))


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_one_large_value_and_constant_groups(ops, dtype, layout):
    g = torch.Generator("cuda").manual_seed(4)
    x = image(g, (2, 16, 30, 40), dtype, layout)
    for at in [(0, 0, 0, 0), (0, 5, 17, 3), (1, 15, 29, 39)]:
        x[at] = 1e4
    x[1, 4:8] = 3.0  # a group without deviation: rstd = 1 / sqrt(eps)
    w, b = (torch.randn(16, generator=g, device="cuda").to(dtype) for _ in range(2))
    gy = image(g, x.shape, dtype, layout)
    y, stats = ops.group_norm_forward(x, w, b, 4, 1e-5, R.ACTS["gelu"])
    got = dict(zip(("gx", "gw", "gb"), ops.group_norm_backward(gy, stats, x, w, b, 4, 1e-5, R.ACTS["gelu"])))
    R.check(dict(y=y, **got), R.group_norm(x, w, b, 4, 1e-5, "gelu", gy), "")


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite_values_stay_in_their_group(ops, dtype, layout, value):
    g = torch.Generator("cuda").manual_seed(5)
    x = image(g, (3, 12, 9, 11), dtype, layout)
    clean, _ = ops.group_norm_forward(x, None, None, 3)
    x[1, 6, 4, 5] = value  # group 1 of image 1
    y, _ = ops.group_norm_forward(x, None, None, 3)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, 4:8] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


def test_views_and_other_layouts(ops):
    g = torch.Generator("cuda").manual_seed(6)
    big = image(g, (4, 5, 7, 3), BF, "nchw")
    w, b = (torch.randn(5, generator=g, device="cuda").to(BF) for _ in range(2))
    x = big[1:3]  # (starts 210 bytes into its memory)
    gy = torch.randn(2, 5, 3, 7, generator=g, device="cuda").to(BF).transpose(2, 3)
    y, stats = ops.group_norm_forward(x, w, b, 5, 1e-3, 1)
    gx, gw, gb = ops.group_norm_backward(gy, stats, x, w, b, 5, 1e-3, 1)
    R.check(dict(y=y, gx=gx, gw=gw, gb=gb), R.group_norm(x, w, b, 5, 1e-3, "relu", gy), "views")
    empty = torch.empty(0, 6, 3, 4, device="cuda")
    y, stats = ops.group_norm_forward(empty, None, None, 2)
    assert y.shape == empty.shape and stats is None
    one = torch.ones(6, device="cuda")
    gx, gw, gb = ops.group_norm_backward(empty, None, empty, one, one, 2)
    assert gx.shape == empty.shape and not gw.any() and not gb.any()


def test_refusals(ops):
    x = torch.zeros(2, 6, 4, 5, device="cuda")
    one = torch.ones(6, device="cuda")
    y, stats = ops.group_norm_forward(x, one, one, 3)
    for call, text in [(lambda: ops.group_norm_forward(x, one, one, 4), "divide"), (lambda: ops.group_norm_forward(x, one, one, 0), "divide"),
                       (lambda: ops.group_norm_forward(x, one[:5], one, 3), "shape"),
                       (lambda: ops.group_norm_forward(x, one.double(), one, 3), "dtype"),
                       (lambda: ops.group_norm_forward(x.half(), None, None, 3), "dtype"),
                       (lambda: ops.group_norm_forward(x[:, :, ::2], None, None, 3), "contiguous"),
                       (lambda: ops.group_norm_forward(x, one, one.cpu(), 3), "CUDA only"),
                       (lambda: ops.group_norm_forward(x, one, one, 3, -1.0), "bad argument"),
                       (lambda: ops.group_norm_forward(x, one, one, 3, 1e-5, 9), "bad argument"),
                       (lambda: ops.group_norm_backward(y, None, x, one, one, 3), "saved"),
                       (lambda: ops.group_norm_backward(y, stats[:8], x, one, one, 3), "saved"),
                       (lambda: ops.group_norm_backward(y[:1], stats, x, one, one, 3), "shape")]:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_layer(dtype, affine):
    g = torch.Generator("cuda").manual_seed(7)
    layer = mnn.GroupNorm(4, 24, 1e-4, affine, activation="silu").to("cuda").to(dtype)
    x = image(g, (3, 24, 10, 11), dtype, "nhwc").requires_grad_(True)
    gy = image(g, x.shape, dtype, "nchw")
    if affine:
        with torch.no_grad():
            layer.weight.normal_(generator=g)
            layer.bias.normal_(generator=g)
    y = layer(x)
    y.backward(gy)
    want = R.group_norm(x.detach(), layer.weight, layer.bias, 4, 1e-4, "silu", gy)
    got = dict(y=y.detach(), gx=x.grad)
    if affine:
        got.update(gw=layer.weight.grad, gb=layer.bias.grad)
    R.check(got, {k: (v[0].detach(), v[1].detach()) for k, v in want.items()}, "layer")
    with torch.no_grad():
        assert torch.equal(layer(x), y)
    for need in ([layer.bias], [x]) if affine else ([x],):
        (only,) = torch.autograd.grad(layer(x), need, gy)
        assert torch.equal(only, need[0].grad)
    (gx,) = torch.autograd.grad(layer(x), x, gy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        gx.sum().backward()


def test_gradients_against_differences():
    torch.manual_seed(0)
    for act in ("gelu", "sigmoid", None):
        layer = mnn.GroupNorm(2, 6, activation=act).to("cuda").double()
        x = torch.randn(2, 6, 3, 4, device="cuda", dtype=F64, requires_grad=True)
        assert torch.autograd.gradcheck(lambda t, w, b: torch.func.functional_call(layer, dict(weight=w, bias=b), (t,)),
                                        (x, layer.weight, layer.bias))


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
def test_captured_calls_and_streams(layout):
    g = torch.Generator("cuda").manual_seed(8)
    layer = mnn.GroupNorm(4, 32, activation="gelu").to("cuda").to(BF)
    x, gy = image(g, (2, 32, 40, 50), BF, layout).requires_grad_(True), image(g, (2, 32, 40, 50), BF, layout)

    def step():
        y = layer(x)
        return [y.detach()] + list(torch.autograd.grad(y, [x, layer.weight, layer.bias], gy))
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
        x.copy_(image(g, x.shape, BF, layout))
    for graph, _ in graphs * 2:
        graph.replay()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
