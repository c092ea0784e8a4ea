"""GPU: the classification loss of pixels whose label is nearly certain, or certain, against the formulas in 64 bits.

Scores are exact here: one product of bf16 numbers each, with few bits, in every type and on every path.  What is left are the roundings
of exponentials, of their sum next to one (2^-24 a step) and of its logarithm."""
import pytest
import torch

from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def loss_type(dtype):
    return F64 if dtype == F64 else F32


# (pixels, channels, classes): CUDA cores with classes in registers and in memory, tensor cores with one tile of classes and with many
SIZES = [(200, 16, 20), (300, 24, 200), (3300, 64, 40), (700, 64, 1000), (1500, 40, 2562), (40_962, 64, 50)]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_confident_pixels(ops, i, dtype, layout):
    """Pixel p has 64 in channel p modulo channels; that channel's weights give its label a score of 50 to 100 in steps of a half and the
    others one that is 4 to 60 less.  Losses from 1e-1 to 1e-26 and gradients as small come out to some 2^-24 of one - a sum of exponentials is
    rounded at one each time when 32 classes join those of the label, and a few times when threads' and tiles' sums do - and, for what
    they are beyond that, to 2^-18 of themselves (exponential and logarithm; gradients are rounded to their type, bf16 twice)."""
    pixels, channels, classes = SIZES[i]
    g = torch.Generator("cuda").manual_seed(i)
    x = torch.zeros(1, channels, 1, pixels, device="cuda")
    at = torch.arange(pixels, device="cuda") % channels
    x[0, at, 0, torch.arange(pixels, device="cuda")] = 64.0
    best = torch.randint(0, classes, (channels,), generator=g, device="cuda")
    high = torch.randint(100, 200, (channels,), generator=g, device="cuda") * 0.5
    below = torch.randint(8, 40, (channels,), generator=g, device="cuda") * 0.5  # the nearest score's distance
    z = high - below - torch.randint(0, 80, (classes, channels), generator=g, device="cuda") * 0.5
    z[best, torch.arange(channels, device="cuda")] = high
    weight = (z / 64.0).to(dtype)[:, :, None].contiguous()
    assert torch.equal(weight[:, :, 0].double() * 64, z.double())
    bias = torch.zeros(classes, device="cuda", dtype=dtype)
    x = x.to(dtype)
    x = x.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else x
    target = best[at].view(1, 1, pixels)
    grad = torch.ones((), device="cuda", dtype=loss_type(dtype))
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, False)
    d = (z - high).double()
    others = d.exp()
    others[best, torch.arange(channels, device="cuda")] = 0.0
    rest = others.sum(0)
    each = torch.log1p(rest)[at]
    step = 2.0 ** -53 if dtype == F64 else 2.0 ** -24
    near, own = (classes / 32 + 8) * step, 2.0 ** -18
    assert loss.item() >= 0 and abs(loss.item() - each.sum().item()) <= pixels * near + own * each.sum().item() + 2.0 ** -24 * each.sum().item()
    p = others / (1 + rest)
    gz = p[:, at]
    gz[best[at], torch.arange(pixels, device="cuda")] = -(rest / (1 + rest))[at]
    u = 2 * torch.finfo(dtype).eps if dtype == BF else 2 * step  # (gz and the sum)
    bound = lambda t, m: near * m + (own + u) * t  # noqa: E731
    hot = torch.zeros_like(gz)
    hot[best[at], torch.arange(pixels, device="cuda")] = 1.0  # labels: within `near` of one
    got = gb.double()
    assert ((got - gz.sum(1)).abs() <= bound(gz.abs().sum(1), hot.sum(1)) + 2.0 ** -100).all()
    # a class's own pixels pull, all others push
    mine = torch.bincount(best[at], minlength=classes)
    assert (got[mine == 0] >= 0).all() and (got[mine == pixels] <= 0).all()
    want = gz.T @ weight[:, :, 0].double()
    size, label = gz.T.abs() @ weight[:, :, 0].double().abs(), weight[:, :, 0].double()[best[at]].abs()
    # (gx: sums over the classes, whose accumulators lose up to 2^-23 of what they hold for every sixteen)
    lost = classes / 16 * 2 * step * size
    assert ((gx[0, :, 0].T.double() - want).abs() <= bound(size, label) + lost + 2.0 ** -100).all()


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("pixels,channels", [(50, 20), (3300, 1000), (2600, 1024)])
def test_one_class(ops, dtype, pixels, channels):
    """there is nothing to learn: loss and gradients are zero, whatever the scores are"""
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(1, channels, 1, pixels, generator=g, device="cuda").to(dtype)
    weight, bias = torch.randn(1, channels, 1, generator=g, device="cuda").to(dtype), torch.randn(1, generator=g, device="cuda").to(dtype)
    target = torch.zeros(1, 1, pixels, dtype=torch.int64, device="cuda")
    target[0, 0, ::7] = -100
    for mean in (True, False):
        loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
        assert loss.item() == 0
        for t in ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target, -100, mean):
            assert not t.any()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("pixels,channels,classes", [(100, 8, 30), (90, 8, 300), (3000, 64, 40), (900, 40, 1000)])
def test_all_classes_at_the_lowest_value(ops, dtype, pixels, channels, classes):
    """a bias of the type's lowest value on every class leaves them as they are among each other: uniform, as zero features make them"""
    low = torch.finfo(dtype).min
    x = torch.zeros(1, channels, 1, pixels, device="cuda", dtype=dtype)
    weight, bias = torch.zeros(classes, channels, 1, device="cuda", dtype=dtype), torch.full((classes,), low, device="cuda", dtype=dtype)
    target = torch.arange(pixels, device="cuda").view(1, 1, -1) % classes
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target)
    gx, gw, gb = ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target)
    want = torch.full((classes,), 1.0 / classes, device="cuda", dtype=F64) - torch.bincount(target.view(-1), minlength=classes) / pixels
    assert abs(loss.item() - torch.tensor(float(classes)).log().item()) <= 2.0 ** -18 * loss.item()
    assert not gx.any() and not gw.any()
    u = torch.finfo(dtype).eps
    assert ((gb.double() - want).abs() <= (2.0 ** -18 + 2 * u) * (1.0 / classes + torch.bincount(target.view(-1), minlength=classes) / pixels)).all()
