"""GPU: group norm, the classification loss and AdamW on tensors of more than 2^31 elements."""
import pytest
import torch

import step_reference as R
from mappedconvolutions_b200 import host

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
ops = host.impl


@pytest.fixture(autouse=True)
def memory_is_given_back():
    yield
    torch.cuda.empty_cache()


def filled(g, shape, dtype, layout):
    """random values, made a part at a time"""
    b, c, h, w = shape
    t = torch.empty(shape, dtype=dtype, device="cuda", memory_format=torch.channels_last if layout == "nhwc" else torch.contiguous_format)
    flat = t.permute(0, 2, 3, 1).view(-1) if layout == "nhwc" else t.view(-1)
    for part in flat.split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=dtype))
    return t


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("batch,pixels", [(1, 8_400_003), (5, 1_700_001)])
def test_group_norm(layout, batch, pixels):
    """Groups are independent: the first and the last one are compared with the formulas on their channels alone."""
    g = torch.Generator("cuda").manual_seed(1)
    shape = (batch, 256, 1, pixels)
    assert batch * 256 * pixels > 1 << 31
    x, gy = filled(g, shape, BF, layout), filled(g, shape, BF, layout)
    weight, bias = torch.rand(256, generator=g, device="cuda").to(BF), torch.randn(256, generator=g, device="cuda").to(BF)
    y, stats = ops.group_norm_forward(x, weight, bias, 32, 1e-5, 0)
    gx, gw, gb = ops.group_norm_backward(gy, stats, x, weight, bias, 32, 1e-5, 0)
    for c in (0, 248):
        at = slice(c, c + 8)
        for b in (0, batch - 1):
            want = R.group_norm(x[b:b + 1, at], weight[at], bias[at], 1, 1e-5, None, gy[b:b + 1, at])
            R.check(dict(y=y[b:b + 1, at], gx=gx[b:b + 1, at]), {k: want[k] for k in ("y", "gx")}, (c, b))
        want = R.group_norm(x[:, at], weight[at], bias[at], 1, 1e-5, None, gy[:, at])
        R.check(dict(gw=gw[at], gb=gb[at]), {k: want[k] for k in ("gw", "gb")}, c)


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_cross_entropy(dtype, layout):
    """Losses and parameter gradients that are sums: against those of parts of the pixels; input gradients of the last part."""
    g = torch.Generator("cuda").manual_seed(2)
    pixels, channels, classes = 4_200_100, 512, 16
    assert pixels * channels > 1 << 31
    x = filled(g, (1, channels, 1, pixels), dtype, layout)
    weight = ((torch.rand(classes, channels, 1, generator=g, device="cuda") * 2 - 1) * 0.1).to(dtype)
    bias = torch.randn(classes, generator=g, device="cuda").to(dtype)
    target = torch.randint(0, classes, (1, 1, pixels), generator=g, device="cuda")
    target[torch.rand(1, 1, pixels, generator=g, device="cuda") < 0.1] = -100
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, False)
    total, w_sum, b_sum, n = 0.0, 0.0, 0.0, 0
    for k in range(0, pixels, 1_400_000):
        part = x[..., k:k + 1_400_000]
        part = part.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else part.contiguous()
        some = target[..., k:k + 1_400_000].contiguous()
        one, kept = ops.cross_entropy_forward(part, weight, bias, some, -100, False)
        px, pw, pb = ops.cross_entropy_backward(grad, kept, part, weight, bias, some, -100, False)
        whole = gx[..., k:k + 1_400_000]
        if px.shape[-1] == 1_400_000:  # (the same kernels in the same tiles: a pixel's gradients are the same)
            assert torch.equal(whole, px)
        else:  # 100 pixels: in float32 too few products for the tensor cores; exponentials and logarithms of either are within 2^-19
            assert (whole.double() - px).norm() <= (2 * torch.finfo(dtype).eps / 2 + 2 * 2.0 ** -19) * px.double().norm()
        total, w_sum, b_sum, n = total + one.double(), w_sum + pw.double(), b_sum + pb.double(), n + 1
    u = torch.finfo(dtype).eps / 2
    assert abs(loss.item() - total.item()) <= (n + 1) * 2.0 ** -24 * total.item()
    # the parts' sums are rounded n times, the whole once; either side's accumulators truncate at most 2^-18 of a sum of magnitudes
    # (float32; less than a rounding in bf16), and the magnitudes of so many terms of both signs add up to sqrt(pixels) their sum's
    for whole, parts in ((gw, w_sum), (gb, b_sum)):
        assert (whole.double() - parts).norm() <= ((n ** 0.5 + 1) * 2 * u + 2 * 2.0 ** -18 * pixels ** 0.5) * parts.norm()
    last = slice(pixels - 999, pixels)
    want = R.cross_entropy(x[..., last], weight, bias, target[..., last], -100, False, grad)
    R.check(dict(gx=gx[..., last]), want, "last pixels")


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw(bits):
    """A step of elements is a step of any of them (8 bits: of any block of 256)."""
    n, part = (1 << 31) + 1000, 1 << 20
    g = torch.Generator("cuda").manual_seed(3)
    p, grad = torch.empty(n, dtype=BF, device="cuda"), torch.empty(n, dtype=BF, device="cuda")
    for t in (p, grad):
        for some in t.split(1 << 28):
            some.copy_(torch.randn(some.shape, generator=g, device="cuda", dtype=BF))
    kinds = (torch.int8, torch.uint8) if bits == 8 else (F32, F32)
    m, v = (torch.zeros(n, dtype=k, device="cuda") for k in kinds)
    scales = [torch.zeros((n + 255) // 256, device="cuda") if bits == 8 else None for _ in range(2)]
    parts = []
    for at in (slice(0, part), slice((n - part) // 256 * 256, n)):
        parts.append((at, [t[at].clone() for t in (p, grad, m, v)],
                      [s if s is None else s[at.start // 256:(at.stop + 255) // 256].clone() for s in scales]))
    for step in (1, 2):
        ops.adamw_step([p], [grad], [m], [v], [scales[0]], [scales[1]], [None], [step], 1e-2, 0.9, 0.99, 1e-8, 0.1)
        for at, (q, h, a, b), s in parts:
            ops.adamw_step([q], [h], [a], [b], [s[0]], [s[1]], [None], [step], 1e-2, 0.9, 0.99, 1e-8, 0.1)
            for whole, one in ((p, q), (m, a), (v, b)):
                assert torch.equal(whole[at], one)
