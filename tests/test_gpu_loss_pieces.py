"""GPU: the bf16 classification loss where the softmax sums of its tiles take more than one piece of the pixels."""
import math

import pytest
import torch

from mappedconvolutions_b200 import host

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ops = host.impl


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
def test_a_short_second_piece(layout):
    """A gigabyte holds the sums (8 bytes a tile) of 2^27 / ceil(classes / 64) pixels; the call is compared with the same in parts.

    A part's loss is rounded to float32 once more, and its scores are the same numbers in tiles that may have another width: the sums of
    exponentials are added up in another order, 2^-19 of a pixel's loss at most (exponential and logarithm of either side).
    Gradients are rounded to bf16 once on either side."""
    g = torch.Generator("cuda").manual_seed(41)
    pixels, channels, classes, part = 3_400_000, 8, 2562, 850_000
    first = (1 << 27) // math.ceil(classes / 64) // 256 * 256
    assert first < pixels < 2 * first
    x = torch.randn(1, channels, 1, pixels, generator=g, device="cuda", dtype=BF)
    if layout == "nhwc":
        x = x.contiguous(memory_format=torch.channels_last)
    weight = ((torch.rand(classes, channels, 1, generator=g, device="cuda") * 2 - 1) * 1.4).to(BF)
    bias = ((torch.rand(classes, generator=g, device="cuda") * 2 - 1) * 1.4).to(BF)
    target = torch.randint(0, classes, (1, 1, pixels), generator=g, device="cuda")
    target[torch.rand(1, 1, pixels, generator=g, device="cuda") < 0.1] = -100
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    again, _ = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    assert torch.equal(loss, again)
    gx = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, False, True, False)[0]
    total = 0.0
    for k in range(0, pixels, part):
        some, t = x[..., k:k + part], target[..., k:k + part].contiguous()
        some = some.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else some.contiguous()
        one, kept = ops.cross_entropy_forward(some, weight, bias, t, -100, False)
        px = ops.cross_entropy_backward(grad, kept, some, weight, bias, t, -100, False, True, False)[0]
        assert (gx[..., k:k + part].double() - px).norm() <= (2 * 2.0 ** -8 + 2 * 2.0 ** -19) * px.double().norm()
        total += one.double().item()
    assert abs(loss.item() - total) <= (5 * 2.0 ** -24 + 2 * 2.0 ** -19) * total


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("batch,pixels,classes", [(1, 9_000_003, 32), (3, 3_500_001, 29), (2, 9_000_000, 31)])
def test_few_classes_in_several_pieces(layout, batch, pixels, classes):
    """Score gradients of 128 bytes a pixel, two parts of 32 classes: 2^23 pixels to a gigabyte.  Whole images to a piece, or part of one;
    compared with the same call in parts, whose parameter gradients are rounded to bf16 once each."""
    g = torch.Generator("cuda").manual_seed(42)
    channels, part = 8, 3_000_000
    x = torch.randn(batch, channels, 1, pixels, generator=g, device="cuda", dtype=BF)
    if layout == "nhwc":
        x = x.contiguous(memory_format=torch.channels_last)
    weight = ((torch.rand(classes, channels, 1, generator=g, device="cuda") * 2 - 1) * 1.4).to(BF)
    bias = ((torch.rand(classes, generator=g, device="cuda") * 2 - 1) * 1.4).to(BF)
    target = torch.randint(0, classes, (batch, 1, pixels), generator=g, device="cuda")
    target[torch.rand(batch, 1, pixels, generator=g, device="cuda") < 0.1] = -100
    grad = torch.tensor(1.0, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    gx, gw, gb = ops.cross_entropy_backward(grad, saved, x, weight, bias, target, -100, False)
    total, w_sum, b_sum, n = 0.0, 0.0, 0.0, 0
    for i in range(batch):
        for k in range(0, pixels, part):
            some, t = x[i:i + 1, :, :, k:k + part], target[i:i + 1, :, k:k + part].contiguous()
            some = some.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else some.contiguous()
            one, kept = ops.cross_entropy_forward(some, weight, bias, t, -100, False)
            px, pw, pb = ops.cross_entropy_backward(grad, kept, some, weight, bias, t, -100, False)
            assert (gx[i:i + 1, :, :, k:k + part].double() - px).norm() <= (2 * 2.0 ** -8 + 2 * 2.0 ** -19) * px.double().norm()
            total, w_sum, b_sum, n = total + one.double().item(), w_sum + pw.double(), b_sum + pb.double(), n + 1
    assert abs(loss.item() - total) <= ((n + 1) * 2.0 ** -24 + 2 * 2.0 ** -19) * total
    # (roundings of n parts at random and of the whole; accumulators truncate 2^-10 of a share's sum of one sign, 2^17 pixels, on either side)
    for whole, parts in ((gw, w_sum), (gb, b_sum)):
        assert (whole.double() - parts).norm() <= ((n ** 0.5 + 1) * 2.0 ** -8 + 2 * 2.0 ** -10) * parts.norm()
