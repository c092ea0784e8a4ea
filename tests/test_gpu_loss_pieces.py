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
