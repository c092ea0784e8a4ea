"""GPU: float32 classification losses on the tensor cores, sums of one sign at their greatest lengths: what their accumulators cut off."""
import pytest
import torch

from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


@pytest.mark.parametrize("pixels,channels,classes", [(2000, 1024, 64), (700, 1024, 4096), (5000, 64, 4096), (40_000, 48, 16)])
def test_sums_of_one_sign(ops, pixels, channels, classes):
    """Features and weights between a half and one (times 8 / channels): no term cancels.  An accumulator cuts off up to 2^-23 of what it
    holds for every sixteen terms: channels / 16 2^-23 of a score at most, classes / 16 2^-23 of an input gradient's terms, 64 2^-23 of a
    parameter gradient's for the 1024 pixels of a share, and half a step for each share that is added.  A score's error is its exponential's."""
    g = torch.Generator("cuda").manual_seed(channels + classes)
    x = (torch.rand(1, channels, 1, pixels, generator=g, device="cuda") + 1) / 2 * (8.0 / channels)
    weight = (torch.rand(classes, channels, 1, generator=g, device="cuda") + 1) / 2
    weight[0] = 0.0  # every pixel's label: its loss is the others' log-sum-exp
    bias = torch.zeros(classes, device="cuda")
    target = torch.zeros(1, 1, pixels, dtype=torch.int64, device="cuda")
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, False)
    gx, gw, gb = ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target, -100, False)
    rows, w = x.double()[0, :, 0].T, weight.double()[:, :, 0]
    z = rows @ w.T
    p, lse = z.softmax(1), z.logsumexp(1)
    e_z = (channels / 16 * 2.0 ** -23 + 2.0 ** -22) * z  # of a score, and a few half steps of its parts and differences
    fn = 2.0 ** -19  # exponential and logarithm (step_reference)
    e_lse = e_z.amax(1)
    assert abs(loss.item() - lse.sum().item()) <= (e_lse.sum() + (fn + 2.0 ** -23) * lse.sum()).item()
    gz = p.clone()
    gz[:, 0] -= 1
    e_gz = p * (e_z + e_lse[:, None] + fn) + 2.0 ** -22 * gz.abs()
    want = gz @ w
    assert ((gx[0, :, 0].T.double() - want).abs() <= e_gz @ w + (classes / 16 * 2.0 ** -23 + 2.0 ** -22) * (gz.abs() @ w)).all()
    own = 64 * 2.0 ** -23 + (pixels / 1024 + 4) * 2.0 ** -24
    assert ((gw[:, :, 0].double() - gz.T @ rows).abs() <= e_gz.T @ rows + own * (gz.abs().T @ rows)).all()
    # (column sums: float32 sums of 64 of a share's pixels to a thread, then the threads' and the shares')
    assert ((gb.double() - gz.sum(0)).abs() <= e_gz.sum(0) + (own + 64 * 2.0 ** -24) * gz.abs().sum(0)).all()


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("shape,channels,classes,mean", [((4, 60, 80), 64, 13, True), ((2, 1, 2562), 32, 32, False), ((1, 50, 41), 40, 9, True),
                                                         ((3, 1, 777), 16, 2, True), ((1, 1, 5000), 300, 24, False), ((1, 7, 9), 5, 1, True),
                                                         ((2, 1, 129), 8, 31, True), ((70, 30, 31), 17, 8, False)])
def test_few_classes_are_rounded_once(ops, shape, channels, classes, mean, layout):
    """bf16, up to 32 classes: gradients of scores are kept in two parts, 16 bits.  What the results are off beside their own rounding is the
    scores' and the exponentials' errors (2^-19 of a probability, step_reference): less than a hundredth of it."""
    bf16 = torch.bfloat16
    g = torch.Generator("cuda").manual_seed(classes)
    x = torch.randn(shape[0], channels, *shape[1:], generator=g, device="cuda").to(bf16)
    x = x.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else x
    weight = ((torch.rand(classes, channels, 1, generator=g, device="cuda") * 2 - 1) * 4 / channels ** 0.5).to(bf16)
    bias = torch.randn(classes, generator=g, device="cuda").to(bf16)
    target = torch.randint(0, classes, shape, generator=g, device="cuda")
    target[torch.rand(shape, generator=g, device="cuda") < 0.2] = -100
    loss, saved = ops.cross_entropy_forward(x, weight, bias, target, -100, mean)
    got = ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target, -100, mean)
    valid = (target != -100).reshape(-1)
    rows = x.double().permute(0, 2, 3, 1).reshape(-1, channels)
    gz = (rows @ weight.double()[:, :, 0].T + bias.double()).softmax(1)
    gz[torch.arange(len(gz), device="cuda"), target.reshape(-1).clamp(min=0)] -= 1
    gz = gz * valid[:, None] / (valid.sum() if mean else 1)
    want = (gz @ weight.double()[:, :, 0]).view(shape[0], *shape[1:], channels).permute(0, 3, 1, 2), (gz.T @ rows)[:, :, None], gz.sum(0)
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 1.05 * (b.to(bf16).double() - b).norm()
    for need in ((False, True), (True, False)):
        part = ops.cross_entropy_backward(torch.ones_like(loss), saved, x, weight, bias, target, -100, mean, *need)
        assert all(a is None or torch.equal(a, b) for a, b in zip(part, got))
