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
