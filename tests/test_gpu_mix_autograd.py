"""GPU: what the channel-mixing layers keep and refuse under autograd."""
import pytest
import torch

from mappedconvolutions_b200 import nn as mnn

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def layers(dtype):
    return [mnn.PointwiseConvolution(16, 24, activation="silu").cuda().to(dtype), mnn.GatedFeedForward(16, 32, 24).cuda().to(dtype)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_second_derivatives_are_refused(dtype):
    for m in layers(dtype):
        x = torch.randn(2, 16, 5, 7, device="cuda").to(dtype).requires_grad_(True)
        w = next(m.parameters())
        first = torch.autograd.grad(m(x).float().sum(), [x, w])
        gx, gw = torch.autograd.grad(m(x).float().sum(), [x, w], create_graph=True)
        assert torch.equal(gx, first[0]) and torch.equal(gw, first[1]) and not first[0].requires_grad
        for g in (gx, gw):
            for leaf in (x, w):
                with pytest.raises(RuntimeError, match="second derivatives"):
                    torch.autograd.grad(g.float().square().sum(), leaf, retain_graph=True, allow_unused=True)
        with pytest.raises(RuntimeError, match="second derivatives"):
            (m(x).float().sum() + gx.float().square().sum()).backward()


def test_a_residuals_gradient_is_linear():
    for m in layers(F32):
        m.requires_grad_(False)
        x, r = torch.randn(2, 16, 5, 7, device="cuda"), torch.randn(2, 24, 5, 7, device="cuda", requires_grad=True)
        gr, = torch.autograd.grad(m(x, r).square().sum(), r, create_graph=True)
        assert torch.equal(torch.autograd.grad(gr.sum(), r)[0], torch.full_like(r, 2.0))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_nothing_is_kept_for_a_residual_alone(dtype):
    def held(m, *args):
        before = torch.cuda.memory_allocated()
        y = m(*args)
        return torch.cuda.memory_allocated() - before, y

    x = torch.randn(2, 16, 50, 70, device="cuda").to(dtype)  # (NCHW: bf16 training calls keep its rows)
    r = torch.randn(2, 24, 50, 70, device="cuda").to(dtype)
    for m in layers(dtype):
        m(x, r)  # (the first call's allocations)
        with torch.no_grad():
            least, _ = held(m, x, r)
        assert held(m, x, r)[0] > least
        m.requires_grad_(False)
        got, y = held(m, x, r.requires_grad_(True))
        assert got == least
        y.float().sum().backward()
        assert torch.equal(r.grad, torch.ones_like(r))
        r = r.detach()


@pytest.mark.parametrize("binding", ["ctypes", "compiled"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_no_output_channels(binding, dtype):
    """an output without elements has gradients: zeros"""
    from mappedconvolutions_b200 import host, ops as twin
    ops = twin if binding == "ctypes" else host.impl
    t = lambda *s: torch.ones(*s, device="cuda", dtype=dtype)
    x, w, b = t(2, 6, 3, 5), t(0, 6, 1), t(0)
    y, saved = ops.pointwise_forward(x, w, b, None, 1, True)
    assert y.shape == (2, 0, 3, 5)
    gx, gw, gb = ops.pointwise_backward(y, saved, x, w, b, 1)
    assert torch.equal(gx, torch.zeros_like(x)) and gw.shape == w.shape and gb.shape == b.shape
    wi, bi, wo = t(8, 6, 1), t(8), t(0, 4, 1)
    y, saved = ops.gated_forward(x, wi, bi, wo, b, None, 4, True)
    g = ops.gated_backward(y, saved, x, wi, bi, wo, 4)
    assert all(torch.equal(p, torch.zeros_like(q)) for p, q in zip(g, (x, wi, bi, wo, b)))
