"""CPU: the channel-mixing layers' Python Functions on stand-ins for the device calls."""
import pytest
import torch

from mappedconvolutions_b200.nn import functions as F


@pytest.fixture
def stand_ins(monkeypatch):
    """y = 2 x w[0] + r, with first derivatives"""
    calls = []

    def forward(x, w, *rest):
        calls.append(("forward", rest[-1]))
        return x * w.flatten()[0] * 2 + (0 if rest[-3] is None else rest[-3]), None

    def pointwise_backward(gy, saved, x, w, b, a, nx, np):
        calls.append(("backward", nx, np))
        gw = torch.zeros_like(w)
        gw.view(-1)[0] = (gy * x * 2).sum()
        return [(gy * w.flatten()[0] * 2).detach() if nx else None, gw.detach() if np else None, torch.zeros_like(b) if np else None]

    def gated_backward(gy, saved, x, wi, bi, wo, a, nx, np):
        return pointwise_backward(gy, saved, x, wi, bi, a, nx, np) + [torch.zeros_like(wo), torch.zeros(1)]
    fakes = dict(pointwise_forward=forward, gated_forward=forward, pointwise_backward=pointwise_backward, gated_backward=gated_backward)
    monkeypatch.setattr(F, "ops", type("Ops", (), {k: staticmethod(v) for k, v in fakes.items()}))
    return calls


def layers():
    p = lambda *s: torch.rand(*s, requires_grad=True)
    w, b = p(1, 1, 1), p(1)
    yield lambda x, r=None: F.PointwiseFn.apply(x, w, b, r, 0), w
    wi, bi, wo, bo = p(2, 1, 1), p(2), p(1, 1, 1), p(1)
    yield lambda x, r=None: F.GatedFn.apply(x, wi, bi, wo, bo, r, 4), wi


def test_second_derivatives_are_refused(stand_ins):
    for layer, w in layers():
        x = torch.rand(1, 1, 2, 3, requires_grad=True)
        gx, gw = torch.autograd.grad(layer(x).sum(), [x, w], create_graph=True)
        assert torch.equal(gx, torch.full_like(x, 2 * w.flatten()[0].item()))  # the first ones are there
        for g in (gx, gw):
            for leaf in (x, w):
                with pytest.raises(RuntimeError, match="second derivatives"):
                    torch.autograd.grad(g.square().sum(), leaf, retain_graph=True, allow_unused=True)
        with pytest.raises(RuntimeError, match="second derivatives"):
            (layer(x).sum() + gx.square().sum()).backward()
        assert not torch.autograd.grad(layer(x).sum(), x)[0].requires_grad


def test_a_residuals_gradient_is_linear(stand_ins):
    """the residual passes through: its gradient is the output's, derivatives included"""
    for layer, w in layers():
        x, r = torch.rand(1, 1, 2, 3), torch.rand(1, 1, 2, 3, requires_grad=True)
        gr, = torch.autograd.grad(layer(x, r).square().sum(), r, create_graph=True)
        assert torch.equal(torch.autograd.grad(gr.sum(), r)[0], torch.full_like(r, 2.0))


def test_nothing_is_kept_for_a_residual_alone(stand_ins):
    for layer, w in layers():
        x, r = torch.rand(1, 1, 2, 3), torch.rand(1, 1, 2, 3, requires_grad=True)
        stand_ins.clear()
        layer(x, r)
        assert stand_ins == [("forward", True)]  # (the parameters)
    frozen = [torch.rand(2, 1, 1), torch.rand(2), torch.rand(1, 1, 1), torch.rand(1)]
    for call in (lambda: F.PointwiseFn.apply(x, frozen[2], frozen[3], r, 0), lambda: F.GatedFn.apply(x, *frozen, r, 4)):
        stand_ins.clear()
        call().sum().backward()
        assert stand_ins == [("forward", False)] and r.grad is not None
