"""CPU: the bounds of mix_strict.py pass a model of the kernels and fail one that keeps pre-activations in bf16."""
import pytest
import torch

import mix_reference as R
import mix_strict as M

BF = torch.bfloat16


def rnd(t):
    return t.to(BF).double()


def tensors(cin, hidden, cout, seed=0, spread=3.0):
    """few channels: the bounds of sums are then not much wider than one value's; pre-activations of a few units, where
    slopes bend"""
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: (torch.randn(s, generator=g) * 1.0).to(BF)
    return dict(x=t(2, cin, 30, 41), gy=t(2, cout, 30, 41), wi=(t(2 * hidden, cin, 1) * spread).to(BF), bi=t(2 * hidden),
                wo=t(cout, hidden, 1), bo=t(cout), w=(t(cout, cin, 1) * spread).to(BF), b=t(cout))


def model_pointwise(p, name, keep):
    """float64 sums, rounded where the kernels round; keep: what becomes of z before the backward pass"""
    X, W, z, _ = M.pre_activations(p["x"], p["w"], p["b"])
    G = R.rows(p["gy"])
    gz = rnd(G * R.slope(name, keep(z))) if name else G
    back = lambda m: R.images(m, 2, 30, 41)
    return dict(y=back(rnd(R.act(name, z))), gx=back(rnd(gz @ W)), gw=rnd(gz.T @ X)[:, :, None], gb=rnd(gz.sum(0)))


def model_gated(p, name, keep):
    X, Wi, z, _ = M.pre_activations(p["x"], p["wi"], p["bi"])
    G, Wo, n = R.rows(p["gy"]), p["wo"].double()[:, :, 0], p["wo"].shape[1]
    h = rnd(R.act(name, z[:, :n]) * z[:, n:])
    z = keep(z)
    gh = G @ Wo
    gz = torch.cat([rnd(gh * z[:, n:] * R.slope(name, z[:, :n])), rnd(gh * R.act(name, z[:, :n]))], 1)
    back = lambda m: R.images(m, 2, 30, 41)
    return dict(y=back(rnd(h @ Wo.T + p["bo"].double())), gx=back(rnd(gz @ Wi)), gw_in=rnd(gz.T @ X)[:, :, None],
                gb_in=rnd(gz.sum(0)), gw_out=rnd(G.T @ h)[:, :, None], gb_out=rnd(G.sum(0)))


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu", "sigmoid"])
def test_bounds_know_rounded_pre_activations(name):
    p = tensors(2, 1, 1)
    want = M.pointwise(p["x"], p["w"], p["b"], None, name, p["gy"])
    R.check(model_pointwise(p, name, lambda z: z), want)
    R.check(model_pointwise(p, name, lambda z: z.float().double()), want)
    with pytest.raises(AssertionError, match="gx"):
        R.check(dict(gx=model_pointwise(p, name, rnd)["gx"]), want)
    R.check(model_pointwise(p, name, rnd), R.pointwise(p["x"], p["w"], p["b"], None, name, p["gy"]))  # (wider ones do not)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu", "sigmoid", None])
def test_bounds_know_rounded_gates(name):
    p = tensors(2, 1, 1, 1)
    want = M.gated(p["x"], p["wi"], p["bi"], p["wo"], p["bo"], None, name, p["gy"])
    R.check(model_gated(p, name, lambda z: z), want)
    if name is not None:  # (a product of two rounded factors alone stays within the bound of a rounded product of two)
        with pytest.raises(AssertionError, match="gx"):
            R.check(dict(gx=model_gated(p, name, rnd)["gx"]), want)
