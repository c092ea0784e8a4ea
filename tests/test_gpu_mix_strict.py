"""GPU: channel mixing against bounds that hold pre-activations to float32 sums; few channels, so that one value's error shows."""
import pytest
import torch

import mix_reference as R
import mix_strict as M
from mappedconvolutions_b200 import host

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def normal(g, shape, dtype, layout=None, scale=1.0):
    t = (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_pre_activations_are_float32(name, layout, dtype):
    for i, (cin, hidden, cout) in enumerate([(2, 1, 1), (8, 2, 3), (5, 8, 16)]):
        g = torch.Generator("cuda").manual_seed(30 + i)
        x, gy = normal(g, (2, cin, 37, 61), dtype, layout), normal(g, (2, cout, 37, 61), dtype, layout)
        r = normal(g, (2, cout, 37, 61), dtype, layout) if i else None
        w, b = normal(g, (cout, cin, 1), dtype, scale=3 / cin ** 0.5), normal(g, (cout,), dtype)
        y, saved = host.impl.pointwise_forward(x, w, b, r, R.ACTS[name], True)
        got = host.impl.pointwise_backward(gy, saved, x, w, b, R.ACTS[name])
        R.check(dict(zip(("gx", "gw", "gb"), got), y=y), M.pointwise(x, w, b, r, name, gy), str((cin, cout)))
        wi, bi = normal(g, (2 * hidden, cin, 1), dtype, scale=3 / cin ** 0.5), normal(g, (2 * hidden,), dtype)
        wo, bo = normal(g, (cout, hidden, 1), dtype), normal(g, (cout,), dtype)
        y, saved = host.impl.gated_forward(x, wi, bi, wo, bo, r, R.ACTS[name], True)
        got = host.impl.gated_backward(gy, saved, x, wi, bi, wo, R.ACTS[name])
        R.check(dict(zip(("gx", "gw_in", "gb_in", "gw_out", "gb_out"), got), y=y), M.gated(x, wi, bi, wo, bo, r, name, gy),
                str((cin, hidden, cout)))


def one_channel(z, name, dtype):
    """act(z) and act'(z) for every element of z, through a layer with one channel, weight one and bias zero"""
    x = z.view(1, 1, 1, -1)
    w, b = torch.ones(1, 1, 1, device="cuda", dtype=dtype), torch.zeros(1, device="cuda", dtype=dtype)
    y, saved = host.impl.pointwise_forward(x, w, b, None, R.ACTS[name], True)
    gx = host.impl.pointwise_backward(torch.ones_like(x), saved, x, w, b, R.ACTS[name], True, False)[0]
    return y.view(-1).double(), gx.view(-1).double()


def error_of_functions(dtype):
    return {BF: 2.0 ** -15, F32: 2.0 ** -20, F64: 2.0 ** -48}[dtype]


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
def test_sigmoid_and_its_slope_are_accurate_relative_to_their_values(dtype):
    z = torch.cat([torch.linspace(-80, 80, 4001, device="cuda"), torch.linspace(-1, 1, 501, device="cuda")]).to(dtype)
    y, s = one_channel(z, "sigmoid", dtype)
    zd = z.double()
    e = (-zd.abs()).exp()
    q = 1 / (1 + e)
    bound = torch.finfo(dtype).eps / 2 + error_of_functions(dtype)
    assert ((y - torch.where(zd < 0, e * q, q)).abs() <= bound * y.abs()).all()
    want = e * q * q
    worst = ((s - want).abs() / want).max().item()
    assert worst <= bound, worst


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_large_finite_values(name, dtype):
    """where squares and exponentials of z overflow, act(z) is z or zero (sigmoid: one or zero), act'(z) one or zero"""
    top = torch.finfo(dtype).max
    z = torch.tensor([50.0, 1e6, 1e18, 3e19, 1e30, top / 4, top], device="cuda", dtype=F64).to(dtype)
    y, s = one_channel(z, name, dtype)
    ym, sm = one_channel(-z, name, dtype)
    if name == "sigmoid":
        assert ((y - 1).abs() <= 2.0 ** -8).all() and (ym.abs() <= 1e-21).all()
        assert (s.abs() <= 1e-21).all() and (sm.abs() <= 1e-21).all()  # (e^-50 = 2e-22)
        return
    assert torch.equal(y, z.double()) and torch.equal(s, torch.ones_like(s))
    if name is None:
        assert torch.equal(ym, -y) and torch.equal(sm, s)
    else:
        assert (ym.abs() <= 1e-19).all() and (sm.abs() <= 1e-19).all()  # (50 e^-50 = 1e-20)
