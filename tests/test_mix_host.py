"""CPU: channel-mixing layers and gradient clipping - parameters, argument checks, refusals, the C ABI's own checks."""
import ctypes
import math
import warnings

import pytest
import torch

from mappedconvolutions_b200 import _lib, host, nn as mnn, ops as twin
from mappedconvolutions_b200 import dist as mdist
from mappedconvolutions_b200.nn import functions as F


def test_names():
    import mapped_convolution.nn as a
    import mapped_convolutions.nn as b
    for n in ("PointwiseConvolution", "GatedFeedForward"):
        assert getattr(a, n) is getattr(b, n) is getattr(mnn, n)


def test_parameters():
    torch.manual_seed(0)
    p = mnn.PointwiseConvolution(6, 10, activation="relu")
    assert p.weight.shape == (10, 6, 1) and p.bias.shape == (10,) and set(p.state_dict()) == {"weight", "bias"}
    m = mnn.MappedConvolution(6, 10, 1)
    m.load_state_dict(p.state_dict())  # the same parameters as a mapped convolution with one tap
    g = mnn.GatedFeedForward(6, 20, 3, bias=False)
    assert g.weight_in.shape == (40, 6, 1) and g.weight_out.shape == (3, 20, 1) and g.activation == "silu"
    assert not g.bias_in.any() and not g.bias_out.any() and g.bias_in.requires_grad
    assert g.weight_in.abs().max() <= 1 / math.sqrt(6) and g.weight_out.abs().max() <= 1 / math.sqrt(20)
    assert mnn.GatedFeedForward(6, 20).out_channels == 6


def test_argument_checks():
    for bad in ("tanh", "ReLU", 1):
        with pytest.raises(AssertionError):
            mnn.PointwiseConvolution(3, 4, activation=bad)
        with pytest.raises(AssertionError):
            mnn.GatedFeedForward(3, 4, activation=bad)
    x = torch.zeros(1, 3, 4, 5)
    for layer in (mnn.PointwiseConvolution(3, 4), mnn.GatedFeedForward(3, 8, 4)):
        for args in [(x[0],), (torch.zeros(1, 2, 4, 5),), (x, torch.zeros(1, 3, 4, 5)), (x, torch.zeros(1, 4, 4, 6)),
                     (x, torch.zeros(1, 4, 4, 5).double())]:
            with pytest.raises(AssertionError):
                layer(*args)


@pytest.mark.parametrize("ops", [twin] + ([host.impl] if host.COMPILED else []), ids=["ctypes", "compiled"][:1 + host.COMPILED])
def test_no_cpu_path(ops):
    x, w, b = torch.zeros(1, 3, 4, 5), torch.zeros(4, 3, 1), torch.zeros(4)
    wi, bi, wo = torch.zeros(16, 3, 1), torch.zeros(16), torch.zeros(4, 8, 1)
    for call in (lambda: ops.pointwise_forward(x, w, b), lambda: ops.pointwise_backward(torch.zeros(1, 4, 4, 5), None, x, w, b),
                 lambda: ops.gated_forward(x, wi, bi, wo, b),
                 lambda: ops.gated_backward(torch.zeros(1, 4, 4, 5), b, x, wi, bi, wo),
                 lambda: ops.gradient_norm([b]), lambda: ops.clip_gradients([b], 1.0),
                 lambda: mnn.PointwiseConvolution(3, 4)(x), lambda: mdist.clip_gradients([None, b], 1.0)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()


def test_abi_checks_come_before_any_cuda_call():
    L = _lib.lib()
    ok = dict(B=1, S=20, C_in=3, C_out=4, hidden=0, act=1, dtype=_lib.MC_F32, layout=_lib.MC_NCHW)

    def desc(**change):
        return _lib.McMixDesc(**{**ok, **change})
    assert L.mc_pointwise_saved_bytes(desc()) >= 20 * 4 * 4 and L.mc_pointwise_saved_bytes(desc(act=0)) == 0
    fwd = lambda d, x=1: L.mc_pointwise_fwd(d, x, 1, None, None, 1, None, None, 0, None)
    for change in (dict(B=0), dict(S=0), dict(C_in=0), dict(C_out=-1), dict(hidden=2), dict(act=6), dict(act=-1),
                   dict(dtype=3), dict(layout=2)):
        assert fwd(desc(**change)) == -1
        assert L.mc_pointwise_workspace_bytes(desc(**change), 1) == 0
    assert fwd(desc(), None) == -1
    for change in (dict(B=1 << 20, S=1 << 20), dict(S=1 << 31), dict(B=1 << 33, S=1 << 30), dict(B=1 << 62, S=1 << 2), dict(C_in=1 << 21)):
        assert fwd(desc(**change)) == -6
    assert L.mc_pointwise_bwd(desc(), 1, 1, 1, 1, None, 1, 1, 1, 1, 1 << 30, None) == -1  # saved is missing
    assert L.mc_pointwise_bwd(desc(), 1, 1, 1, 1, 1, 1, 1, 1, None, 0, None) == -3
    gated = dict(hidden=8, act=4)
    assert L.mc_gated_fwd(desc(), *[1] * 9, 1 << 30, None) == -1                       # no hidden channels
    assert L.mc_gated_fwd(desc(**gated), 1, 1, 1, 1, 1, None, 1, None, None, 0, None) == -3
    assert L.mc_gated_bwd(desc(**gated), *[1] * 11, None, 0, None) == -3
    assert L.mc_gated_bwd(desc(**gated), 1, 1, 1, 1, 1, None, 1, 1, 1, 1, 1, 1, 1 << 30, None) == -1
    b16 = dict(dtype=_lib.MC_BF16, layout=_lib.MC_NHWC)                               # unaligned bf16 tensors
    assert L.mc_pointwise_fwd(desc(**b16), 24, 16, None, None, 16, None, 256, 1 << 30, None) == -1
    assert L.mc_gated_fwd(desc(**b16, **gated), 16, 16, 2, 24, 2, None, 16, None, 256, 1 << 30, None) == -1
    one = (ctypes.c_void_p * 1)(256)
    n, t, bad = (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(0), (ctypes.c_int32 * 1)(7)
    assert L.mc_grad_norm(-1, one, n, t, 2.0, 1, None, 1, 1 << 20, None) == -1
    assert L.mc_grad_norm(1, one, n, bad, 2.0, 1, None, 1, 1 << 20, None) == -1
    assert L.mc_grad_norm(1, one, n, t, 3.0, 1, None, 1, 1 << 20, None) == -2
    assert L.mc_grad_norm(1, one, n, t, 2.0, 1, None, 1, 8, None) == -3
    assert L.mc_grad_clip(1, one, t, one, t, n, 2.0, -1.0, 1, None, 1, 1 << 20, None) == -1
    assert L.mc_grad_clip(1, one, t, None, t, n, 2.0, 1.0, 1, None, 1, 1 << 20, None) == -1


@pytest.mark.parametrize("dtype", [_lib.MC_F32, _lib.MC_F64, _lib.MC_BF16])
def test_abi_refuses_memory_that_starts_anywhere(dtype):
    """activations and weights on their elements (bf16: 16 bytes), vectors on their elements, memory of a call on 16 bytes"""
    L, big = _lib.lib(), 1 << 30
    element = {_lib.MC_F32: 4, _lib.MC_F64: 8, _lib.MC_BF16: 2}[dtype]
    tensor = 16 if dtype == _lib.MC_BF16 else element
    d = _lib.McMixDesc(B=1, S=20, C_in=3, C_out=4, hidden=0, act=1, dtype=dtype, layout=_lib.MC_NCHW)
    g = _lib.McMixDesc(B=1, S=20, C_in=3, C_out=4, hidden=8, act=1, dtype=dtype, layout=_lib.MC_NCHW)
    calls = [  # (call, which alignment each pointer needs)
        (lambda *p: L.mc_pointwise_fwd(d, *p, big, None), [tensor, tensor, element, tensor, tensor, 16, 16]),
        (lambda *p: L.mc_pointwise_bwd(d, *p, big, None), [tensor, tensor, tensor, element, 16, tensor, element, element, 16]),
        (lambda *p: L.mc_gated_fwd(g, *p, big, None), [tensor, tensor, element, tensor, element, tensor, tensor, 16, 16]),
        (lambda *p: L.mc_gated_bwd(g, *p, big, None),
         [tensor, tensor, tensor, element, tensor, 16, tensor, element, element, element, element, 16]),
    ]
    for call, need in calls:
        for i, n in enumerate(need):
            pointers = [4096] * len(need)
            pointers[i] += n // 2
            assert call(*pointers) == -1, (i, n)
    one, n, t = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(dtype)
    assert L.mc_grad_norm(1, one, n, t, 2.0, 16, None, 4100, 1 << 20, None) == -1


def test_traced_layers_run_again_on_replay(monkeypatch):
    """a tracer sees one Python operation, which computes the layer on every replay"""
    if not host.COMPILED:
        pytest.skip("extension not built: only the Functions exist")
    fake = dict(pointwise_forward=lambda x, w, b, r, a, k: (x[:, :1] * 2, None),
                gated_forward=lambda x, wi, bi, wo, bo, r, a, k: (x[:, :1] * 3, None))
    monkeypatch.setattr(F, "ops", type("Ops", (), {k: staticmethod(v) for k, v in fake.items()}
                                       | {n: staticmethod(getattr(host.impl, n)) for n in ("pointwise_layer", "gated_layer")}))
    monkeypatch.setattr(F, "pointwise", F._layer_call(F.PointwiseFn, "pointwise_layer"))
    monkeypatch.setattr(F, "gated", F._layer_call(F.GatedFn, "gated_layer"))
    x, z = torch.randn(2, 3, 4, 6), torch.randn(2, 3, 4, 6)
    for layer, k in ((mnn.PointwiseConvolution(3, 1), 2), (mnn.GatedFeedForward(3, 2, 1), 3)):
        with warnings.catch_warnings(), torch.no_grad():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(layer, (x,), check_trace=False)
        assert torch.equal(traced(z), z[:, :1] * k)
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda t: layer(t[None]))(x)
