"""GPU: clipping into tensors that lie in memory otherwise than their gradients."""
import pytest
import torch

from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def test_dense_results_in_another_order_share_no_memory(ops):
    """results that are copied to where they belong would overwrite each other without a word"""
    a = torch.zeros(8, 6, device="cuda")
    g0, g1 = torch.randn(6, 8, device="cuda"), torch.randn(6, device="cuda")
    for out in ([a.t(), a[3]], [a.t(), a.t()[:, 7]], [a.t(), torch.as_strided(a, (6,), (1,), 42)]):
        with pytest.raises(RuntimeError, match="share memory"):
            ops.clip_gradients([g0, g1], 1.0, 2.0, out)
        assert not a.any()
    b = torch.zeros(6, device="cuda")
    norm = ops.clip_gradients([g0, g1], 0.5, 2.0, [a.t(), b])
    c = 0.5 / (norm.double() + 1e-6)
    for got, g in ((a.t(), g0), (b, g1)):
        # (the norm: eight roundings of a float32 sum, half of them behind the root; its own, the coefficient's, the product's)
        assert ((got.double() - g.double() * c).abs() <= 8 * 2.0 ** -24 * (g.double() * c).abs()).all()


def test_tensors_of_inference_mode(ops):
    """refused outside of it before anything is written, scaled inside"""
    with torch.inference_mode():
        t = torch.full((100,), 3.0, device="cuda")
    g = torch.ones(100, device="cuda")
    for call in (lambda: ops.clip_gradients([t], 1.0), lambda: ops.clip_gradients([g], 1.0, 2.0, [t])):
        with pytest.raises(RuntimeError, match="inference mode"):
            call()
        assert (t == 3.0).all()
    with torch.inference_mode():
        assert ops.clip_gradients([t], 1.0).item() == 30.0
        assert ((t - 0.1).abs() <= 2.0 ** -20).all()
