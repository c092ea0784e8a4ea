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


@pytest.mark.parametrize("max_norm", [1e-3, 1e-6, 1e-20, 1e-35])
@pytest.mark.parametrize("source,result", [(F32, F32), (BF, BF), (BF, F32), (F32, F64)])
def test_coefficients_below_the_float32_range(ops, source, result, max_norm):
    """gradients that exploded: max_norm / norm is far below 1e-38, its products with the gradients are not"""
    g = torch.Generator("cuda").manual_seed(2)
    ts = [(torch.randn(n, generator=g, device="cuda", dtype=F64) * 5e36).to(source) for n in (3, 50_000)]
    out = [torch.empty(t.shape, device="cuda", dtype=result) for t in ts]
    norm = torch.cat([t.double().view(-1) for t in ts]).norm().item()
    ops.clip_gradients(ts, max_norm, 2.0, out)
    # squares above 1e38 are summed in double; a rounding of the coefficient and of the product, and the result's
    tol = 2.0 ** -22 + torch.finfo(result).eps / 2
    # below the normal range steps have a fixed size, tiny * eps (bf16 2^-133, float32 2^-149): half of one of the result's type
    # (float64: none is reached), and of float32 for each of the two products
    denormal = torch.finfo(F32).tiny * (torch.finfo(F32).eps + torch.finfo(result).eps / 2)
    for t, o in zip(ts, out):
        want = t.double() * (max_norm / norm)
        assert ((o.double() - want).abs() <= tol * want.abs() + denormal).all()
