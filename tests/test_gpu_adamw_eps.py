"""GPU: AdamW with an eps from none at all to large ones, gradients of all sizes side by side in every block of 256."""
import math

import pytest
import torch

from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("beta2", [0.9, 0.999, 0.999999])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-20, 1e-18, 1e-17, 2.0 ** -50, 1e-12, 4e-12, 5.6e-11, 5.8e-11, 1.8e-9, 1e-8, 1e-3])
def test_first_steps(ops, eps, beta2, bits):
    """Gradients from 1 down to 3e-19, whose squares are below the smallest normal number: the update is m / (sqrt(v) root + eps) of the
    float32 moments, in 64 bits.  The kernel's root, product, sum, quotient and difference are a few 2^-24 of the result each, and what
    a root that it takes for zero would add is 2^-24 of the divisor: 2^-21 of the update and of the parameter hold all of them."""
    gen = torch.Generator("cuda").manual_seed(11)
    n, lr, beta1 = 2000, 1e-2, 0.9
    g = 10.0 ** (torch.rand(n, generator=gen, device="cuda") * -18.5) * (torch.randint(0, 2, (n,), generator=gen, device="cuda") * 2 - 1)
    g[::256] = 1.0
    g = g.to(F32)
    p = torch.randn(n, generator=gen, device="cuda") * 1e-3
    f = lambda v: torch.tensor(v, dtype=F32, device="cuda")  # noqa: E731
    m32, v32 = g * f(1 - beta1), g * g * f(1 - beta2)  # (moments are zero before the first step)
    assert (v32 > 0).all()
    e = f(eps).double()
    update = lr / (1 - beta1) * m32.double() / (v32.double().sqrt() / math.sqrt(1 - beta2) + e)
    want = p.double() - update
    parts = p.double().abs() + update.abs()
    q = p.clone()
    m, v = torch.zeros(n, dtype=torch.int8 if bits == 8 else F32, device="cuda"), torch.zeros(n, dtype=torch.uint8 if bits == 8 else F32, device="cuda")
    scales = [torch.zeros((n + 255) // 256, device="cuda") if bits == 8 else None for _ in range(2)]
    ops.adamw_step([q], [g], [m], [v], [scales[0]], [scales[1]], [None], [1], lr, beta1, beta2, eps, 0.0)
    off = (q.double() - want).abs()
    assert (off <= 2.0 ** -21 * parts).all(), (off / parts).max().item()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [4e37, 1e38, 3e38])
def test_divisors_near_the_largest_number(ops, eps, bits):
    """m / (sqrt(v) root + eps) with moments as large: no reciprocal may be flushed to zero.  Roundings as above."""
    n, lr = 600, 1.0
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m32, v32 = torch.full((n,), 2e38, device="cuda"), torch.full((n,), 1.0, device="cuda")
    if bits == 8:
        scale = torch.full(((n + 255) // 256,), 2e38 / 127 ** 2, device="cuda")
        root = torch.full_like(scale, 1.0 / 255 ** 2)
        m, v = torch.full((n,), 127, dtype=torch.int8, device="cuda"), torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        m32, v32 = (t[0] for t in ops.adamw_moments([m], [v], [scale], [root]))
    else:
        m, v, scale, root = m32.clone(), v32.clone(), None, None
    want = -(lr / (1 - 0.5 ** 3)) * (m32.double() * 0.5) / ((v32.double() * 0.5).sqrt() / math.sqrt(1 - 0.5 ** 3) + torch.tensor(eps, dtype=F32).double().item())
    ops.adamw_step([p], [g], [m], [v], [scale], [root], [None], [3], lr, 0.5, 0.5, eps, 0.0)
    assert ((p.double() - want).abs() <= 2.0 ** -21 * want.abs()).all(), (p[0].item(), want[0].item())
