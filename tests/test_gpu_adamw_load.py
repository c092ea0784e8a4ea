"""GPU: AdamW goes on from states of torch.optim.AdamW, whatever the types of parameters and moments."""
import copy
import math

import pytest
import torch

from mappedconvolutions_b200.optim import AdamW

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_the_next_step(dtype, bits, master):
    """against the formula in 64 bits on the state's own values: products, roots and quotients are a few roundings of the result each
    (2^-21 of what is added up in float32, 2^-50 in float64), the parameter is rounded once"""
    gen = torch.Generator("cuda").manual_seed(4)
    rand = lambda: torch.randn(50, 31, generator=gen, device="cuda").to(dtype)  # noqa: E731
    p = torch.nn.Parameter(rand())
    theirs = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), weight_decay=0.1)
    for _ in range(3):
        p.grad = rand()
        theirs.step()
    opt = AdamW([p], state_bits=bits, master_weights=master)
    opt.load_state_dict(copy.deepcopy(theirs.state_dict()))
    (m, v), p0, g = opt.moments()[0], p.detach().double().clone(), rand()
    m, v = (t.double().clone() for t in (m, v))
    p.grad = g
    opt.step()
    state = opt.state[p]
    assert int(state["step"]) == 4 and ("master" in state) == (master and dtype == BF)
    m, v = 0.8 * m + 0.2 * g.double(), 0.95 * v + 0.05 * g.double().square()
    size = m.abs() + 0.4 * g.double().abs()  # (at least the terms of m, which may cancel)
    rate = 1e-2 / (1 - 0.8 ** 4) / (v.sqrt() / math.sqrt(1 - 0.95 ** 4) + 1e-8)
    want = p0 * (1 - 1e-3) - rate * m
    got = state["master"] if "master" in state else p.detach()
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** (-50 if dtype == F64 else -21) * (p0.abs() + rate * size)
    assert ((got.double() - want).abs() <= bound).all()
    assert "master" not in state or torch.equal(p.detach(), state["master"].to(BF))
    again = AdamW([torch.nn.Parameter(p.detach().clone())])
    again.load_state_dict(copy.deepcopy(opt.state_dict()))  # and its own state comes back as it is
    assert all(torch.equal(a, b) if torch.is_tensor(a) else a == b for a, b in zip(again.state_dict()["state"][0].values(), state.values()))
