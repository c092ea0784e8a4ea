"""CPU: AdamW takes states of torch's optimisers as they go on, or refuses them before anything changes."""
import copy

import pytest
import torch

from mappedconvolutions_b200 import optim

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def trained(dtype, shape=(40, 30), kind=torch.optim.AdamW, order=None, **args):
    """a parameter and its torch optimiser after three steps"""
    gen = torch.Generator().manual_seed(3)
    p = torch.randn(shape, generator=gen).to(dtype)
    p = torch.nn.Parameter(p if order is None else p.contiguous(memory_format=order))
    opt = kind([p], lr=1e-2, **args)
    for _ in range(3):
        p.grad = torch.randn(shape, generator=gen).to(dtype).contiguous(memory_format=order or torch.contiguous_format)
        opt.step()
    return p, opt


@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_options_stay_and_moments_take_their_form(dtype, bits, master):
    p, theirs = trained(dtype)
    q = torch.nn.Parameter(p.detach().clone())
    opt = optim.AdamW([q], lr=1, state_bits=bits, master_weights=master)
    opt.load_state_dict(copy.deepcopy(theirs.state_dict()))
    group, state, old = opt.param_groups[0], opt.state[q], theirs.state[p]
    assert group["state_bits"] == bits and group["master_weights"] == master and group["lr"] == 1e-2 and int(state["step"]) == 3
    if bits == 8 and dtype != F64:
        assert state["exp_avg"].dtype == torch.int8 and state["exp_avg_sq"].dtype == torch.uint8
        s, r = (state[k].repeat_interleave(256)[:q.numel()].view(q.shape) for k in ("exp_avg_scale", "exp_avg_sq_scale"))
        m, v = state["exp_avg"].float(), state["exp_avg_sq"].float()
        # nearest codes of the square roots: half a code, and what float32 roots and products add to it
        assert ((old["exp_avg"].float().abs() / s).sqrt() - m.abs()).abs().max() <= 0.5 + 1e-4
        assert (m * old["exp_avg"].float() >= 0).all()
        root = (old["exp_avg_sq"].float().sqrt() / r).sqrt()
        assert ((root - v).abs()[root > 0.5]).max() <= 0.5 + 1e-4 and (v[old["exp_avg_sq"] > 0] > 0).all()
    else:
        wide = F64 if dtype == F64 else F32
        for k in ("exp_avg", "exp_avg_sq"):
            assert state[k].dtype == wide and torch.equal(state[k], old[k].to(wide)) and state[k].data_ptr() != old[k].data_ptr()


def test_moments_lie_as_their_parameter_does():
    p, theirs = trained(F32, (6, 5, 4, 3))
    kept = theirs.state_dict()
    for bits in (8, 32):
        q = torch.nn.Parameter(p.detach().contiguous(memory_format=torch.channels_last))
        opt = optim.AdamW([q], state_bits=bits)
        opt.load_state_dict(copy.deepcopy(kept))
        assert opt.state[q]["exp_avg"].stride() == opt.state[q]["exp_avg_sq"].stride() == q.stride()
    assert torch.equal(opt.state[q]["exp_avg"], theirs.state[p]["exp_avg"])
    r = torch.nn.Parameter(p.detach().clone())
    a = optim.AdamW([q], state_bits=8)
    a.load_state_dict(copy.deepcopy(kept))
    with pytest.raises(ValueError, match="lie as they do"):  # (codes belong to blocks of the other order)
        optim.AdamW([r]).load_state_dict(copy.deepcopy(a.state_dict()))


def test_states_that_cannot_go_on_are_refused_before_anything_changes():
    p, theirs = trained(BF)
    good = copy.deepcopy(theirs.state_dict())
    coupled = copy.deepcopy(trained(BF, kind=torch.optim.Adam, weight_decay=0.1)[1].state_dict())
    other = copy.deepcopy(trained(BF, (30, 40))[1].state_dict())
    part = copy.deepcopy(good)
    del part["state"][0]["exp_avg_sq"]
    wide, opt8 = torch.nn.Parameter(torch.zeros(40, 30, dtype=F64)), optim.AdamW([p], state_bits=8)
    opt8.load_state_dict(copy.deepcopy(good))
    bad8 = copy.deepcopy(opt8.state_dict())
    bad8["state"][0]["exp_avg_scale"] = bad8["state"][0]["exp_avg_scale"][:1]
    mast = copy.deepcopy(good)
    mast["state"][0]["master"] = torch.zeros(40, 30)
    for q, state, text in [(p, coupled, "weight decay"), (p, other, "shape"), (p, part, "exp_avg_sq"), (p, bad8, "scale"),
                           (wide, opt8.state_dict(), "8 bits"), (torch.nn.Parameter(torch.zeros(40, 30)), mast, "master")]:
        opt = optim.AdamW([q], lr=0.5, weight_decay=0.25)
        with pytest.raises(ValueError, match=text):
            opt.load_state_dict(state)
        assert opt.param_groups[0]["lr"] == 0.5 and opt.param_groups[0]["weight_decay"] == 0.25 and not opt.state
    none = copy.deepcopy(trained(BF, kind=torch.optim.Adam)[1].state_dict())  # Adam without decay takes the same steps
    opt = optim.AdamW([p])
    opt.load_state_dict(none)
    assert opt.param_groups[0]["weight_decay"] == 0 and opt.state[p]["exp_avg"].dtype == F32
    with pytest.raises(ValueError, match="group"):  # torch's own
        optim.AdamW([dict(params=[p]), dict(params=[wide])]).load_state_dict(good)
