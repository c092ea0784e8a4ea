"""CPU: group norm, classification loss and AdamW - parameters, argument checks, refusals, the C ABI's own checks."""
import copy
import warnings

import pytest
import torch

from mappedconvolutions_b200 import _lib, host, nn as mnn, ops as twin, optim
from mappedconvolutions_b200.nn import functions as F


def test_names():
    import mapped_convolution.nn as a
    import mapped_convolutions.nn as b
    for n in ("GroupNorm", "PointwiseCrossEntropy"):
        assert getattr(a, n) is getattr(b, n) is getattr(mnn, n)


def test_parameters():
    n, t = mnn.GroupNorm(4, 12, activation="relu"), torch.nn.GroupNorm(4, 12)
    t.load_state_dict(n.state_dict())
    n.load_state_dict(t.state_dict())
    assert (n.weight == 1).all() and not n.bias.any() and not list(mnn.GroupNorm(4, 12, affine=False).parameters())
    c = mnn.PointwiseCrossEntropy(6, 10, bias=False)
    mnn.PointwiseConvolution(6, 10).load_state_dict(c.state_dict())
    assert c.weight.shape == (10, 6, 1) and not c.bias.any() and c.ignore_index == -100 and c.reduction == "mean"


def test_argument_checks():
    x, t = torch.zeros(1, 6, 4, 5), torch.zeros(1, 4, 5, dtype=torch.int64)
    for make in (lambda: mnn.GroupNorm(4, 6), lambda: mnn.GroupNorm(0, 6), lambda: mnn.GroupNorm(3, 6, eps=-1),
                 lambda: mnn.GroupNorm(3, 6, activation="tanh"), lambda: mnn.PointwiseCrossEntropy(6, 3, reduction="none"),
                 lambda: mnn.GroupNorm(3, 6)(x[0]), lambda: mnn.GroupNorm(5, 5)(x), lambda: mnn.PointwiseCrossEntropy(5, 3)(x, t),
                 lambda: mnn.PointwiseCrossEntropy(6, 3)(x, t.int()), lambda: mnn.PointwiseCrossEntropy(6, 3)(x, t[:, :3]),
                 lambda: mnn.PointwiseCrossEntropy(6, 3)(x, t[None])):
        with pytest.raises(AssertionError):
            make()
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=16),
                dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            optim.AdamW(p, **bad)


def test_options_of_groups_and_loaded_states():
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(4))
    opt = optim.AdamW([p])
    for bad in (dict(state_bits=16), dict(betas=(0.9, 1.0)), dict(lr=-1.0), dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[q], **bad))
        with pytest.raises(ValueError):
            optim.AdamW([dict(params=[q], **bad)])
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[q], state_bits=8, lr=0.5))
    assert opt.param_groups[1]["state_bits"] == 8 and opt.param_groups[0]["state_bits"] == 32
    for name in ("amsgrad", "maximize"):  # a state whose next step is another one
        other = torch.optim.AdamW([p], lr=0.25, **{name: True})
        with pytest.raises(ValueError, match=name):
            optim.AdamW([p]).load_state_dict(other.state_dict())
    opt = optim.AdamW([p])
    opt.load_state_dict(torch.optim.AdamW([p], lr=0.25).state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["state_bits"] == 32


@pytest.mark.parametrize("ops", [twin] + ([host.impl] if host.COMPILED else []), ids=["ctypes", "compiled"][:1 + host.COMPILED])
def test_no_cpu_path(ops):
    x, one, t = torch.zeros(1, 6, 4, 5), torch.ones(6), torch.zeros(1, 4, 5, dtype=torch.int64)
    w, b = torch.zeros(3, 6, 1), torch.zeros(3)
    for call in (lambda: ops.group_norm_forward(x, one, one, 2), lambda: ops.group_norm_backward(x, None, x, one, one, 2),
                 lambda: ops.cross_entropy_forward(x, w, b, t), lambda: ops.cross_entropy_backward(b[0], None, x, w, b, t),
                 lambda: ops.adamw_step([b], [b], [b], [b], [None], [None], [None], [1], 1e-3, 0.9, 0.99, 1e-8, 0.0),
                 lambda: ops.adamw_moments([b], [b], [b], [b]),
                 lambda: mnn.GroupNorm(2, 6)(x), lambda: mnn.PointwiseCrossEntropy(6, 3)(x, t)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="CUDA only"):
        optim.AdamW([p]).step()


def test_state_keeps_its_types_when_loaded():
    p = torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16))
    for bits, master in ((8, True), (32, False)):
        opt = optim.AdamW([p], state_bits=bits, master_weights=master)
        opt.state[p] = opt._new_state(p, opt.param_groups[0])
        opt.state[p]["step"] = 5
        other = optim.AdamW([p])
        other.load_state_dict(copy.deepcopy(opt.state_dict()))
        for k, v in opt.state[p].items():
            got = other.state[p][k]
            assert got == v if k == "step" else got.dtype == v.dtype and got.shape == v.shape and got.data_ptr() != v.data_ptr()
        assert other.param_groups[0]["state_bits"] == bits and ("exp_avg_scale" in other.state[p]) == (bits == 8)


def test_abi_checks_come_before_any_cuda_call():
    L, big = _lib.lib(), 1 << 40
    ok = dict(B=2, S=20, C=6, groups=3, act=1, dtype=_lib.MC_F32, layout=_lib.MC_NCHW, eps=1e-5)
    desc = lambda **k: _lib.McNormDesc(**{**ok, **k})  # noqa: E731
    assert L.mc_group_norm_stats_bytes(desc()) == 2 * 3 * 8 and L.mc_group_norm_workspace_bytes(desc(), 0) > 0
    fwd = lambda d, *p, n=big: L.mc_group_norm_fwd(d, *(p or [256] * 6), n, None)  # noqa: E731
    for k in (dict(B=0), dict(S=-1), dict(C=0), dict(groups=0), dict(groups=4), dict(act=6), dict(dtype=3), dict(layout=2), dict(eps=-1.0),
              dict(eps=float("nan"))):
        assert fwd(desc(**k)) == -1 and L.mc_group_norm_workspace_bytes(desc(**k), 1) == 0
    for k in (dict(B=1 << 20, S=1 << 20), dict(S=1 << 31), dict(B=1 << 62, S=4), dict(C=(1 << 20) + 3, groups=1)):
        assert fwd(desc(**k)) == -6
    for i, n in enumerate([16, 4, 4, 16, 16, 16]):
        p = [256] * 6
        p[i] += n // 2
        assert fwd(desc(), *p) == -1
    assert fwd(desc(), None, 256, 256, 256, 256, 256) == -1 and fwd(desc(), 256, 256, 256, 256, None, 256) == -1
    assert fwd(desc(), n=16) == -3 and L.mc_group_norm_bwd(desc(), *[256] * 9, 16, None) == -3
    assert L.mc_group_norm_bwd(desc(), 256, 256, 256, 256, None, *[256] * 4, big, None) == -1

    ok = dict(B=2, S=20, ignore_index=-100, C=6, V=9, reduction=1, dtype=_lib.MC_BF16, layout=_lib.MC_NCHW)
    desc = lambda **k: _lib.McCeDesc(**{**ok, **k})  # noqa: E731
    assert L.mc_cross_entropy_saved_bytes(desc()) >= 40 * 4 and L.mc_cross_entropy_workspace_bytes(desc(), 1) > 0
    fwd = lambda d, *p, n=big: L.mc_cross_entropy_fwd(d, *(p or [256] * 7), n, None)  # noqa: E731
    for k in (dict(B=0), dict(S=0), dict(C=0), dict(V=0), dict(reduction=2), dict(dtype=5), dict(layout=-1)):
        assert fwd(desc(**k)) == -1 and L.mc_cross_entropy_saved_bytes(desc(**k)) == 0
    for k in (dict(B=1 << 31), dict(S=1 << 31), dict(C=1 << 21), dict(V=1 << 21), dict(C=1 << 16, V=1 << 16)):
        assert fwd(desc(**k)) == -6
    for i, n in enumerate([16, 16, 2, 8, 4, 16, 16]):
        p = [256] * 7
        p[i] += n // 2
        assert fwd(desc(), *p) == -1
    for i in (0, 1, 3, 4, 5):
        p = [256] * 7
        p[i] = None
        assert fwd(desc(), *p) == -1
    assert fwd(desc(), n=16) == -3 and L.mc_cross_entropy_bwd(desc(), *[256] * 10, 16, None) == -3
    assert L.mc_cross_entropy_bwd(desc(), None, *[256] * 9, big, None) == -1

    def tensor(**k):
        t = dict(p=256, g=256, m=256, v=256, numel=5, step=1, p_dtype=0, g_dtype=0, bits=32)
        return (_lib.McAdamwTensor * 1)(_lib.McAdamwTensor(**{**t, **k}))
    hyper = lambda **k: _lib.McAdamwHyper(**{**dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0), **k})  # noqa: E731
    step = lambda t, h: L.mc_adamw_step(1, t, h, None)  # noqa: E731
    for k in (dict(numel=-1), dict(step=0), dict(bits=16), dict(p_dtype=3), dict(p=None), dict(m=None), dict(g=258), dict(v=257), dict(bits=8)):
        assert step(tensor(**k), hyper()) == -1
    for k in (dict(p_dtype=1), dict(g_dtype=1), dict(p_dtype=1, g_dtype=1, bits=8, m_scale=256, v_scale=256), dict(master=256)):
        assert step(tensor(**k), hyper()) == -2
    for k in (dict(lr=-1.0), dict(beta1=1.0), dict(beta2=float("nan")), dict(eps=-1.0), dict(weight_decay=-1.0)):
        assert step(tensor(), hyper(**k)) == -1
    for n in ((1 << 63) - 1, 1 << 62, 2048 << 30):
        assert step(tensor(numel=n), hyper()) == -6
    assert L.mc_adamw_step(-1, tensor(), hyper(), None) == -1 and L.mc_adamw_step(0, None, hyper(), None) == 0
    assert L.mc_adamw_moments(1, tensor(), None) == -1


def test_traced_layers_run_again_on_replay(monkeypatch):
    if not host.COMPILED:
        pytest.skip("extension not built: only the Functions exist")
    fake = dict(group_norm_forward=lambda x, w, b, *a: (x * 2, None), cross_entropy_forward=lambda x, w, b, t, *a: (x.sum() * 3, None))
    monkeypatch.setattr(F, "ops", type("Ops", (), {k: staticmethod(v) for k, v in fake.items()}
                                       | {n: staticmethod(getattr(host.impl, n)) for n in ("group_norm_layer", "cross_entropy_layer")}))
    monkeypatch.setattr(F, "group_norm", F._layer_call(F.GroupNormFn, "group_norm_layer"))
    monkeypatch.setattr(F, "cross_entropy", F._layer_call(F.CrossEntropyFn, "cross_entropy_layer"))
    x, z, t = torch.randn(2, 6, 4, 5), torch.randn(2, 6, 4, 5), torch.zeros(2, 4, 5, dtype=torch.int64)
    for layer, more, want in ((mnn.GroupNorm(3, 6), (), z * 2), (mnn.PointwiseCrossEntropy(6, 4), (t,), z.sum() * 3)):
        with warnings.catch_warnings(), torch.no_grad():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(layer, (x, *more), check_trace=False)
        assert torch.equal(traced(z, *more), want)
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda u: layer(u[None], *(m[:1] for m in more)))(x)
