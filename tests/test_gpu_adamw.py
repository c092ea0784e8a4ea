"""GPU: AdamW over many tensors against the same step in 64 bits; moments in 8 bits against the definition of their codes."""
import copy
import math

import pytest
import torch

from mappedconvolutions_b200 import host, ops as twin
from mappedconvolutions_b200 import dist as mdist, nn as mnn
from mappedconvolutions_b200.optim import AdamW

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


# A plain implementation of the codes: float32 operations of torch, one rounding each
def rows256(t):
    t = t.reshape(-1)
    return torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)


def scales(largest, codes):
    s = largest * torch.tensor(1.0 / codes, dtype=F32, device=largest.device)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    return s, torch.where(s == 0, torch.zeros_like(s), torch.ones_like(s) / s)


def encode(m, v):
    a, r = rows256(m), torch.sqrt(rows256(v))
    s, i = scales(a.abs().amax(1, keepdim=True), 127.0 ** 2)
    q, j = scales(r.amax(1, keepdim=True), 255.0 ** 2)
    c = torch.sqrt(a.abs() * i).round().clamp(max=127) * a.sign()
    d = torch.sqrt(r * j).round().clamp(max=255)
    d = torch.where((r > 0) & (q > 0), d.clamp(min=1), d)
    cut = lambda t, k: t.to(k).reshape(-1)[:m.numel()].view(m.shape)  # noqa: E731
    return cut(c, torch.int8), s[:, 0].contiguous(), cut(d, torch.uint8), q[:, 0].contiguous()


def values(c, s, d, q):
    a, r = rows256(c.float()), rows256(d.float())
    m, v = a * a.abs() * s[:, None], (r * r * q[:, None]).square()
    cut = lambda t: t.reshape(-1)[:c.numel()].view(c.shape)  # noqa: E731
    return cut(m), cut(v)


def moments32(m, v, g, beta1, beta2):
    """float32, each operation rounded"""
    f = lambda x: torch.tensor(x, dtype=F32, device=m.device)  # noqa: E731
    return m * f(beta1) + g.float() * f(1 - beta1), v * f(beta2) + g.float() * g.float() * f(1 - beta2)


def step64(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay):
    """also what the update is made of: m = beta1 m + (1 - beta1) g may cancel, and its roundings are 2^-24 of either term, not of
    their sum; what follows are products and quotients, a few 2^-24 of the result"""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    size = beta1 * m.abs() + (1 - beta1) * g.abs()
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    rate = lr / (1 - beta1 ** step) / (v.sqrt() / math.sqrt(1 - beta2 ** step) + eps)
    return p * (1 - lr * weight_decay) - rate * m, m, v, rate * size


def close(got, want, parts, u):
    """u: half a step of the result's type; `parts`: the sizes of what was added up, each a few float32 roundings off"""
    f = 2.0 ** -50 if got.dtype == F64 else 2.0 ** -21
    bound = u * want.abs() + f * parts + 1e-38
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()


SHAPES = {"one": [(1,)], "odd": [(3,), (1,), (7, 5), (0,), (255,), (256,), (257,), (2047,), (2049,), (2, 3, 5, 7)],
          "layers": [(64, 3, 7), (64,), (256, 256, 7), (256,)], "many": [(17 + 3 * i,) for i in range(600)]}
KINDS = [(F32, F32, 32, False), (F32, BF, 32, False), (BF, BF, 32, False), (BF, F32, 32, False), (BF, BF, 32, True), (BF, F32, 32, True),
         (F64, F64, 32, False), (F32, F32, 8, False), (F32, BF, 8, False), (BF, BF, 8, False), (BF, F32, 8, False), (BF, BF, 8, True),
         (BF, F32, 8, True)]


def problem(name, kinds, seed=0, size=1.0):
    """lists as adamw_step takes them; the i-th tensor is of kind i modulo their number"""
    gen = torch.Generator("cuda").manual_seed(seed)
    lists = [[] for _ in range(8)]
    for i, shape in enumerate(SHAPES[name]):
        pt, gt, bits, master = kinds[i % len(kinds)]
        wide = F64 if pt == F64 else F32
        rand = lambda: torch.randn(shape, generator=gen, device="cuda", dtype=F64)  # noqa: E731
        scale = size * 10.0 ** (i % 5 - 2)
        w, g, m, v = rand(), rand() * scale, (rand() * 0.3 * scale).to(wide), (rand().square() * scale ** 2 + 1e-3 * scale ** 2).to(wide)
        lists[0].append(w.to(pt))
        lists[1].append(g.to(gt))
        if bits == 8:
            c, s, d, q = encode(m, v)
        else:
            c, s, d, q = m, None, v, None
        for k, t in zip((2, 3, 4, 5, 6), (c, d, s, q, w.float() if master else None)):
            lists[k].append(t)
        lists[7].append(1 + i % 7 * 50)
    return lists


def copied(lists):
    return [[t.clone() if torch.is_tensor(t) else t for t in v] for v in lists]


@pytest.mark.parametrize("name", list(SHAPES))
@pytest.mark.parametrize("kinds", [[k] for k in KINDS] + [KINDS], ids=lambda k: "mixed" if len(k) > 1 else "-".join(str(x).split(".")[-1] for x in k[0]))
def test_step(ops, kinds, name):
    lists = problem(name, kinds)
    before = copied(lists)
    version = lists[0][0]._version
    ops.adamw_step(*lists, **HYPER)
    assert lists[0][0]._version > version and lists[2][0]._version > 0
    for p, g, m, v, s, q, w, step, p0, g0, m0, v0, s0, q0, w0, _ in zip(*lists, *before):
        assert torch.equal(g, g0)
        if p.numel() == 0:
            continue
        old_m, old_v = (m0, v0) if s0 is None else values(m0, s0, v0, q0)
        want_p, want_m, want_v, update = step64(p0 if w0 is None else w0, g0, old_m, old_v, step, **HYPER)
        parts = (p0 if w0 is None else w0).double().abs() + update.abs()
        close(p if w is None else w, want_p, parts, torch.finfo((p if w is None else w).dtype).eps / 2)
        if w is not None:
            assert torch.equal(p, w.to(BF))
        if s is None:
            close(m, want_m, (old_m.double().abs() + g0.double().abs()), 0)
            close(v, want_v, want_v, 0)
        else:
            codes = encode(*moments32(old_m, old_v, g0, HYPER["beta1"], HYPER["beta2"]))
            for a, b in zip((m, s, v, q), codes):
                assert torch.equal(a, b)
            # and what they stand for is the nearest that there is, in 64 bits
            block = lambda t: t.double().repeat_interleave(256)[:m.numel()].view(m.shape)  # noqa: E731
            assert ((want_m.abs() / block(s)).nan_to_num(0).sqrt() - m.double().abs()).abs().max() <= 0.5 + 1e-4
            root = (want_v.sqrt() / block(q)).nan_to_num(0).sqrt()
            assert ((root - v.double()).abs()[root > 0.5]).max() <= 0.5 + 1e-4
            assert (v[want_v > 0] > 0).all()
    again = copied(before)
    ops.adamw_step(*again, **HYPER)
    for a, b in zip(lists[:7], again[:7]):
        assert all(x is y is None or torch.equal(x, y) for x, y in zip(a, b))


def test_moments_of_codes(ops):
    lists = problem("odd", [k for k in KINDS if k[2] == 8])
    m, v = ops.adamw_moments(lists[2], lists[3], lists[4], lists[5])
    for a, b, c, d, s, q in zip(m, v, *lists[2:6]):
        want = values(c, s, d, q)
        assert a.dtype == F32 and torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.parametrize("size", [1e-25, 1e-19, 1e15])
def test_8_bits_of_small_and_large_gradients(ops, size):
    """moments far below and above one; squares that float32 does not hold are zero or, as in float32, infinite"""
    lists = problem("odd", [(F32, F32, 8, False)], 3, size)
    before = copied(lists)
    ops.adamw_step(*lists, **HYPER)
    for p, m, v, s, q, g0, m0, v0, s0, q0 in zip(lists[0], *lists[2:6], before[1], *before[2:6]):
        codes = encode(*moments32(*values(m0, s0, v0, q0), g0, HYPER["beta1"], HYPER["beta2"]))
        assert all(torch.equal(a, b) for a, b in zip((m, s, v, q), codes)) and p.isfinite().all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite_gradients(ops, bits, value):
    lists = problem("layers", [(F32, F32, bits, False)])
    lists[1][2].view(-1)[1000] = value
    clean = copied(lists)
    clean[1][2].view(-1)[1000] = 0.0
    for v in (lists, clean):
        ops.adamw_step(*v, **HYPER)
    p, q = lists[0][2].view(-1), clean[0][2].view(-1)
    assert p[1000].isnan()
    keep = torch.ones_like(p, dtype=torch.bool)
    keep[1000] = False
    assert torch.equal(p[keep], q[keep])
    m = lists[2][2] if bits == 32 else ops.adamw_moments(*lists[2:6])[0][2]
    bad = ~m.view(-1).isfinite()
    assert bad[1000] and bad.sum() == (1 if bits == 32 else 256) and (bits == 32 or bad[768:1024].all())


def test_zeros(ops):
    for bits in (8, 32):
        lists = problem("odd", [(F32, F32, bits, False)])
        for k in range(1, 6):
            for t in lists[k]:
                if t is not None:
                    t.zero_()
        before = copied(lists)
        ops.adamw_step(*lists, **{**HYPER, "weight_decay": 0.0})
        for a, b in zip(lists[:6], before[:6]):
            assert all(x is y is None or torch.equal(x, y) for x, y in zip(a, b))


def test_views_orders_and_offsets(ops):
    """parameters that start anywhere, in any dense order; gradients in another order"""
    gen = torch.Generator("cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    for bits in (32, 8):
        base = rand(4000)
        p = [base[1:1201].view(30, 40), rand(8, 6, 5, 4).contiguous(memory_format=torch.channels_last)]
        g = [rand(40, 30).t(), rand(8, 6, 5, 4)]
        m = [torch.zeros_like(t, dtype=torch.int8 if bits == 8 else F32) for t in p]
        v = [torch.zeros_like(t, dtype=torch.uint8 if bits == 8 else F32) for t in p]
        s, q = ([torch.zeros((t.numel() + 255) // 256, device="cuda") if bits == 8 else None for t in p] for _ in range(2))
        want = [step64(a, b, torch.zeros_like(a), torch.zeros_like(a), 1, **HYPER) for a, b in zip(p, g)]
        rest = base.clone()
        ops.adamw_step(p, g, m, v, s, q, [None] * 2, [1, 1], **HYPER)
        for a, (w, _, _, u) in zip(p, want):
            close(a, w, w.abs() + u.abs(), 2.0 ** -24)
        assert torch.equal(base[:1], rest[:1]) and torch.equal(base[1201:], rest[1201:])


def test_refusals(ops):
    def call(change, hyper=HYPER):
        lists = problem("layers", [(F32, F32, 32, False)])
        change(lists)
        ops.adamw_step(*lists, **hyper)

    def put(k, t, i=0):
        return lambda v: v[k].__setitem__(i, t(v[k][i]) if callable(t) else t)
    strided = torch.zeros(64, 3, 14, device="cuda")[:, :, ::2]
    for change, text in [(put(0, lambda t: t.half()), "dtype"), (put(1, lambda t: t.double()), "gradient"), (put(1, lambda t: t[:1]), "gradient"),
                         (put(1, lambda t: t.cpu()), "CUDA only"), (put(2, lambda t: t.bfloat16()), "moments"),
                         (put(2, lambda t: t.to(torch.int8)), "moments"), (put(3, lambda t: t[:1]), "moments"),
                         (put(0, strided), "gaps"), (put(4, torch.zeros(6, device="cuda")), "scales"),
                         (put(6, lambda t: torch.zeros(64, 3, 7, device="cuda")), "master"), (put(7, 0), "counted"),
                         (lambda v: v[0].__setitem__(1, v[0][0].view(-1)[:64]), "share memory"),
                         (lambda v: v[2].__setitem__(0, v[1][0]), "share memory"), (lambda v: v[7].pop(), "entries"),
                         (lambda v: v[1].__setitem__(0, v[1][0].to_sparse()), "")]:
        with pytest.raises(RuntimeError, match=text):
            call(change)
    for bad in (dict(lr=-1.0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(weight_decay=float("nan"))):
        with pytest.raises(RuntimeError, match="bad argument"):
            call(lambda v: None, {**HYPER, **bad})
    with pytest.raises(RuntimeError, match="no tensor"):
        ops.adamw_step(*[[]] * 8, **HYPER)


@pytest.mark.parametrize("dtype", [F32, F64])
def test_many_steps_as_torch(dtype):
    gen = torch.Generator("cuda").manual_seed(6)
    shapes = [(40, 30), (7,), (300, 5)]
    mine = [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda", dtype=dtype)) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().double()) for p in mine]
    args = dict(lr=1e-2, betas=(0.8, 0.95), eps=1e-7, weight_decay=0.05)
    a, b = AdamW(mine, **args), torch.optim.AdamW(theirs, **args)
    for k in range(20):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            p.grad = None if k % 3 == i else torch.randn(p.shape, generator=gen, device="cuda", dtype=dtype)
            q.grad = None if p.grad is None else p.grad.double()
        a.step()
        b.step()
    for p, q in zip(mine, theirs):
        assert a.state[p]["step"] == int(b.state[q]["step"])
        # 20 updates of at most 2 lr, the roundings of each a few 2^-24 of it and of the parameter
        assert ((p - q).abs() <= 20 * (2.0 ** -21 if dtype == F32 else 2.0 ** -48) * (q.abs() + 0.02)).all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_state_dict(bits, master):
    def make():
        return [torch.nn.Parameter(torch.randn(33, 20, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF))]

    def steps(params, opt, seeds):
        for k in seeds:
            params[0].grad = torch.randn(33, 20, generator=torch.Generator("cuda").manual_seed(k), device="cuda").to(BF)
            opt.step()
    one, two = make(), make()
    a = AdamW(one, state_bits=bits, master_weights=master)
    steps(one, a, range(5))
    kept = copy.deepcopy(a.state_dict())
    with torch.no_grad():
        two[0].copy_(one[0])
    b = AdamW(two)  # (what the state was kept in comes with it)
    b.load_state_dict(kept)
    assert b.state[two[0]]["exp_avg"].dtype == (torch.int8 if bits == 8 else F32) and ("master" in b.state[two[0]]) == master
    steps(one, a, range(5, 9))
    steps(two, b, range(5, 9))
    assert torch.equal(one[0], two[0])
    for x, y in zip(a.moments()[0], b.moments()[0]):
        assert x.dtype == F32 and torch.equal(x, y)


def test_state_of_torch():
    """a checkpoint of torch.optim.AdamW goes on as float32 moments"""
    gen = torch.Generator("cuda").manual_seed(2)
    mine, theirs = (torch.nn.Parameter(torch.ones(50, 7, device="cuda")) for _ in range(2))
    a, b = AdamW([mine], lr=0.1), torch.optim.AdamW([theirs], lr=1e-2, weight_decay=0.3)
    for k in range(6):
        theirs.grad = torch.randn(50, 7, generator=gen, device="cuda")
        if k == 3:
            with torch.no_grad():
                mine.copy_(theirs)
            a.load_state_dict(copy.deepcopy(b.state_dict()))
            assert a.param_groups[0]["lr"] == 1e-2 and a.param_groups[0]["state_bits"] == 32
        b.step()
        if k >= 3:
            mine.grad = theirs.grad
            a.step()
    assert a.state[mine]["step"] == 6
    assert ((mine - theirs).abs() <= 3 * 2.0 ** -20 * (theirs.abs() + 0.02)).all()  # three updates, some roundings each


def test_capture_is_refused():
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    p.grad = torch.ones(10, device="cuda")
    opt = AdamW([p])
    opt.step()
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros(1, device="cuda")
    with torch.cuda.graph(graph):
        out += 1
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    graph.replay()
    assert out.item() == 1 and opt.state[p]["step"] == 1


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_a_training_step(dtype):
    """convolution, norm, classification loss, clipping and the optimiser together, against torch's own in 64 bits"""
    g = torch.Generator("cuda").manual_seed(9)
    H, W, K = 12, 16, 4
    torch.manual_seed(3)
    conv, norm, head = mnn.MappedConvolution(8, 24, K, "nearest"), mnn.GroupNorm(4, 24, activation="silu"), mnn.PointwiseCrossEntropy(24, 40)
    layers = [l.to("cuda").to(dtype) for l in (conv, norm, head)]
    params = [p for l in layers for p in l.parameters()]
    wide = [p.detach().double().requires_grad_(True) for p in params]
    ys, xs = torch.meshgrid(torch.arange(H), torch.arange(W), indexing="ij")
    taps = torch.stack([torch.stack([(xs + i) % W, (ys + j) % H], -1) for i in (0, 1) for j in (0, 1)], 2).cuda()
    x = torch.randn(3, 8, H, W, generator=g, device="cuda").to(dtype).contiguous(memory_format=torch.channels_last)
    target = torch.randint(0, 40, (3, H, W), generator=g, device="cuda")
    target[:, 0] = -100
    opt = AdamW(params, lr=1e-2, master_weights=dtype == BF)
    ref = torch.optim.AdamW(wide, lr=1e-2)
    for _ in range(2):
        loss = head(norm(conv(x, taps.float())), target)
        grads = torch.autograd.grad(loss, params)
        for p, q in zip(params, grads):
            p.grad = q
        total = mdist.clip_gradients([p.grad for p in params], 0.05)
        opt.step()
        f = torch.nn.functional
        cols = x.double()[:, :, taps[..., 1], taps[..., 0]]
        z = torch.einsum("ock,bchwk->bohw", wide[0], cols) + wide[1][:, None, None]
        z = f.silu(f.group_norm(z, 4, wide[2], wide[3]))
        want = f.cross_entropy(torch.einsum("oc,bchw->bohw", wide[4][:, :, 0], z) + wide[5][:, None, None], target)
        ref.zero_grad()
        want.backward()
        norm64 = torch.nn.utils.clip_grad_norm_(wide, 0.05)
        tol = 2e-2 if dtype == BF else 1e-4
        assert abs(loss.item() - want.item()) <= tol * want.item() and abs(total.item() - norm64.item()) <= 2 * tol * norm64.item()
        for p, q in zip(params, wide):
            assert (p.grad.double() - q.grad).norm() <= 2 * tol * q.grad.norm()
        with torch.no_grad():  # the next pass from the same point: Adam's first steps are signs, and a rounding may turn one
            ref.step()
            for p, q in zip(params, wide):
                q.copy_(p)
