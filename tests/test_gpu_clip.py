"""GPU: norm of many gradients and clipping against the same sums in 64 bits."""
import math

import pytest
import torch

from mappedconvolutions_b200 import dist as mdist
from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
INF = math.inf


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def norm64(ts, p):
    each = [torch.linalg.vector_norm(t.double(), p) for t in ts if t.numel()]
    return torch.linalg.vector_norm(torch.stack(each), p).item() if each else 0.0


def norm_tolerance(ts):
    """float32 sums of eight squares (8 roundings, half of them behind the root) and a rounding of a float32 result; where
    every element is float64, the sums are too"""
    return 2.0 ** -45 if all(t.dtype == F64 for t in ts) else 2.0 ** -20


def close(norm, want, ts):
    assert norm.dim() == 0 and abs(norm.item() - want) <= norm_tolerance(ts) * want, (norm.item(), want)


def check_scaled(src, dst, norm, max_norm):
    """the coefficient is as far off as the norm; it and the product are float32 unless the source is float64; one
    rounding to the destination's type"""
    c = min(1.0, max_norm / (norm + 1e-6))
    for s, d in zip(src, dst):
        tol = torch.finfo(d.dtype).eps / 2 + norm_tolerance(src) + (2.0 ** -51 if s.dtype == F64 else 2.0 ** -23)
        ref = s.double() * c
        assert ((d.double() - ref).abs() <= tol * ref.abs() + torch.finfo(d.dtype).tiny).all()


LISTS = {
    "one": [(1,)],
    "odd": [(3,), (1,), (7, 5), (0,), (8191,), (8192,), (8193,), (2, 3, 5, 7)],
    "layers": [(64, 3, 7), (64,), (256, 256, 7), (256,), (128, 64, 1)] * 3,
    "many": [(17 + i,) for i in range(1300)],
    "large": [(3, 1000, 1001), (5,), (70_000,)],
}


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("types", [(F32,), (BF,), (F64,), (BF, F32, F64)], ids=["f32", "bf16", "f64", "mixed"])
@pytest.mark.parametrize("name", list(LISTS))
def test_norm_and_clip(ops, name, types, p):
    g = torch.Generator("cuda").manual_seed(len(name))
    ts = [(torch.randn(s, generator=g, device="cuda", dtype=F64) * 10.0 ** (i % 5 - 2)).to(types[i % len(types)])
          for i, s in enumerate(LISTS[name])]
    want = norm64(ts, p)
    norm = ops.gradient_norm(ts, p)
    assert norm.dtype == (F64 if F64 in [t.dtype for t in ts] else F32)
    close(norm, want, ts)
    assert torch.equal(norm, ops.gradient_norm(ts, p))  # fixed order
    before = [t.clone() for t in ts]
    for max_norm in (want * 2, want / 3):
        out = [torch.full(t.shape, 7.0, device="cuda", dtype=(t.dtype, F32, BF, F64)[i % 4]) for i, t in enumerate(ts)]
        assert torch.equal(ops.clip_gradients(ts, max_norm, p, out), norm)
        check_scaled(before, out, want, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(ts, before))
    version = ts[0]._version
    assert torch.equal(ops.clip_gradients(ts, want / 3, p), norm)
    check_scaled(before, ts, want, want / 3)
    assert ts[0]._version > version


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-38, 3e18])
def test_squares_neither_overflow_nor_underflow(ops, dtype, scale):
    g = torch.Generator("cuda").manual_seed(1)
    ts = [(torch.randn(n, generator=g, device="cuda", dtype=F64) * scale).to(dtype) for n in (5, 10_000)]
    norm = ops.gradient_norm(ts)
    assert abs(norm.item() - norm64(ts, 2)) <= 2.0 ** -20 * norm64(ts, 2)


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dtype", [F32, BF, F64])
def test_not_finite(ops, dtype, p):
    for at in (0, 4097, 8195):
        t = torch.ones(9000, device="cuda", dtype=dtype)
        t[at] = float("nan")
        other = torch.ones(3, device="cuda", dtype=dtype)
        assert ops.gradient_norm([t, other], p).isnan()
        ops.clip_gradients([t, other], 1.0, p)
        assert t.isnan().all() and other.isnan().all()
        t = torch.ones(9000, device="cuda", dtype=dtype)
        t[at] = -INF
        assert ops.clip_gradients([t], 1.0, p).item() == INF
        assert t[at].isnan() and t.isnan().sum() == 1 and not t.nan_to_num(0.0).any()


def test_zeros_and_nothing(ops):
    z = [torch.zeros(100, device="cuda"), torch.empty(0, device="cuda")]
    assert ops.gradient_norm(z).item() == 0 and ops.clip_gradients(z, 1.0).item() == 0
    assert ops.gradient_norm(z[1:]).item() == 0 and ops.clip_gradients(z[1:], 0.0).item() == 0
    t = [torch.ones(10, device="cuda")]
    ops.clip_gradients(t, 0.0)
    assert not t[0].any()
    with pytest.raises(RuntimeError, match="no tensor"):
        ops.gradient_norm([])


def test_views_and_layouts(ops):
    """any dense order of dimensions as it lies; anything else through a copy; nothing around a view is touched"""
    g = torch.Generator("cuda").manual_seed(4)
    base = torch.randn(12, 10, 8, generator=g, device="cuda")
    keep = base.clone()
    views = [base[1:3], base[4, 1:], base[6:, 3:5, ::2]]  # dense at an odd start, dense, strided
    views.append(torch.randn(4, 6, 3, 5, generator=g, device="cuda").to(memory_format=torch.channels_last))
    views.append(torch.randn(33, generator=g, device="cuda").to(BF)[1:])
    before = [v.clone() for v in views]
    want = norm64(before, 2)
    close(ops.gradient_norm(views), want, views)
    out = [torch.zeros(v.shape, device="cuda") for v in views]  # other strides than the gradients'
    ops.clip_gradients(views, want / 2, 2.0, out)
    check_scaled(before, out, want, want / 2)
    close(ops.clip_gradients(views, want / 2), want, views)
    check_scaled(before, views, want, want / 2)
    mask = torch.ones_like(base, dtype=torch.bool)
    for v in (mask[1:3], mask[4, 1:], mask[6:, 3:5, ::2]):
        v.fill_(False)
    assert torch.equal(base[mask], keep[mask])


def test_refusals(ops):
    t = torch.randn(100, device="cuda")
    other = torch.randn(100, device="cuda")
    for call in (lambda: ops.gradient_norm([t.cpu()]), lambda: ops.gradient_norm([t, t.cpu()]),
                 lambda: ops.gradient_norm([t.half()]), lambda: ops.gradient_norm([t.long()]),
                 lambda: ops.gradient_norm([t], 3.0), lambda: ops.gradient_norm([t], -INF),
                 lambda: ops.clip_gradients([t], -1.0), lambda: ops.clip_gradients([t], float("nan")),
                 lambda: ops.clip_gradients([t, other], 1.0, 2.0, [other]),
                 lambda: ops.clip_gradients([t], 1.0, 2.0, [other[:50]]),
                 lambda: ops.clip_gradients([t], 1.0, 2.0, [other.half()]),
                 lambda: ops.clip_gradients([t, t], 1.0),                        # the same tensor twice
                 lambda: ops.clip_gradients([t[:60], t[40:]], 1.0),              # overlapping pieces of one buffer
                 lambda: ops.clip_gradients([t, other], 1.0, 2.0, [other, t]),   # one's result is another's input
                 lambda: ops.clip_gradients([t[:99]], 1.0, 2.0, [t[1:]]),
                 lambda: ops.clip_gradients([torch.ones(1, device="cuda").expand(5)], 1.0)):
        keep = t.clone()
        with pytest.raises(RuntimeError):
            call()
        assert torch.equal(t, keep)
    ops.gradient_norm([t, t])                            # reading twice is no conflict
    ops.clip_gradients([t[:50], t[50:]], 1.0)            # neighbours in one bucket are none either


def test_strided_results_given_twice(ops):
    t = torch.randn(6, 8, device="cuda")
    for call in (lambda: ops.clip_gradients([t[:, ::2], t[:, ::2]], 1.0), lambda: ops.clip_gradients([t[:, :3], t], 1.0)):
        keep = t.clone()
        with pytest.raises(RuntimeError, match="share memory"):
            call()
        assert torch.equal(t, keep)
    want = t * (0.5 / (t.double().square().sum().sqrt() + 1e-6)).float()
    ops.clip_gradients([t[:, ::2], t[:, 1::2]], 0.5)     # what lies between them is another's
    # (the norm is a double sum of float32 sums of eight squares: the coefficient is off by 8 roundings at most, and its own)
    assert ((t - want).abs() <= 10 * 2.0 ** -24 * want.abs()).all()


def test_dist_entry_points():
    g = torch.Generator("cuda").manual_seed(8)
    ts = [torch.randn(64, 3, 7, generator=g, device="cuda"), None, torch.randn(64, generator=g, device="cuda").to(BF)]
    some = [t for t in ts if t is not None]
    before = [t.clone() for t in some]
    want = norm64(some, 2)
    close(mdist.gradient_norm(ts), want, some)
    out = [torch.zeros(64, 3, 7, device="cuda"), None, torch.zeros(64, device="cuda")]
    close(mdist.clip_gradients(ts, 1.0, out=out), want, some)
    check_scaled(before, [out[0], out[2]], want, 1.0)
    close(mdist.clip_gradients(ts, 1.0), want, some)
    check_scaled(before, some, want, 1.0)
    assert mdist.gradient_norm([None]) is None and mdist.clip_gradients([], 1.0) is None


def test_captured_and_on_another_stream():
    ts = [torch.randn(n, device="cuda") for n in (5, 100_000)]
    out = [torch.empty_like(t) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mdist.clip_gradients(ts, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = mdist.clip_gradients(ts, 1.0, out=out)
    for scale in (2.0, 0.25):
        for t in ts:
            t.copy_(torch.randn_like(t) * scale)
        graph.replay()
        want = norm64(ts, 2)
        close(norm, want, ts)
        check_scaled(ts, out, want, 1.0)


def test_training_step_of_the_new_layers():
    """layers, gradients, norm and clipping as a training loop chains them, against torch's own clipping"""
    from mappedconvolutions_b200 import nn as mnn
    torch.manual_seed(0)
    block = torch.nn.ModuleList([mnn.PointwiseConvolution(6, 32, activation="gelu"), mnn.GatedFeedForward(32, 64)]).cuda()
    x = torch.randn(2, 6, 10, 30, device="cuda")
    h = block[0](x)
    (block[1](h, h) ** 2).sum().backward()
    grads = [p.grad for p in block.parameters()]
    copies = [g.clone() for g in grads]
    want = norm64(copies, 2)
    close(mdist.clip_gradients(grads, 0.5), want, copies)
    check_scaled(copies, grads, want, 0.5)
    assert norm64(grads, 2) <= 0.5 * (1 + 2.0 ** -18)
