"""GPU: the paths that the channel-mixing kernels take for large layers, and what they leave behind."""
import math

import pytest
import torch

import mix_reference as R
import mix_strict as M
from mappedconvolutions_b200 import host

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def image(g, shape, dtype, layout, scale=1.0):
    t = (torch.randn(shape, generator=g, device="cuda", dtype=F32) * scale).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


def params(g, n_out, n_in, dtype):
    s = 1 / math.sqrt(n_in)
    u = lambda *shape: ((torch.rand(shape, generator=g, device="cuda") * 2 - 1) * s).to(dtype)
    return u(n_out, n_in, 1), u(n_out)


@pytest.mark.parametrize("channels", [(16, 8), (136, 320), (512, 64)])
def test_short_kernels_one_behind_the_other(channels):
    """blocks that end a few microseconds after they start, the next kernel's already waiting: a block may leave only when
    every arrival and copy of its pair has come"""
    cin, cout = channels
    g = torch.Generator("cuda").manual_seed(cin)
    x, gy = image(g, (1, cin, 1, 300), BF, "nhwc"), image(g, (1, cout, 1, 300), BF, "nhwc")
    w, b = params(g, cout, cin, BF)
    y0, saved = host.impl.pointwise_forward(x, w, b, None, 4, True)
    g0 = host.impl.pointwise_backward(gy, saved, x, w, b, 4)
    for _ in range(100):
        y, saved = host.impl.pointwise_forward(x, w, b, None, 4, True)
        got = host.impl.pointwise_backward(gy, saved, x, w, b, 4)
    assert torch.equal(y, y0) and all(torch.equal(p, q) for p, q in zip(got, g0))


def test_waits_of_both_kinds_of_kernels_are_reported():
    """the convolutions' and the channel-mixing kernels' status words, one code a call, none cleared unread"""
    from mappedconvolutions_b200 import _lib
    L, st = _lib.lib(), torch.cuda.current_stream().cuda_stream
    assert L.mc_device_status(st, 1) == 0
    seen = torch.zeros(2, dtype=torch.int32, device="cuda")
    _lib.check(L.mc_selftest_mix_wait_expiry(seen[:1].data_ptr(), st))
    _lib.check(L.mc_selftest_wait_expiry(seen[1:].data_ptr(), st))
    assert L.mc_device_status(st, 0) == 0x7F1 and seen.tolist() == [2, 2]
    assert [L.mc_device_status(st, 1) for _ in range(3)] == [0x7F1, 0x7F2, 0]
    _lib.check(L.mc_selftest_mix_wait_expiry(None, st))
    assert [L.mc_device_status(st, r) for r in (0, 1, 0)] == [0x7F2, 0x7F2, 0]


@pytest.mark.parametrize("i", range(len(M.PATHS)))
def test_paths(i):
    """every way of dividing the products, as the table beside the reference says"""
    from mappedconvolutions_b200 import _lib
    case, ways = M.PATHS[i]
    b, h, w, cin, hidden, cout, layout, name, residual = case
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert {k: M.plan(_lib.lib(), M.path_desc(case), k, 0)[0] for k in ways} == ways
    g = torch.Generator("cuda").manual_seed(50 + i)
    x, gy = image(g, (b, cin, h, w), BF, layout), image(g, (b, cout, h, w), BF, layout, 0.01)
    r = image(g, (b, cout, h, w), BF, layout) if residual else None
    act = R.ACTS[name]
    if hidden:
        wi, bi = params(g, 2 * hidden, cin, BF)
        wo, bo = params(g, cout, hidden, BF)
        y, saved = host.impl.gated_forward(x, wi, bi, wo, bo, r, act, True)
        call = lambda: host.impl.gated_backward(gy, saved, x, wi, bi, wo, act)
        names, want = ("gx", "gw_in", "gb_in", "gw_out", "gb_out"), M.gated(x, wi, bi, wo, bo, r, name, gy)
    else:
        weight, bias = params(g, cout, cin, BF)
        y, saved = host.impl.pointwise_forward(x, weight, bias, r, act, True)
        call = lambda: host.impl.pointwise_backward(gy, saved, x, weight, bias, act)
        names, want = ("gx", "gw", "gb"), M.pointwise(x, weight, bias, r, name, gy)
    grads = call()
    R.check(dict(zip(names, grads), y=y), want, str(case))
    assert all(torch.equal(p, q) for p, q in zip(grads, call()))  # fixed order of every sum


def test_parameter_gradients_of_a_thousand_million_pixels():
    """Sums whose terms have one sign, where what a sum loses does not cancel.  A share is 2^17 pixels at most: 2^13 additions
    to an accumulator that truncates (at most 2^-23 of it, 2^-10 in all), 2^13 float32 additions of a column's sum (2^-11),
    half a bf16 step of the result (2^-8), and float32 sums of 2^13 shares in 32 parts (2^-15)."""
    g = torch.Generator("cuda").manual_seed(61)
    block, times = (torch.rand(1 << 16, 8, generator=g, device="cuda") + 0.5).to(BF), 1 << 14
    x = block.repeat(times, 1).view(1, 1, -1, 8).permute(0, 3, 1, 2)
    w, b = torch.zeros(8, 8, 1, device="cuda", dtype=BF), torch.zeros(8, device="cuda", dtype=BF)
    _, gw, gb = host.impl.pointwise_backward(x, None, x, w, b, 0, False, True)
    d = block.double()
    off = [((got.double() - want) / want).abs().max().item()
           for got, want in ((gw[:, :, 0], d.T @ d * times), (gb, d.sum(0) * times))]
    assert max(off) <= 2.0 ** -8 + 2.0 ** -10 + 2.0 ** -15, off


@pytest.mark.parametrize("binding", ["ctypes", "compiled"])
def test_channel_counts_beyond_32_bits_are_refused(binding):
    """2^32 + 8 channels are not eight"""
    from mappedconvolutions_b200 import ops as twin
    ops = twin if binding == "ctypes" else host.impl
    n = (1 << 32) + 8
    x = torch.empty(1, n, 1, 1, device="cuda", dtype=BF)
    w, b = torch.empty(1, n, 1, device="cuda", dtype=BF), torch.empty(1, device="cuda", dtype=BF)
    with pytest.raises(RuntimeError, match="size beyond"):
        ops.pointwise_forward(x, w, b)
    with pytest.raises(RuntimeError, match="size beyond"):
        ops.pointwise_backward(b.view(1, 1, 1, 1), None, x, w, b)
    with pytest.raises(RuntimeError, match="size beyond"):
        ops.gated_forward(b.view(1, 1, 1, 1), torch.empty(2 * (n // 2), 1, 1, device="cuda", dtype=BF), torch.empty(n, device="cuda", dtype=BF),
                          torch.empty(1, n // 2, 1, device="cuda", dtype=BF), b)
