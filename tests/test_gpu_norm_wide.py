"""GPU: group normalisation of more channels than a block holds vectors of."""
import pytest
import torch

import step_reference as R
from mappedconvolutions_b200 import host, ops as twin

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(params=["ctypes", "compiled"])
def ops(request):
    return twin if request.param == "ctypes" else host.impl


def image(g, shape, dtype, layout, scale=1.0, offset=0.0):
    t = (torch.randn(shape, generator=g, device="cuda", dtype=F64) * scale + offset).to(dtype)
    return t.contiguous(memory_format=torch.channels_last) if layout == "nhwc" else t


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype,channels,groups", [(F64, 1200, 8), (F64, 1536, 48), (F64, 515, 5), (F64, 2049, 3), (F32, 2100, 20), (F32, 3001, 1)])
@pytest.mark.parametrize("offset", [0.0, 1e4, -1e4])
def test_values_far_from_zero(ops, dtype, channels, groups, layout, offset):
    """every group as accurate as the first: groups that lie in later columns of vectors among them"""
    g = torch.Generator("cuda").manual_seed(1)
    shape = (2, channels, 3, 5)
    x, gy = image(g, shape, dtype, layout, 1.0, offset), image(g, shape, dtype, layout)
    w, b = (torch.randn(channels, generator=g, device="cuda").to(dtype) for _ in range(2))
    y, stats = ops.group_norm_forward(x, w, b, groups, 1e-5, R.ACTS["silu"])
    got = dict(zip(("gx", "gw", "gb"), ops.group_norm_backward(gy, stats, x, w, b, groups, 1e-5, R.ACTS["silu"])))
    # (x - offset is exact, and its normalised values are the same: the formulas' own sums in 64 bits are off by steps of the mean)
    want, near = (R.group_norm(t, w, b, groups, 1e-5, "silu", gy) for t in (x, x - offset))
    assert torch.equal((x - offset).double(), x.double() - offset) and torch.equal(x.double() - offset + offset, x.double())
    R.check(dict(y=y, **got), {k: (near[k][0], want[k][1]) for k in want}, (channels, groups, offset))
    rstd = stats.view(F64 if dtype == F64 else F32).view(2, groups, 2)[:, :, 1].double()
    var = x.double().contiguous().reshape(2, groups, -1).var(2, unbiased=False)
    # Runs of up to 33 differences, merged in double: see the bound of rstd in step_reference.  And the means of a thread's run and of a
    # tile are each rounded to half a step of |mean|, d in all: the variance of the means changes by 2 sum n_i (mean_i - mean) d_i / n,
    # at most 2 d deviations, rstd by d / deviation of itself.  (Squares of means instead of differences: 10^8 steps of float64.)
    t = R.Bounds(dtype)
    far = 2 * t.step * (abs(offset) + 1) * rstd
    assert ((rstd * (var + 1e-5).sqrt() - 1).abs() <= t.sum(256) + 4 * t.step + 2.0 ** -50 + far).all()


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [F32, F64], ids=["f32", "f64"])
@pytest.mark.parametrize("shape,groups", [((3, 64, 40, 50), 4), ((2, 48, 1, 15), 48), ((1, 30, 9, 33), 5), ((1, 8, 1, 40962), 1), ((40, 32, 2, 7), 2)])
def test_means_far_from_zero(ops, shape, groups, dtype, layout):
    """A mean is off by roundings of itself where runs, tiles and the group leave theirs, half a step each, and by those of the
    differences."""
    g = torch.Generator("cuda").manual_seed(2)
    t = R.Bounds(dtype)
    for offset in (1e4, -3.7e5, 1.7):
        x = image(g, shape, dtype, layout, 1.0, offset)
        stats = ops.group_norm_forward(x, None, None, groups)[1].view(dtype).view(shape[0], groups, 2)
        rows = x.double().contiguous().reshape(shape[0], groups, -1)
        mean = rows[:, :, :1] + (rows - rows[:, :, :1]).mean(2, keepdim=True)
        dev = (rows - mean).abs().mean(2)
        assert ((stats[:, :, 0].double() - mean[:, :, 0]).abs() <= 3 * t.step * mean[:, :, 0].abs() + t.sum(256) * dev).all(), offset


# rows of several columns of vectors: one pixel or some to a row, fewer pixels than a row has, groups of one channel, within columns and over
# them, one group, ends around the last channel; one column and one vector more
SHAPES = [((1, 1 << 20, 1, 1), 1 << 10), ((2, 70_000, 1, 1), 7), ((3, 5000, 2, 3), 8), ((1, 30_011, 1, 5), 1), ((1, 30_011, 1, 5), 30_011),
          ((2, 4100, 1, 2), 2050), ((2, 4100, 1, 2), 1), ((2, 4100, 4, 5), 41), ((1, 2049, 1, 3), 3), ((1, 2049, 3, 11), 683), ((2, 2056, 2, 4), 257),
          ((1, 16_385, 1, 1), 5), ((1, 16_385, 1, 9), 3277), ((4, 8192, 5, 7), 16), ((2, 6150, 1, 4), 2), ((2, 257, 5, 8), 257), ((1, 1025, 7, 7), 41)]


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("dtype", [BF, F32, F64], ids=["bf16", "f32", "f64"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_many_channels(ops, i, dtype, layout):
    shape, groups = SHAPES[i]
    g = torch.Generator("cuda").manual_seed(i)
    x, gy = image(g, shape, dtype, layout, 2.0, 0.5), image(g, shape, dtype, layout)
    w, b = (torch.randn(shape[1], generator=g, device="cuda").to(dtype) for _ in range(2))
    name = [None, "relu", "silu"][i % 3]
    y, stats = ops.group_norm_forward(x, w, b, groups, 1e-5, R.ACTS[name])
    got = dict(zip(("gx", "gw", "gb"), ops.group_norm_backward(gy, stats, x, w, b, groups, 1e-5, R.ACTS[name])))
    R.check(dict(y=y, **got), R.group_norm(x, w, b, groups, 1e-5, name, gy), SHAPES[i])
    again = ops.group_norm_forward(x, w, b, groups, 1e-5, R.ACTS[name])
    assert torch.equal(y, again[0]) and torch.equal(stats, again[1])
    assert torch.equal(got["gx"], ops.group_norm_backward(gy, stats, x, w, b, groups, 1e-5, R.ACTS[name])[0])


@pytest.mark.parametrize("layout", ["nhwc", "nchw"])
@pytest.mark.parametrize("shape,groups", [((1 << 21, 64, 1, 1), 32), ((1 << 20, 64, 1, 3), 64), ((70, 1 << 20, 1, 1), 1 << 20)])
def test_many_groups(shape, groups, layout):
    """2^26 groups and more: the first, the last and images between them against the formulas"""
    g = torch.Generator("cuda").manual_seed(7)
    assert shape[0] * groups >= 1 << 26
    x, gy = (torch.empty(shape, dtype=BF, device="cuda", memory_format=torch.channels_last if layout == "nhwc" else torch.contiguous_format).normal_(generator=g)
             for _ in range(2))
    w, b = (torch.randn(shape[1], generator=g, device="cuda").to(BF) for _ in range(2))
    y, stats = host.impl.group_norm_forward(x, w, b, groups, 1e-5, 1)
    gx, gw, gb = host.impl.group_norm_backward(gy, stats, x, w, b, groups, 1e-5, 1)
    for at in (slice(0, 3), slice(shape[0] // 2, shape[0] // 2 + 3), slice(shape[0] - 3, shape[0])):
        want = R.group_norm(x[at], w, b, groups, 1e-5, "relu", gy[at])
        R.check(dict(y=y[at], gx=gx[at]), {k: want[k] for k in ("y", "gx")}, at)
    assert gw.isfinite().all() and gb.isfinite().all()
