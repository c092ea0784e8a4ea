"""Group norm, the pixel classification loss and AdamW in 64 bits, with bounds on what the kernels' arithmetic may change.

U is half a step of the tensors' type relative to the value, `step` half a step of the arithmetic (2^-24; 2^-53 for float64).  A sum of n
terms may be off by sum_of(n) of the sum of their magnitudes: eight times a random walk of n roundings.  Errors are carried through
the formulas to first order, each product and sum adding its own rounding.
"""
import math

import torch

from mix_reference import ACTS, CURVE, SLOPE, act, slope  # noqa: F401


class Bounds:
    def __init__(self, dtype):
        self.u = torch.finfo(dtype).eps / 2
        self.step = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
        # elementary functions: a few steps of float32; of bf16 kernels short forms of 16 bits
        self.fn = {torch.float64: 2.0 ** -48, torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -15}[dtype]

    def sum(self, n):
        return (8 * math.sqrt(n) + 8) * self.step


def group_norm(x, w, b, groups, eps, name, gy=None):
    """{output name: (value, bound)}"""
    t, (B, C, H, W) = Bounds(x.dtype), x.shape
    split = (B, groups, C // groups, H * W)
    dims, n = (2, 3), C // groups * H * W
    X = x.double().reshape(split)
    one = torch.ones(C, dtype=torch.float64, device=x.device)
    wd, bd = (v.double().view(1, groups, -1, 1) for v in (one if w is None else w, 0 * one if b is None else b))
    mean = X.mean(dims, keepdim=True)
    var = (X - mean).square().mean(dims, keepdim=True)
    rstd = (var + eps).rsqrt()
    xhat = (X - mean) * rstd
    # runs of up to 256 values are summed in float32 before they are merged; the mean keeps a rounding of its own
    run = t.sum(256)
    e_mean = run * (X - mean).abs().mean(dims, keepdim=True) + 2 * t.step * mean.abs()
    e_rstd = run + 4 * t.step  # (relative; half of the variance's)
    e_xhat = xhat.abs() * e_rstd + rstd * e_mean + 2 * t.step * (xhat.abs() + rstd * 0)
    z = xhat * wd + bd
    ez = wd.abs() * e_xhat + 2 * t.step * ((xhat * wd).abs() + bd.abs())
    y = act(name, z)
    ey = SLOPE * ez + t.fn * (y.abs() + z.abs() * 2.0 ** -3) * (name is not None) + t.u * y.abs()
    full = lambda v: v.expand(split).reshape(B, C, H, W)  # noqa: E731
    out = dict(y=(full(y), full(ey)))
    if gy is None:
        return out
    G = gy.double().reshape(split)
    d = slope(name, z)
    dz = G * d
    e_dz = G.abs() * (CURVE * ez + (t.fn if name not in (None, "relu") else 0)) + t.step * dz.abs()
    h, e_h = dz * wd, wd.abs() * e_dz + t.step * (dz * wd).abs()
    m = lambda v: v.mean(dims, keepdim=True)  # noqa: E731
    a, e_a = m(h), m(e_h) + t.sum(n) * m(h.abs())
    c, e_c = m(h * xhat), m(e_h * xhat.abs() + h.abs() * e_xhat) + t.sum(n) * m((h * xhat).abs())
    gx = rstd * (h - a - xhat * c)
    e_gx = rstd * (e_h + e_a + xhat.abs() * e_c + e_xhat * c.abs() + 6 * t.step * (h.abs() + a.abs() + (xhat * c).abs())) \
        + e_rstd * rstd * (h.abs() + a.abs() + (xhat * c).abs()) + t.u * gx.abs()
    out["gx"] = full(gx), full(e_gx)
    s = lambda v: v.sum((0, 3)).reshape(C)  # noqa: E731
    N = B * H * W
    gw, gb = s(dz * xhat), s(dz)
    out["gw"] = gw, s(e_dz * xhat.abs() + dz.abs() * e_xhat) + t.sum(N) * s((dz * xhat).abs()) + t.u * gw.abs()
    out["gb"] = gb, s(e_dz) + t.sum(N) * s(dz.abs()) + t.u * gb.abs()
    return out


def cross_entropy(x, w, b, target, ignore, mean, grad=None):
    """{output name: (value, bound)}; grad: the gradient of the loss"""
    t, (B, C, H, W) = Bounds(x.dtype), x.shape
    rows = x.double().permute(0, 2, 3, 1).reshape(-1, C)
    wd, bd, label = w.double()[:, :, 0], b.double(), target.reshape(-1)
    valid = label != ignore
    rows = torch.where(valid[:, None], rows, torch.zeros_like(rows))  # what a pixel without a label holds does not count
    at = torch.where(valid, label, torch.zeros_like(label))[:, None]
    z = rows @ wd.T + bd
    ez = t.sum(C) * (rows.abs() @ wd.abs().T + bd.abs()) + t.step * z.abs()
    lse = z.logsumexp(1, keepdim=True)
    p = (z - lse).exp()
    fn = {torch.float64: 2.0 ** -46}.get(x.dtype, 2.0 ** -19)  # exp and log, a few steps each
    e_lse = (p * ez).sum(1, keepdim=True) + fn + 4 * t.step * lse.abs() + t.sum(z.shape[1])
    count = int(valid.sum()) if mean else 1
    each, e_each = (lse - z.gather(1, at))[:, 0] * valid, (e_lse + ez.gather(1, at))[:, 0] * valid
    loss = each.sum() / count
    unit = 2.0 ** -52 if x.dtype == torch.float64 else 2.0 ** -24
    out = dict(loss=(loss, e_each.sum() / count + (each.abs().sum() / count) * 4 * t.step + unit * loss.abs()))
    if grad is None:
        return out
    scale = float(grad) / count
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    gz = (p - hot) * valid[:, None]
    mid = t.u if x.dtype == torch.bfloat16 else 2 * t.step  # the kernels may round what the next products read
    e_gz = (p * (ez + e_lse + fn + t.step * (z.abs() + lse.abs())) + (mid + 2 * t.step) * gz.abs()) * valid[:, None]
    gx = scale * gz @ wd
    e_gx = abs(scale) * (e_gz @ wd.abs() + t.sum(z.shape[1]) * (gz.abs() @ wd.abs())) + t.u * gx.abs()
    image = lambda v: v.view(B, H, W, C).permute(0, 3, 1, 2)  # noqa: E731
    n = rows.shape[0]
    gw, gb = scale * gz.T @ rows, scale * gz.sum(0)
    e_gw = abs(scale) * (e_gz.T @ rows.abs() + t.sum(n) * (gz.abs().T @ rows.abs())) + t.u * gw.abs()
    e_gb = abs(scale) * (e_gz.sum(0) + t.sum(n) * gz.abs().sum(0)) + t.u * gb.abs()
    out.update(gx=(image(gx), image(e_gx)), gw=(gw[:, :, None], e_gw[:, :, None]), gb=(gb, e_gb))
    return out


def check(got, want, what):
    for name, v in got.items():
        ref, bound = want[name]
        assert v.shape == ref.shape, (what, name, v.shape, ref.shape)
        off = (v.double() - ref).abs()
        bad = ~(off <= bound + 1e-40)  # (what float32 and bf16 flush to zero)
        assert not bad.any(), "%s %s: %d of %d values off, at most %.3g times the bound" % (
            what, name, int(bad.sum()), bad.numel(), (off / (bound + 1e-40)).max().item())
