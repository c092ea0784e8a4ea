"""The channel-mixing layers in 64 bits, with a bound on what float32 sums and the roundings of the kernels may change.

Every bound is carried through the formulas: a value v that the kernels hold with error at most e enters the next product
with weight |w|, so its result is off by at most sum |w| e, plus what summing n products in float32 adds, plus its own
rounding.  U is half a step of the tensors' type relative to the value.  Rounding errors of a float32 sum of n terms
behave like a random walk of n steps of 2^-24 of the running sum; SUM(n) allows eight times that (2^-53 for float64).
"""
import math

import torch

ACTS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "sigmoid": 5}
SLOPE, CURVE = 1.2, 0.85  # no activation here is steeper, or bends more


def act(name, z):
    f = torch.nn.functional
    return {None: lambda: z, "relu": lambda: z.clamp_min(0), "gelu": lambda: f.gelu(z),
            "gelu_tanh": lambda: f.gelu(z, approximate="tanh"), "silu": lambda: f.silu(z),
            "sigmoid": lambda: z.sigmoid()}[name]()


def slope(name, z):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act(name, z).sum(), z)[0]


class Bounds:
    def __init__(self, dtype):
        self.u = torch.finfo(dtype).eps / 2
        self.step = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
        # elementary functions: a few steps of float32; the bf16 kernels may use short forms of 16 bits
        self.fn = {torch.float64: 2.0 ** -48, torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -15}[dtype]
        # float32 kernels keep intermediate values, bf16 kernels round them
        self.mid = self.u

    def sum(self, n):
        return (8 * math.sqrt(n) + 8) * self.step


def rows(t):
    return t.detach().double().permute(0, 2, 3, 1).reshape(-1, t.shape[1])


def images(m, b, h, w):
    return m.view(b, h, w, -1).permute(0, 3, 1, 2)


def pointwise(x, w, b, r, name, gy=None):
    """{output name: (value, bound)} with tensors shaped as the layer's"""
    B, _, H, W = x.shape
    t = Bounds(x.dtype)
    X, Wd, bd = rows(x), w.detach().double()[:, :, 0], b.detach().double()
    z = X @ Wd.T + bd
    ez = t.sum(X.shape[1]) * (X.abs() @ Wd.abs().T + bd.abs())
    a = act(name, z)
    y, ey = a, SLOPE * ez + t.fn * (a.abs() + 2.0 ** -20)
    if r is not None:
        R = rows(r)
        y, ey = y + R, ey + t.step * (a.abs() + R.abs())
    out = {"y": (y, ey + t.u * y.abs())}
    if gy is not None:
        G = rows(gy)
        s = slope(name, z)
        if name is None:
            gz, egz = G, torch.zeros_like(G)
        else:
            gz = G * s
            kink = (z.abs() <= ez).double() if name == "relu" else 0
            egz = G.abs() * (CURVE * (ez + t.mid * z.abs()) + t.fn + kink) + t.mid * gz.abs()
            if name == "relu":
                egz = G.abs() * kink + t.mid * gz.abs()
        out.update(_grads(t, gz, egz, X, Wd, ("gx", "gw", "gb")))
    return {k: (images(v, B, H, W), images(e, B, H, W)) if k in ("y", "gx") else (v, e) for k, (v, e) in out.items()}


def _grads(t, gz, egz, X, Wd, names, eX=None):
    P = X.shape[0]
    eX = torch.zeros_like(X) if eX is None else eX
    gx = gz @ Wd
    gw, gb = gz.T @ X, gz.sum(0)
    res = {
        names[0]: (gx, egz @ Wd.abs() + t.sum(gz.shape[1]) * (gz.abs() @ Wd.abs()) + t.u * gx.abs()),
        names[1]: (gw[:, :, None], (egz.T @ X.abs() + gz.abs().T @ eX + t.sum(P) * (gz.abs().T @ X.abs())
                                    + t.u * gw.abs())[:, :, None]),
        names[2]: (gb, egz.sum(0) + t.sum(P) * gz.abs().sum(0) + t.u * gb.abs()),
    }
    return res


def gated(x, wi, bi, wo, bo, r, name, gy=None):
    B, _, H, W = x.shape
    t = Bounds(x.dtype)
    X, Wi, bid = rows(x), wi.detach().double()[:, :, 0], bi.detach().double()
    Wo, bod = wo.detach().double()[:, :, 0], bo.detach().double()
    n = Wo.shape[1]
    z = X @ Wi.T + bid
    ez = t.sum(X.shape[1]) * (X.abs() @ Wi.abs().T + bid.abs())
    g, u, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    a = act(name, g)
    ea = SLOPE * eg + t.fn * (a.abs() + 2.0 ** -20)
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + t.mid * h.abs()
    y = h @ Wo.T + bod
    ey = eh @ Wo.abs().T + t.sum(n) * (h.abs() @ Wo.abs().T + bod.abs())
    if r is not None:
        R = rows(r)
        ey = ey + t.step * (y.abs() + R.abs())
        y = y + R
    out = {"y": (y, ey + t.u * y.abs())}
    if gy is not None:
        G = rows(gy)
        eg2, eu2 = eg + t.mid * g.abs(), eu + t.mid * u.abs()
        gh = G @ Wo
        egh = t.sum(G.shape[1]) * (G.abs() @ Wo.abs())
        s = slope(name, g)
        es = CURVE * eg2 + t.fn
        if name == "relu":
            es = (g.abs() <= eg).double()
        elif name is None:
            es = torch.zeros_like(g)
        ea2 = SLOPE * eg2 + t.fn * (a.abs() + 2.0 ** -20)
        gg, gu = gh * u * s, gh * a
        egg = egh * u.abs() * SLOPE + gh.abs() * (eu2 * SLOPE + u.abs() * es) + t.mid * gg.abs()
        egu = egh * a.abs() + gh.abs() * ea2 + t.mid * gu.abs()
        gz, egz = torch.cat([gg, gu], 1), torch.cat([egg, egu], 1)
        out.update(_grads(t, gz, egz, X, Wi, ("gx", "gw_in", "gb_in")))
        o = _grads(t, G, torch.zeros_like(G), h, Wo, ("gh", "gw_out", "gb_out"), eh)
        out.update({k: o[k] for k in ("gw_out", "gb_out")})
    return {k: (images(v, B, H, W), images(e, B, H, W)) if k in ("y", "gx") else (v, e) for k, (v, e) in out.items()}


def check(got, want, what=""):
    for k, v in got.items():
        if v is None:
            continue
        ref, bound = want[k]
        assert v.shape == ref.shape, (what, k, v.shape, ref.shape)
        d = (v.detach().double() - ref).abs()
        bad = ~(d <= bound + 1e-300)
        assert not bad.any(), "%s %s: %d of %d values off, worst %.2f of its bound, error %.3e" % (
            what, k, int(bad.sum()), bad.numel(), (d / (bound + 1e-300)).max().item(), d.max().item())
