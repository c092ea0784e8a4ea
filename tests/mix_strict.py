"""The channel-mixing layers in 64 bits, with bounds that hold pre-activations to float32.

As in mix_reference.py, an error e of a value enters the next product with its weight, sums of n terms add SUM(n), and what
a kernel rounds to the tensors' type is off by half a step of it.  Rounded are: outputs, h, and the gradients of the
pre-activations (gz; gg, gu).  Not rounded are z, g and u: they are float32 sums (double for float64) in the forward call
and in the backward call, and so are gh and every factor of a product of three.
"""
import torch

import mix_reference as R

CURVE = 0.85  # no activation here bends more
# (batch, height, width, channels in, hidden, channels out, layout, activation, residual) and what the kernels choose for
# each product on 148 SMs; hidden 0: the pointwise layer.  Products: output, gate, gradients of the pre-activations, input
# gradient: (channels of a tile, channel tiles, tiles that a pair of blocks keeps the weights of, 0: weights travel);
# gradient of w or w_in, of w_out: (rows, columns of a tile).
PATHS = [
    # tiles of 256 channels, weights stay
    ((1, 1, 40_001, 128, 0, 256, "nhwc", "relu", True), dict(output=(256, 1, 1), act=(256, 1, 1), input=(128, 1, 1), weight=(256, 128))),
    ((2, 97, 211, 128, 0, 250, "nchw", "gelu", True), dict(output=(256, 1, 1), act=(256, 1, 1), input=(128, 1, 1), weight=(256, 128))),
    # several channel tiles per pair of blocks, the last one ragged
    ((1, 1, 20_003, 64, 0, 700, "nhwc", "silu", True), dict(output=(256, 3, 3), act=(256, 3, 3), weight=(512, 128))),
    ((3, 100, 203, 72, 0, 328, "nchw", "gelu_tanh", False), dict(output=(128, 3, 3), act=(128, 3, 3), weight=(512, 128))),
    # several groups of pairs, each with its channel tile; three pipeline stages
    ((1, 1, 40_001, 384, 0, 512, "nhwc", "sigmoid", True), dict(output=(256, 2, 1), act=(256, 2, 1), input=(128, 3, 1), weight=(512, 256))),
    # weights travel, many tiles per pair of blocks
    ((1, 1, 40_001, 1024, 0, 1024, "nhwc", "gelu", True), dict(output=(256, 4, 0), act=(256, 4, 0), input=(256, 4, 0), weight=(512, 256))),
    ((5, 63, 127, 1001, 0, 520, "nchw", None, True), dict(output=(256, 3, 0), input=(256, 4, 0), weight=(512, 256))),
    # few channels, many pixels
    ((1, 1, 60_001, 40, 0, 56, "nhwc", "silu", True), dict(output=(64, 1, 1), act=(64, 1, 1), input=(64, 1, 1), weight=(256, 128))),
    # more channel tiles than pairs of blocks
    ((1, 5, 6, 1500, 0, 9700, "nhwc", "silu", False), dict(output=(128, 76, 0), act=(128, 76, 0), weight=(512, 256))),
    # gates: eight groups of pairs; three; one; weights that travel with several tiles per pair
    ((1, 1, 30_001, 256, 1024, 256, "nhwc", "silu", True),
     dict(gate=(128, 8, 1), act=(64, 16, 0), output=(256, 1, 0), input=(256, 1, 0), weight=(512, 256), weight_out=(256, 256))),
    ((4, 125, 199, 96, 384, 96, "nchw", "gelu", True),
     dict(gate=(128, 3, 1), act=(64, 6, 0), output=(128, 1, 1), input=(128, 1, 1), weight=(512, 128), weight_out=(256, 256))),
    ((1, 1, 60_001, 24, 40, 48, "nhwc", "relu", False),
     dict(gate=(64, 1, 1), act=(64, 1, 0), output=(64, 1, 1), input=(64, 1, 1), weight=(256, 128), weight_out=(256, 128))),
    ((1, 1, 30_001, 600, 200, 296, "nhwc", "gelu_tanh", False), dict(gate=(128, 2, 0), act=(64, 4, 0), input=(256, 3, 0))),
]
PRODUCTS = ("output", "gate", "act", "input", "weight", "weight_out")


def plan(lib, desc, product, sms):
    """what mc_mix_plan says for a product, in the form of PATHS, and the tiles (stages of work) of a pair of blocks"""
    import ctypes
    v = (ctypes.c_int32 * 6)()
    rc = lib.mc_mix_plan(desc, PRODUCTS.index(product), sms, v)
    assert rc == 0, (product, rc)
    if product.startswith("weight"):
        return (v[0], v[1]), v[5]
    return (v[0], v[1], v[3]), v[1] * v[2] / v[4]


def path_desc(case):
    from mappedconvolutions_b200 import _lib
    b, h, w, cin, hidden, cout, layout, act, _ = case
    return _lib.McMixDesc(b, h * w, cin, cout, hidden, R.ACTS[act], _lib.MC_BF16, _lib.MC_NHWC if layout == "nhwc" else _lib.MC_NCHW)


def slope(name, z):
    """the sigmoid's as s(z) s(-z): 1 - s(z) cancels in 64 bits too (2^-53 of one where the slope is e^-|z|)"""
    return z.sigmoid() * (-z).sigmoid() if name == "sigmoid" else R.slope(name, z)


def value_error(t, name, z, ez, a, s):
    """z is off by ez; the functions are held to t.fn of the value, or (1 + erf, 1 + tanh in float32 / float64) of one"""
    if name is None:
        return ez
    if name == "relu":
        return ez
    e = (s.abs() + CURVE * ez) * ez + t.fn * (a.abs() + 2.0 ** -20)
    if name.startswith("gelu") and t.fn < 2.0 ** -16:
        e = e + 4 * t.step * z.abs()
    return e


def slope_error(t, name, z, ez, s):
    """absolute, but relative for the sigmoid (whose slope's logarithm has slopes of at most one)"""
    if name is None:
        return torch.zeros_like(z)
    if name == "relu":
        return (z.abs() <= ez).double()
    if name == "sigmoid":
        return s * (torch.expm1(ez) + t.fn)
    return CURVE * ez + t.fn


def _product(t, factors):
    """(value, bound) of a product of factors that are off by their bounds, rounded to the tensors' type"""
    v, hi, lo = 1, 1, 1
    for f, e in factors:
        v, hi, lo = v * f, hi * (f.abs() + e), lo * f.abs()
    return v, hi - lo + (t.u + 4 * t.step) * hi


def pre_activations(x, w, b):
    t = R.Bounds(x.dtype)
    X, W, bd = R.rows(x), w.detach().double()[:, :, 0], b.detach().double()
    return X, W, X @ W.T + bd, t.sum(X.shape[1]) * (X.abs() @ W.abs().T + bd.abs())


def _shaped(out, x):
    B, _, H, W = x.shape
    return {k: (R.images(v, B, H, W), R.images(e, B, H, W)) if k in ("y", "gx") else (v, e) for k, (v, e) in out.items()}


def pointwise(x, w, b, r, name, gy=None, spoil=None):
    """{output name: (value, bound)}; spoil: what a worse implementation does to z before its backward pass"""
    t = R.Bounds(x.dtype)
    X, Wd, z, ez = pre_activations(x, w, b)
    a, s = R.act(name, z), slope(name, z)
    y, ey = a, value_error(t, name, z, ez, a, s)
    if r is not None:
        rr = R.rows(r)
        y, ey = y + rr, ey + 2 * t.step * (a.abs() + rr.abs())
    out = {"y": (y, ey + t.u * (y.abs() + ey))}
    if gy is not None:
        G = R.rows(gy)
        if spoil is not None:
            s = slope(name, spoil(z))
        gz, egz = (G, torch.zeros_like(G)) if name is None else _product(t, [(G, 0), (s, slope_error(t, name, z, ez, s))])
        out.update(R._grads(t, gz, egz, X, Wd, ("gx", "gw", "gb")))
    return _shaped(out, x)


def gated(x, wi, bi, wo, bo, r, name, gy=None, spoil=None):
    t = R.Bounds(x.dtype)
    X, Wi, z, ez = pre_activations(x, wi, bi)
    Wo, bod = wo.detach().double()[:, :, 0], bo.detach().double()
    n = Wo.shape[1]
    g, u, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    a, s = R.act(name, g), slope(name, g)
    ea = value_error(t, name, g, eg, a, s)
    h, eh = _product(t, [(a, ea), (u, eu)])
    y = h @ Wo.T + bod
    ey = eh @ Wo.abs().T + t.sum(n) * ((h.abs() + eh) @ Wo.abs().T + bod.abs())
    if r is not None:
        rr = R.rows(r)
        ey = ey + 2 * t.step * (y.abs() + rr.abs())
        y = y + rr
    out = {"y": (y, ey + t.u * (y.abs() + ey))}
    if gy is not None:
        G = R.rows(gy)
        if spoil is not None:
            g, u = spoil(g), spoil(u)
            a, s = R.act(name, g), slope(name, g)
        gh = G @ Wo
        egh = t.sum(G.shape[1]) * (G.abs() @ Wo.abs())
        gg, egg = _product(t, [(gh, egh), (u, eu), (s, slope_error(t, name, g, eg, s))])
        gu, egu = _product(t, [(gh, egh), (a, ea)])
        out.update(R._grads(t, torch.cat([gg, gu], 1), torch.cat([egg, egu], 1), X, Wi, ("gx", "gw_in", "gb_in")))
        o = R._grads(t, G, torch.zeros_like(G), h, Wo, ("gh", "gw_out", "gb_out"), eh)
        out.update({k: o[k] for k in ("gw_out", "gb_out")})
    return _shaped(out, x)
