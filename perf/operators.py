"""The channel-mixing and training-step operators whose speed matters, as cases that can be timed and compared.

  pointwise  `nn.PointwiseConvolution`: act(W x + b) + residual at every pixel or mesh vertex; inference, or training with
             the gradients of input, weight, bias and residual
  gated      `nn.GatedFeedForward`: W_out (act(W_g x + b_g) * (W_u x + b_u)) + b_out + residual; inference or training
  clip       `dist.clip_gradients`: the norm of all gradients together, and the gradients scaled to at most `max_norm`

`own` chooses between the layer calls of this library and the plain arithmetic: float32 products, sums and element-wise
functions of torch, rounded once at the end.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


def vertices(level):
    return 10 * 4 ** level + 2


# ---- the cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # projection of one coarse sphere, a viewer that waits for the answer: latency counts
        dict(name="pointwise_infer_1", kind="pointwise", height=1, width=vertices(4), batch=1, cin=64, cout=64, act="relu",
             residual=False, dtype="bf16", layout="nhwc", train=False),
        # closing projection of a residual block of the icosphere encoder: level 6, its 128 -> 256 channels
        dict(name="pointwise_train_16", kind="pointwise", height=1, width=vertices(6), batch=16, cin=128, cout=256,
             act="relu", residual=True, dtype="bf16", layout="nhwc", train=True),
        # wide projection at the encoder's coarsest level and full batch
        dict(name="pointwise_wide_infer_64", kind="pointwise", height=1, width=vertices(5), batch=64, cin=1024, cout=1024,
             act="gelu", residual=True, dtype="bf16", layout="nhwc", train=False),
        # panoramas in torch's default type and layout, odd channel counts
        dict(name="pointwise_pano_f32_train", kind="pointwise", height=128, width=256, batch=4, cin=50, cout=99, act="silu",
             residual=False, dtype="f32", layout="nchw", train=True),
        # lens images in bf16 and torch's default layout, odd size, per-pixel class scores of a segmentation head
        dict(name="pointwise_head_train", kind="pointwise", height=125, width=251, batch=8, cin=64, cout=13, act=None,
             residual=False, dtype="bf16", layout="nchw", train=True),
        # feed-forward block on one coarse sphere
        dict(name="gated_infer_1", kind="gated", height=1, width=vertices(4), batch=1, cin=256, hidden=680, cout=256,
             act="silu", residual=True, dtype="bf16", layout="nhwc", train=False),
        # feed-forward block behind the encoder's last layer (256 channels, level 5, batch 64), training
        dict(name="gated_train_64", kind="gated", height=1, width=vertices(5), batch=64, cin=256, hidden=1024, cout=256,
             act="silu", residual=True, dtype="bf16", layout="nhwc", train=True),
        # the same in torch's default type and layout on panoramas, ragged hidden size
        dict(name="gated_f32_train", kind="gated", height=64, width=128, batch=4, cin=64, hidden=171, cout=64, act="gelu",
             residual=True, dtype="f32", layout="nchw", train=True),
        # feature images in bf16 and torch's default layout, odd image size
        dict(name="gated_pano_infer", kind="gated", height=125, width=250, batch=4, cin=96, hidden=384, cout=96, act="gelu",
             residual=True, dtype="bf16", layout="nchw", train=False),
        # gradients of the icosphere encoder: eight tensors
        dict(name="clip_encoder", kind="clip", model="encoder", blocks=1, channels=0, hidden=0, dtype="bf16", out="bf16",
             norm_type=2.0, clipped=True),
        # bf16 gradients of twelve blocks into the float32 ones that the optimiser of float32 weights takes
        dict(name="clip_blocks_to_f32", kind="clip", model="blocks", blocks=12, channels=256, hidden=1024, dtype="bf16",
             out="f32", norm_type=2.0, clipped=True),
        # a large float32 model
        dict(name="clip_blocks_f32", kind="clip", model="blocks", blocks=15, channels=1024, hidden=2730, dtype="f32",
             out="f32", norm_type=2.0, clipped=True),
    ]


def _log(rng, lo, hi):
    """A whole number, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _fit(rng, lo, hi, most):
    """The same with an upper end that keeps the case within the largest listed one."""
    return _log(rng, lo, max(lo, min(hi, int(most))))


def _grid(rng):
    """Mesh vertices of a level, or an image of any size."""
    if rng.random() < 0.5:
        return 1, vertices(rng.randint(2, 7))
    return _log(rng, 16, 400), _log(rng, 16, 800)


def draw(rng):
    kind = rng.choice(("pointwise", "pointwise", "gated", "gated", "clip"))
    if kind == "clip":
        model = rng.choice(("encoder", "blocks", "blocks"))
        dtype = rng.choice(("bf16", "f32"))
        channels, hidden = _log(rng, 16, 1024), _log(rng, 32, 4096)
        blocks = _fit(rng, 1, 15, 14 * 1024 * 2730 / (channels * hidden))
        return dict(kind=kind, model=model, blocks=blocks, channels=channels, hidden=hidden, dtype=dtype,
                    out=rng.choice((dtype, "f32")), norm_type=rng.choice((2.0, 2.0, math.inf)), clipped=rng.random() < 0.7)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    height, width = _grid(rng)
    wide = rng.random() < 0.5  # whole blocks of channels, or any count
    top = 512 if dtype == "bf16" else 128

    def count(lo, hi):
        return 32 * _log(rng, 1, hi // 32) if wide else _log(rng, lo, hi)
    cin, cout = count(3, top), count(3, top)
    train, residual = rng.random() < 0.6, rng.random() < 0.5
    act = rng.choice(("relu", "gelu", "gelu_tanh", "silu", "sigmoid"))
    common = dict(kind=kind, height=height, width=width, dtype=dtype, residual=residual, train=train,
                  layout=rng.choice(("nchw", "nhwc")))
    if kind == "pointwise":
        if dtype == "bf16":
            most = 16 * vertices(6) * 128 * 256 / (height * width * cin * cout)
        else:
            most = 4 * 128 * 256 * 64 * 128 / (height * width * cin * cout)
        return dict(common, batch=_fit(rng, 1, 64, most), cin=cin, cout=cout, act=rng.choice((None, act)))
    hidden = count(8, 1024 if dtype == "bf16" else 256)
    most = (64 * vertices(5) * 256 * 1024 * 3 / 4 if dtype == "bf16" else 4 * 64 * 128 * 64 * 256 * 3) \
        / (height * width * hidden * (2 * cin + cout))
    if most < 1:
        height, width = 1, vertices(4)
        common.update(height=height, width=width)
    return dict(common, batch=_fit(rng, 1, 64, most), cin=cin, hidden=hidden, cout=cout, act=act)


# ---- inputs ------------------------------------------------------------------------------------------

def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _uniform(g, s, *shape):
    return (torch.rand(*shape, generator=g, device=DEV) * 2 - 1) * s


def _image(g, case, channels, scale=1.0):
    """(batch, channels, height, width) activations in the case's type and layout."""
    b, h, w = case["batch"], case["height"], case["width"]
    if case["layout"] == "nhwc":
        return _randn(g, b, h, w, channels, scale=scale).to(DTYPES[case["dtype"]]).permute(0, 3, 1, 2)
    return _randn(g, b, channels, h, w, scale=scale).to(DTYPES[case["dtype"]])


def _gradient_shapes(case):
    if case["model"] == "encoder":
        ch = (3, 64, 128, 256, 256)
        return [s for i in range(4) for s in ((ch[i + 1], ch[i], 7), (ch[i + 1],))]
    c, h = case["channels"], case["hidden"]
    return [(2 * h, c, 1), (2 * h,), (c, h, 1), (c,)] * case["blocks"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case)
    if case["kind"] == "clip":
        # the gradients of one step: layers differ in size by orders of magnitude
        dt = DTYPES[case["dtype"]]
        shapes = _gradient_shapes(case)
        state["grads"] = [_randn(g, *s, scale=10.0 ** (-3 + 2 * (i % 5) / 4)).to(dt) for i, s in enumerate(shapes)]
        state["out"] = [torch.empty(s, dtype=DTYPES[case["out"]], device=DEV) for s in shapes]
        numel = sum(t.numel() for t in state["grads"])
        # norms here lie between 1e-3 sqrt(n) and 1e-1 sqrt(n); largest elements above 1e-3
        tight = 1e-4 * math.sqrt(numel) if case["norm_type"] == 2.0 else 1e-3
        state["max_norm"] = tight if case["clipped"] else 1e6
        return state
    dt = DTYPES[case["dtype"]]
    cin, cout = case["cin"], case["cout"]
    state["x"] = _image(g, case, cin)
    state["r"] = _image(g, case, cout) if case["residual"] else None
    state["gy"] = _image(g, case, cout, 0.01) if case["train"] else None
    s = 1.0 / math.sqrt(cin)
    if case["kind"] == "pointwise":
        params = dict(weight=_uniform(g, s, cout, cin, 1), bias=_uniform(g, s, cout))
    else:
        h = case["hidden"]
        s2 = 1.0 / math.sqrt(h)
        params = dict(weight_in=_uniform(g, s, 2 * h, cin, 1), bias_in=_uniform(g, s, 2 * h),
                      weight_out=_uniform(g, s2, cout, h, 1), bias_out=_uniform(g, s2, cout))
    state["params"] = {k: v.to(dt) for k, v in params.items()}
    if own:
        from mapped_convolution import nn as mnn
        if case["kind"] == "pointwise":
            layer = mnn.PointwiseConvolution(cin, cout, activation=case["act"])
        else:
            layer = mnn.GatedFeedForward(cin, case["hidden"], cout, activation=case["act"])
        layer = layer.to(DEV).to(dt).requires_grad_(case["train"])
        with torch.no_grad():
            for k, v in state["params"].items():
                getattr(layer, k).copy_(v)
        state["layer"] = layer
        if case["train"]:
            state["x"].requires_grad_(True)
            if state["r"] is not None:
                state["r"].requires_grad_(True)
    return state


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["kind"] == "clip":
        return _own_clip(state) if own else _plain_clip(state)
    if own:
        return _own_layer(state)
    return _plain_pointwise(state) if case["kind"] == "pointwise" else _plain_gated(state)


def _own_clip(state):
    from mappedconvolutions_b200 import dist as mdist
    case = state["case"]
    norm = mdist.clip_gradients(state["grads"], state["max_norm"], norm_type=case["norm_type"], out=state["out"])
    return [norm] + state["out"]


def _own_layer(state):
    case, layer = state["case"], state["layer"]
    if not case["train"]:
        with torch.no_grad():
            return layer(state["x"], state["r"])
    y = layer(state["x"], state["r"])
    leaves = [state["x"]] + [getattr(layer, k) for k in state["params"]] + ([state["r"]] if case["residual"] else [])
    return [y.detach()] + list(torch.autograd.grad(y, leaves, state["gy"]))


def _plain_clip(state):
    case, grads, out = state["case"], state["grads"], state["out"]
    if case["norm_type"] == 2.0:
        norm = torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()
    else:
        norm = torch.stack([g.float().abs().max() for g in grads]).max()
    coefficient = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
    for g, o in zip(grads, out):
        o.copy_(g.float() * coefficient)
    return [norm] + out


def _phi(z):  # standard normal distribution function and density
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _activation(name, z):
    if name is None:
        return z
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return z * _phi(z)[0]
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    s = 1 / (1 + torch.exp(-z))
    return s if name == "sigmoid" else z * s


def _derivative(name, z):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        p, d = _phi(z)
        return p + z * d
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 - s) if name == "sigmoid" else s * (1 + z * (1 - s))


def _rows(t):
    """(B, C, H, W) -> (pixels, C) in float32."""
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1]).float()


def _images(rows, case, channels):
    t = rows.to(DTYPES[case["dtype"]]).view(case["batch"], case["height"], case["width"], channels).permute(0, 3, 1, 2)
    return t if case["layout"] == "nhwc" else t.contiguous()


def _plain_pointwise(state):
    case, dt, x = state["case"], DTYPES[state["case"]["dtype"]], _rows(state["x"])
    w, b = state["params"]["weight"][:, :, 0].float(), state["params"]["bias"].float()
    z = x @ w.T + b
    y = _activation(case["act"], z)
    if case["residual"]:
        y = y + _rows(state["r"])
    y = _images(y, case, case["cout"])
    if not case["train"]:
        return y
    gz = _rows(state["gy"]) * _derivative(case["act"], z)
    grads = [_images(gz @ w, case, case["cin"]), (gz.T @ x).to(dt)[:, :, None], gz.sum(0).to(dt)]
    return [y] + grads + ([state["gy"]] if case["residual"] else [])


def _plain_gated(state):
    case, dt, x = state["case"], DTYPES[state["case"]["dtype"]], _rows(state["x"])
    p, h = {k: v.float() for k, v in state["params"].items()}, state["case"]["hidden"]
    w_in, w_out = p["weight_in"][:, :, 0], p["weight_out"][:, :, 0]
    z = x @ w_in.T + p["bias_in"]
    gate, up = z[:, :h], z[:, h:]
    a = _activation(case["act"], gate)
    y = (a * up) @ w_out.T + p["bias_out"]
    if case["residual"]:
        y = y + _rows(state["r"])
    y = _images(y, case, case["cout"])
    if not case["train"]:
        return y
    gy = _rows(state["gy"])
    gw_out, gb_out = gy.T @ (a * up), gy.sum(0)
    gh = gy @ w_out
    gz = torch.cat([gh * up * _derivative(case["act"], gate), gh * a], 1)
    grads = [_images(gz @ w_in, case, case["cin"]), (gz.T @ x).to(dt)[:, :, None], gz.sum(0).to(dt),
             gw_out.to(dt)[:, :, None], gb_out.to(dt)]
    return [y] + grads + ([state["gy"]] if case["residual"] else [])


# ---- work --------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _gradient_shapes(case))
        return {"bytes": n * (SIZE[case["dtype"]] + SIZE[case["out"]]) + 4, "flops": 3 * n}
    e, pixels = SIZE[case["dtype"]], case["batch"] * case["height"] * case["width"]
    cin, cout, r = case["cin"], case["cout"], int(case["residual"])
    if case["kind"] == "pointwise":
        params, products = cin * cout + cout, cin * cout
    else:
        h = case["hidden"]
        params, products = 2 * h * (cin + 1) + cout * (h + 1), h * (2 * cin + cout)
    moved = pixels * (cin + cout * (1 + r)) + params
    if case["train"]:  # grad_output in, the gradients of input and parameters out (the residual's is grad_output)
        moved += pixels * (cin + cout) + params
    return {"bytes": e * moved, "flops": 2 * pixels * products * (3 if case["train"] else 1)}


# ---- the definition in 64 bits -----------------------------------------------------------------------

_EXACT_ACT = {
    None: lambda z: z,
    "relu": torch.relu,
    "gelu": lambda z: z * torch.special.ndtr(z),
    "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
    "silu": lambda z: z * torch.sigmoid(z),
    "sigmoid": torch.sigmoid,
}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "clip":
        p = case["norm_type"]
        each = torch.stack([torch.linalg.vector_norm(g, p, dtype=torch.float64) for g in state["grads"]])
        norm = torch.linalg.vector_norm(each, p)
        factor = min(1.0, state["max_norm"] / (norm.item() + 1e-6))
        return [norm] + [g.double() * factor for g in state["grads"]]
    params = [v.double().requires_grad_(case["train"]) for v in state["params"].values()]
    act, ys, gxs = _EXACT_ACT[case["act"]], [], []
    for i in range(case["batch"]):  # an image at a time: the parameters' gradients add up
        x = state["x"][i].double().requires_grad_(case["train"])
        with torch.set_grad_enabled(case["train"]):
            if case["kind"] == "pointwise":
                y = act(torch.einsum("oi,ihw->ohw", params[0].squeeze(2), x) + params[1][:, None, None])
            else:
                z = torch.einsum("oi,ihw->ohw", params[0].squeeze(2), x) + params[1][:, None, None]
                gate, up = z.chunk(2)
                y = torch.einsum("oi,ihw->ohw", params[2].squeeze(2), act(gate) * up) + params[3][:, None, None]
        if case["train"]:
            y.backward(state["gy"][i].double())
            gxs.append(x.grad)
        ys.append(y.detach() + state["r"][i].double() if case["residual"] else y.detach())
    y = torch.stack(ys)
    if not case["train"]:
        return y
    return [y, torch.stack(gxs)] + [q.grad for q in params] + ([state["gy"].double()] if case["residual"] else [])
