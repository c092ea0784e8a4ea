"""Operators of a training step around the layers, as cases that can be timed and compared.

  norm      `nn.GroupNorm`: act((x - mean) / sqrt(var + eps) * weight + bias) with the statistics of a group of channels over an
            image or mesh; inference, or training with the gradients of input, weight and bias
  classify  `nn.PointwiseCrossEntropy`: softmax cross entropy of W x + b at every pixel or vertex against a label each, without
            keeping the class scores; the loss alone, or training with the gradients of input, weight and bias
  adamw     `optim.AdamW`: a step over all parameters at once, moments in 32 bits or in 8 bits with a scale for 256 of them

`own` chooses between the calls of this library and the plain arithmetic: float32 products, sums and element-wise functions of
torch, rounded once at the end.

Moments in 8 bits, in the order in which a tensor lies in memory, 256 elements to a block: with a the largest |m| of the block and
s = a (1 / 16129), m is kept as c = round(sqrt(|m| (1 / s))) with its sign and stands for c |c| s; with a the largest sqrt(v) and
s = a (1 / 65025), v is kept as c = round(sqrt(sqrt(v) (1 / s))), at least 1 where v > 0, and stands for (c^2 s)^2.  Scales below 2^-126
are zero.  All of it in float32, each operation rounded: both sides then keep the same codes.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
BETAS, EPS, DECAY, STEP = (0.9, 0.999), 1e-8, 1e-2, 100
BLOCK = 256


def vertices(level):
    return 10 * 4 ** level + 2


# ---- the cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # features of one coarse sphere, a viewer that waits for the answer: latency counts
        dict(name="norm_infer_1", kind="norm", height=1, width=vertices(4), batch=1, channels=64, groups=8, act="silu",
             dtype="bf16", layout="nhwc", train=False),
        # behind the icosphere encoder's last layer: 256 channels, level 5, batch 64
        dict(name="norm_train_64", kind="norm", height=1, width=vertices(5), batch=64, channels=256, groups=32, act="relu",
             dtype="bf16", layout="nhwc", train=True),
        # panoramas in torch's default type and layout, odd channel count
        dict(name="norm_pano_f32_train", kind="norm", height=128, width=256, batch=4, channels=50, groups=10, act="silu",
             dtype="f32", layout="nchw", train=True),
        # lens images in bf16 and torch's default layout, odd image size
        dict(name="norm_lens_train", kind="norm", height=125, width=251, batch=8, channels=96, groups=8, act="gelu",
             dtype="bf16", layout="nchw", train=True),
        # validation loss of a dense correspondence: which vertex of a level-4 sphere each vertex of one sphere is
        dict(name="classify_match_1", kind="classify", height=1, width=vertices(4), batch=1, cin=64, classes=vertices(4),
             ignore=False, reduction="mean", dtype="bf16", layout="nhwc", train=False),
        # training of the same at level 5, 256 channels, four spheres
        dict(name="classify_match_train_4", kind="classify", height=1, width=vertices(5), batch=4, cin=256,
             classes=vertices(5), ignore=False, reduction="mean", dtype="bf16", layout="nhwc", train=True),
        # segmentation head of lens images: 13 classes, unlabelled pixels, bf16 in torch's default layout, odd image size
        dict(name="classify_head_train", kind="classify", height=125, width=251, batch=8, cin=64, classes=13, ignore=True,
             reduction="mean", dtype="bf16", layout="nchw", train=True),
        # panoramas in torch's default type and layout, more classes
        dict(name="classify_pano_f32_train", kind="classify", height=128, width=256, batch=4, cin=50, classes=99, ignore=True,
             reduction="sum", dtype="f32", layout="nchw", train=True),
        # the icosphere encoder's eight tensors: latency counts
        dict(name="adamw_encoder", kind="adamw", model="encoder", blocks=1, channels=0, hidden=0, dtype="f32", bits=32,
             master=False),
        # bf16 blocks with float32 copies of their parameters
        dict(name="adamw_blocks_master", kind="adamw", model="blocks", blocks=4, channels=1024, hidden=2730, dtype="bf16",
             bits=32, master=True),
        # a large bf16 model whose moments are kept in 8 bits
        dict(name="adamw_blocks_8bit", kind="adamw", model="blocks", blocks=4, channels=1024, hidden=2730, dtype="bf16",
             bits=8, master=False),
        # a large float32 model
        dict(name="adamw_blocks_f32", kind="adamw", model="blocks", blocks=5, channels=1500, hidden=4001, dtype="f32", bits=32,
             master=False),
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
    kind = rng.choice(("norm", "classify", "adamw"))
    if kind == "adamw":
        model = rng.choice(("encoder", "blocks", "blocks", "blocks"))
        dtype = rng.choice(("bf16", "f32"))
        channels, hidden = _log(rng, 16, 1024), _log(rng, 32, 4096)
        return dict(kind=kind, model=model, blocks=rng.randint(1, 4), channels=channels, hidden=hidden, dtype=dtype,
                    bits=rng.choice((8, 32)), master=dtype == "bf16" and rng.random() < 0.5)
    dtype = rng.choice(("bf16", "bf16", "f32"))
    height, width = _grid(rng)
    common = dict(kind=kind, height=height, width=width, dtype=dtype, layout=rng.choice(("nchw", "nhwc")),
                  train=rng.random() < 0.6)
    if kind == "norm":
        groups = _log(rng, 1, 32)
        channels = groups * _log(rng, 1, (512 if dtype == "bf16" else 256) // groups)
        most = 64 * vertices(5) * 256 / (2 if dtype == "f32" else 1) / (height * width * channels)
        if most < 1:
            height, width = 1, vertices(5)
            common.update(height=height, width=width)
        act = rng.choice((None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"))
        return dict(common, batch=_fit(rng, 1, 64, most), channels=channels, groups=groups, act=act)
    cin = 32 * _log(rng, 1, 8) if rng.random() < 0.5 else _log(rng, 3, 256)
    classes = vertices(rng.randint(2, 5)) if rng.random() < 0.4 else _log(rng, 2, 4000)
    if dtype == "f32":
        cin, classes = min(cin, 128), min(classes, 700)
    most = 4 * vertices(5) * vertices(5) / (height * width * classes)
    if most < 1:
        height, width = 1, vertices(4)
        common.update(height=height, width=width)
        most = 4 * vertices(5) * vertices(5) / (width * classes)
    return dict(common, batch=_fit(rng, 1, 16, min(most, 16 * vertices(7) / (height * width))), cin=cin, classes=classes,
                ignore=rng.random() < 0.5, reduction=rng.choice(("mean", "mean", "sum")))


# ---- inputs ------------------------------------------------------------------------------------------

def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _uniform(g, s, *shape):
    return (torch.rand(*shape, generator=g, device=DEV) * 2 - 1) * s


def _image(g, case, channels, scale=1.0, spread=None):
    """(batch, channels, height, width) activations in the case's type and layout; `spread`: an offset for each channel."""
    b, h, w = case["batch"], case["height"], case["width"]
    t = _randn(g, b, h, w, channels, scale=scale)
    if spread is not None:
        t = t + spread
    t = t.permute(0, 3, 1, 2)
    return t.to(DTYPES[case["dtype"]]) if case["layout"] == "nhwc" else t.contiguous().to(DTYPES[case["dtype"]])


def _shapes(case):
    if case["model"] == "encoder":
        ch = (3, 64, 128, 256, 256)
        return [s for i in range(4) for s in ((ch[i + 1], ch[i], 7), (ch[i + 1],))]
    c, h = case["channels"], case["hidden"]
    return [(2 * h, c, 1), (2 * h,), (c, h, 1), (c,)] * case["blocks"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return dict(norm=_prepare_norm, classify=_prepare_classify, adamw=_prepare_adamw)[case["kind"]](case, g)


def _prepare_norm(case, g):
    c, dt = case["channels"], DTYPES[case["dtype"]]
    state = dict(case=case, x=_image(g, case, c, 2.0, _randn(g, c)),
                 gy=_image(g, case, c, 0.01) if case["train"] else None,
                 params=dict(weight=(1 + _randn(g, c, scale=0.2)).to(dt), bias=_randn(g, c, scale=0.2).to(dt)))
    if own:
        from mapped_convolution import nn as mnn
        _layer(state, mnn.GroupNorm(case["groups"], c, activation=case["act"]))
    return state


def _prepare_classify(case, g):
    cin, classes, dt = case["cin"], case["classes"], DTYPES[case["dtype"]]
    s = 4.0 / math.sqrt(cin)  # class scores of a model that has learned something: several units apart
    state = dict(case=case, x=_image(g, case, cin),
                 params=dict(weight=_uniform(g, s, classes, cin, 1).to(dt), bias=_uniform(g, s, classes).to(dt)))
    target = torch.randint(0, classes, (case["batch"], case["height"], case["width"]), generator=g, device=DEV)
    if case["ignore"]:
        target[torch.rand(target.shape, generator=g, device=DEV) < 0.1] = -100
    state["target"] = target
    if own:
        from mapped_convolution import nn as mnn
        _layer(state, mnn.PointwiseCrossEntropy(cin, classes, reduction=case["reduction"]))
    return state


def _layer(state, layer):
    case = state["case"]
    layer = layer.to(DEV).to(DTYPES[case["dtype"]]).requires_grad_(case["train"])
    with torch.no_grad():
        for k, v in state["params"].items():
            getattr(layer, k).copy_(v)
    state["layer"] = layer
    state["x"].requires_grad_(case["train"])


def _prepare_adamw(case, g):
    dt = DTYPES[case["dtype"]]
    state = dict(case=case, step=STEP, lr=1e-3, params=[], grads=[], moments=[], masters=[])
    for i, shape in enumerate(_shapes(case)):
        size = 10.0 ** (-3 + 2 * (i % 5) / 4)  # the gradients of layers differ in size by orders of magnitude
        p = _uniform(g, 1.0 / math.sqrt(max(shape[-2:])), *shape)
        m, v = _randn(g, *shape, scale=0.3 * size), (_randn(g, *shape).square() + 0.01) * size ** 2
        state["params"].append(p.to(dt))
        state["grads"].append(_randn(g, *shape, scale=size).to(dt))
        state["masters"].append(p if case["master"] else None)
        state["moments"].append(_encode_m(m) + _encode_v(v) if case["bits"] == 8 else (m, v))
    if own:
        from mappedconvolutions_b200 import optim
        state["params"] = [torch.nn.Parameter(p) for p in state["params"]]
        for p, gr in zip(state["params"], state["grads"]):
            p.grad = gr
        opt = optim.AdamW(state["params"], lr=state["lr"], betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                          master_weights=case["master"])
        for p, kept, master in zip(state["params"], state["moments"], state["masters"]):
            if case["bits"] == 8:
                names = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
            else:
                names = ("exp_avg", "exp_avg_sq")
            opt.state[p] = dict(zip(names, kept), step=STEP, **({"master": master} if case["master"] else {}))
        state["optimizer"] = opt
    return state


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(norm=_own_norm, classify=_own_classify, adamw=_own_adamw)[kind](state)
    return dict(norm=_plain_norm, classify=_plain_classify, adamw=_plain_adamw)[kind](state)


def _own_norm(state):
    case, layer = state["case"], state["layer"]
    if not case["train"]:
        with torch.no_grad():
            return layer(state["x"])
    y = layer(state["x"])
    return [y.detach()] + list(torch.autograd.grad(y, [state["x"], layer.weight, layer.bias], state["gy"]))


def _own_classify(state):
    case, layer = state["case"], state["layer"]
    if not case["train"]:
        with torch.no_grad():
            return layer(state["x"], state["target"])
    loss = layer(state["x"], state["target"])
    return [loss.detach()] + list(torch.autograd.grad(loss, [state["x"], layer.weight, layer.bias]))


def _own_adamw(state):
    opt = state["optimizer"]
    opt.step()
    out = [p.detach() for p in state["params"]] + [t for pair in opt.moments() for t in pair]
    return out + [opt.state[p]["master"] for p in state["params"]] if state["case"]["master"] else out


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


def _in_layout(t, case):
    """(B, C, H, W) in float32 -> the case's type and layout"""
    fmt = torch.channels_last if case["layout"] == "nhwc" else torch.contiguous_format
    return t.to(DTYPES[case["dtype"]]).contiguous(memory_format=fmt)


def _plain_norm(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    b, c, h, w = state["x"].shape
    split = (b, case["groups"], c // case["groups"], h, w)
    x = state["x"].float().reshape(split)
    weight, bias = (state["params"][k].float().view(1, case["groups"], -1, 1, 1) for k in ("weight", "bias"))
    d = x - x.mean((2, 3, 4), keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean((2, 3, 4), keepdim=True) + 1e-5)
    xhat = d * rstd
    z = xhat * weight + bias
    y = _in_layout(_activation(case["act"], z).view(b, c, h, w), case)
    if not case["train"]:
        return y
    gz = state["gy"].float().reshape(split) * _derivative(case["act"], z)
    gweight, gbias = (gz * xhat).sum((0, 3, 4)).view(c), gz.sum((0, 3, 4)).view(c)
    gh = gz * weight
    gx = rstd * (gh - gh.mean((2, 3, 4), keepdim=True) - xhat * (gh * xhat).mean((2, 3, 4), keepdim=True))
    return [y, _in_layout(gx.view(b, c, h, w), case), gweight.to(dt), gbias.to(dt)]


def _plain_classify(state):
    case, dt, x = state["case"], DTYPES[state["case"]["dtype"]], state["x"]
    rows = x.permute(0, 2, 3, 1).reshape(-1, case["cin"]).float()
    weight, bias = state["params"]["weight"][:, :, 0].float(), state["params"]["bias"].float()
    target = state["target"].reshape(-1)
    valid = target != -100
    label = torch.where(valid, target, torch.zeros_like(target))
    z = rows @ weight.T + bias
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    each = torch.where(valid, (top + torch.log(total) - z.gather(1, label[:, None]))[:, 0], torch.zeros_like(top[:, 0]))
    scale = 1 / valid.sum() if case["reduction"] == "mean" else torch.ones((), device=x.device)
    loss = (each.sum(dtype=torch.float64) * scale).float()
    if not case["train"]:
        return loss
    p = p / total
    p.scatter_add_(1, label[:, None], torch.full_like(top, -1.0))
    p = p * (valid * scale)[:, None]
    gx = (p @ weight).view(case["batch"], case["height"], case["width"], -1).permute(0, 3, 1, 2)
    return [loss, _in_layout(gx, case), (p.T @ rows).to(dt)[:, :, None], p.sum(0).to(dt)]


def _blocks(t):
    """A tensor's elements, 256 to a row, the last row filled up with zeros."""
    t = t.reshape(-1)
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def _scales(largest, codes):
    s = largest * (1 / codes)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    return s, torch.where(s == 0, torch.zeros_like(s), 1 / s)


def _encode_m(m):
    rows = _blocks(m)
    s, inverse = _scales(rows.abs().amax(1, keepdim=True), 16129.0)
    c = torch.sqrt(rows.abs() * inverse).round().clamp(max=127)
    return torch.copysign(c, rows).to(torch.int8).reshape(-1)[:m.numel()].view(m.shape), s[:, 0].contiguous()


def _encode_v(v):
    rows = torch.sqrt(_blocks(v))
    s, inverse = _scales(rows.amax(1, keepdim=True), 65025.0)
    c = torch.sqrt(rows * inverse).round().clamp(max=255)
    c = torch.where((rows > 0) & (s > 0) & (c == 0), torch.ones_like(c), c)
    return c.to(torch.uint8).reshape(-1)[:v.numel()].view(v.shape), s[:, 0].contiguous()


def _decode(codes, s, square):
    c = _blocks(codes.float())
    c = (c * c * s[:, None]).square() if square else c * c.abs() * s[:, None]
    return c.reshape(-1)[:codes.numel()].view(codes.shape)


def _plain_adamw(state):
    case = state["case"]
    state["step"] += 1
    b1, b2 = BETAS
    rate, root = state["lr"] / (1 - b1 ** state["step"]), math.sqrt(1 - b2 ** state["step"])
    moments = []
    for i, (p, gr, kept, master) in enumerate(zip(state["params"], state["grads"], state["moments"], state["masters"])):
        gr = gr.float()
        m, v = (_decode(*kept[:2], False), _decode(*kept[2:], True)) if case["bits"] == 8 else kept
        m = m * b1 + gr * (1 - b1)
        v = v * b2 + gr * gr * (1 - b2)
        value = (p.float() if master is None else master) * (1 - state["lr"] * DECAY)
        value = value - rate * (m / (torch.sqrt(v) / root + EPS))
        p.copy_(value)
        if master is not None:
            master.copy_(value)
        state["moments"][i] = _encode_m(m) + _encode_v(v) if case["bits"] == 8 else (m, v)
        kept = state["moments"][i]
        moments += [_decode(*kept[:2], False), _decode(*kept[2:], True)] if case["bits"] == 8 else [m, v]
    return state["params"] + moments + (state["masters"] if case["master"] else [])


# ---- work --------------------------------------------------------------------------------------------

def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        # parameters (and their float32 copies) both ways, gradients in, moments both ways; 8-bit ones also out as values
        moments = 16 if case["bits"] == 32 else 2 * (2 + 8 / BLOCK) + 8
        each = (2 * 4 + e if case["master"] else 2 * e) + e + moments
        return {"bytes": n * each, "flops": 16 * n}
    pixels = case["batch"] * case["height"] * case["width"]
    if case["kind"] == "norm":
        n = pixels * case["channels"]
        return {"bytes": e * (n * (4 if case["train"] else 2) + case["channels"] * (4 if case["train"] else 2)),
                "flops": n * (30 if case["train"] else 12)}
    cin, classes = case["cin"], case["classes"]
    params = classes * (cin + 1)
    both = 2 if case["train"] else 1
    return {"bytes": e * both * (pixels * cin + params) + 8 * pixels + 4,
            "flops": 2 * pixels * cin * classes * (3 if case["train"] else 1)}


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
    return dict(norm=_exact_norm, classify=_exact_classify, adamw=_exact_adamw)[case["kind"]](state)


def _exact_norm(state):
    case = state["case"]
    params = [v.double().requires_grad_(case["train"]) for v in state["params"].values()]
    ys, gxs = [], []
    for i in range(case["batch"]):  # an image at a time: the parameters' gradients add up
        x = state["x"][i:i + 1].double().requires_grad_(case["train"])
        with torch.set_grad_enabled(case["train"]):
            y = _EXACT_ACT[case["act"]](torch.nn.functional.group_norm(x, case["groups"], *params, eps=1e-5))
        if case["train"]:
            y.backward(state["gy"][i:i + 1].double())
            gxs.append(x.grad)
        ys.append(y.detach())
    y = torch.cat(ys)
    return [y, torch.cat(gxs)] + [p.grad for p in params] if case["train"] else y


def _exact_classify(state):
    case = state["case"]
    weight, bias = (v.double().squeeze().view(case["classes"], *(() if k == "bias" else (-1,)))
                    for k, v in state["params"].items())
    weight.requires_grad_(case["train"])
    bias.requires_grad_(case["train"])
    count = int((state["target"] != -100).sum()) if case["reduction"] == "mean" else 1
    total, gxs = 0.0, []
    for i in range(case["batch"]):
        x = state["x"][i].double().requires_grad_(case["train"])
        with torch.set_grad_enabled(case["train"]):
            scores = torch.einsum("oc,chw->ohw", weight, x) + bias[:, None, None]
            loss = torch.nn.functional.cross_entropy(scores[None], state["target"][i:i + 1], reduction="sum",
                                                     ignore_index=-100) / count
        if case["train"]:
            loss.backward()
            gxs.append(x.grad)
        total = total + loss.detach()
    return [total, torch.stack(gxs), weight.grad[:, :, None], bias.grad] if case["train"] else total


def _exact_adamw(state):
    case, t = state["case"], STEP + 1
    params, moments = [], []
    for p, gr, kept, master in zip(state["params"], state["grads"], state["moments"], state["masters"]):
        if case["bits"] == 8:
            scale_of = lambda s, like: s.double().repeat_interleave(BLOCK)[:like.numel()].view(like.shape)  # noqa: E731
            m = kept[0].double() * kept[0].double().abs() * scale_of(kept[1], kept[0])
            v = (kept[2].double() ** 2 * scale_of(kept[3], kept[2])) ** 2
        else:
            m, v = kept[0].double(), kept[1].double()
        gr, value = gr.double(), (p if master is None else master).double()
        m, v = torch.lerp(m, gr, 1 - BETAS[0]), torch.lerp(v, gr ** 2, 1 - BETAS[1])
        mhat, vhat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
        params.append(value - state["lr"] * (DECAY * value + mhat / (vhat.sqrt() + EPS)))
        # (what a code next to the border between two stands for jumps: moments in 8 bits have no value that 64 bits come near)
        moments += [None, None] if case["bits"] == 8 else [m, v]
    return params + moments + (params if case["master"] else [])

