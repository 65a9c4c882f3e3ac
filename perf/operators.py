"""The channels-last layer operators as they are measured: group normalisation with an activation, and a matrix product with
bias, activation and residual in its epilogue, each forward and backward.

`run` is one pass through an operator, either in plain torch operations in 32 bits (`own` false) or through the calls of
optimaltextures_amd.ops (`own` true)."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5

if torch.cuda.is_available():
    DEVICE = torch.device("cuda")
else:
    DEVICE = torch.device("cpu")


# ------------------------------------------------------------------------------------------------ cases
def _norm(name, op, dtype, images, height, width, channels, groups, act, per_image=False, train=False):
    return dict(name=name, op=op, dtype=dtype, images=images, height=height, width=width, channels=channels, groups=groups,
                act=act, per_image=per_image, train=train)


def _product(name, op, dtype, rows, inner, outer, act, bias=True, residual=False, train=False):
    return dict(name=name, op=op, dtype=dtype, rows=rows, inner=inner, outer=outer, act=act, bias=bias, residual=residual,
                train=train)


def listed():
    return [
        # one small map at the narrowest width of the codec: what a single call costs
        _norm("norm f32 one 16x16x64", "norm", "f32", 1, 16, 16, 64, 8, "silu"),
        # ragged maps with a scale and a shift of each image's own (a style's statistics put onto a content's features)
        _norm("norm f16 3 37x53x96 styled", "norm", "f16", 3, 37, 53, 96, 6, "relu", per_image=True),
        # relu3_1 features of 64 textures at 512 pixels a side, the framework's benchmark batch, in a training step
        _norm("norm bf16 64 128x128x256", "norm", "bf16", 64, 128, 128, 256, 32, "silu", train=True),
        # relu4_1 features of eight such images, backward
        _norm("norm grad bf16 8 64x64x512", "norm_grad", "bf16", 8, 64, 64, 512, 32, "silu"),
        # relu2_1 features of a middle pass of the schedule, backward in full precision
        _norm("norm grad f32 4 112x112x128", "norm_grad", "f32", 4, 112, 112, 128, 8, "relu"),
        # one token or one pooled feature vector through a widening layer: latency and the weights' bytes
        _product("product bf16 1 512>2048", "product", "bf16", 1, 512, 2048, "silu"),
        # a handful of rows through the narrowing layer behind it, onto the residual stream
        _product("product f16 16 2048>512", "product", "f16", 16, 2048, 512, "none", residual=True),
        # sizes that divide nothing: rows that are not aligned, tiles that end in the middle
        _product("product bf16 1237 201>331", "product", "bf16", 1237, 201, 331, "gelu", residual=True),
        # a 1x1 convolution over the pixels of the benchmark batch
        _product("product bf16 1048576 256>256", "product", "bf16", 64 * 128 * 128, 256, 256, "gelu", residual=True),
        # a training step's projection of one image's relu3_1 features in full precision, with what its backward pass needs
        _product("product f32 16384 256>512", "product", "f32", 16384, 256, 512, "silu", train=True),
        # the widening layer of a training step of eight images at relu4_1: large products in both directions
        _product("product grad bf16 32768 512>2048", "product_grad", "bf16", 32768, 512, 2048, "gelu"),
        # a ragged layer's gradients in full precision (130 = a kept rank of a PCA, say)
        _product("product grad f32 5000 130>514", "product_grad", "f32", 5000, 130, 514, "silu"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "product", "product_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if op.startswith("norm"):
        groups = rng.choice([1, 2, 3, 5, 8, 16, 32])
        channels = groups * max(1, min(64, _log_int(rng, 3, 1024) // groups))
        height, width = _log_int(rng, 4, 160), _log_int(rng, 4, 160)
        images = max(1, min(_log_int(rng, 1, 64), (1 << 26) // (height * width * channels)))
        c = _norm("", op, dtype, images, height, width, channels, groups, act, per_image=rng.random() < 0.3,
                  train=op == "norm" and rng.random() < 0.5)
    else:
        inner, outer = _log_int(rng, 3, 4096), _log_int(rng, 3, 4096)
        if rng.random() < 0.5:  # half of the layers have widths that the 16-byte accesses divide
            inner, outer = (inner + 63) // 64 * 64, (outer + 63) // 64 * 64
        most = min((1 << 26) // max(inner, outer), int(1.3e11) // (2 * inner * outer) // (1 if dtype != "f32" else 8))
        rows = _log_int(rng, 1, max(2, min(1 << 18, most)))
        c = _product("", op, dtype, rows, inner, outer, act, bias=rng.random() < 0.8, residual=op == "product" and rng.random() < 0.5,
                     train=op == "product" and rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    t = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"].startswith("norm"):
        b, h, w, c = case["images"], case["height"], case["width"], case["channels"]
        # a convolution's outputs: every channel has a level and a spread of its own
        level, spread = _normal(gen, c) * 0.7, _normal(gen, c).abs() + 0.4
        s["x"] = torch.addcmul(level, _normal(gen, b, h, w, c), spread).to(t)
        shape = (b, c) if case["per_image"] else (c,)
        s["weight"] = (1 + 0.3 * _normal(gen, *shape)).to(t)
        s["bias"] = (0.3 * _normal(gen, *shape)).to(t)
        if case["op"] == "norm_grad":
            s["dy"] = _normal(gen, b, h, w, c).to(t)
            g = case["groups"]
            xg = s["x"].double().view(b, h * w, g, c // g)
            mean = xg.mean(dim=(1, 3))
            var = (xg - mean.view(b, 1, g, 1)).square().mean(dim=(1, 3))
            s["mean"], s["rstd"] = mean.float(), (var + EPS).rsqrt().float()
    else:
        n, k, m = case["rows"], case["inner"], case["outer"]
        s["x"] = _normal(gen, n, k).to(t)
        s["w"] = (_normal(gen, m, k) / math.sqrt(k)).to(t)
        s["bias"] = (0.3 * _normal(gen, m)).to(t) if case["bias"] else None
        s["residual"] = _normal(gen, n, m).to(t) if case["residual"] else None
        if case["op"] == "product_grad":
            pre = s["x"].float() @ s["w"].float().t()
            s["pre"] = (pre if s["bias"] is None else pre + s["bias"].float()).to(t)
            s["dy"] = _normal(gen, n, m).to(t)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _per_channel(p, like):
    """weight or bias in 32 bits, over [images, pixels, groups, channels of a group]"""
    b, _, g, c = like.shape
    return p.float().view(-1, 1, g, c)


def _norm_plain(s):
    c = s["case"]
    x = s["x"]
    b, g, ch = c["images"], c["groups"], c["channels"]
    v = x.float().view(b, -1, g, ch // g)
    mean = v.mean(dim=(1, 3), keepdim=True)
    v = v - mean
    rstd = 1 / torch.sqrt((v * v).mean(dim=(1, 3), keepdim=True) + EPS)
    z = v * rstd * _per_channel(s["weight"], v) + _per_channel(s["bias"], v)
    y = _act(z, c["act"]).to(x.dtype).view(x.shape)
    return (y, mean.view(b, g), rstd.view(b, g)) if c["train"] else y


def _norm_grad_plain(s):
    c = s["case"]
    x = s["x"]
    b, g, ch = c["images"], c["groups"], c["channels"]
    v = x.float().view(b, -1, g, ch // g)
    rstd = s["rstd"].view(b, 1, g, 1)
    xhat = (v - s["mean"].view(b, 1, g, 1)) * rstd
    w = _per_channel(s["weight"], v)
    dz = s["dy"].float().view(v.shape) * _act_grad(xhat * w + _per_channel(s["bias"], v), c["act"])
    over = (1,) if c["per_image"] else (0, 1)
    shape = (b, ch) if c["per_image"] else (ch,)
    dweight, dbias = (dz * xhat).sum(dim=over).view(shape), dz.sum(dim=over).view(shape)
    dxhat = dz * w
    dx = rstd * (dxhat - dxhat.mean(dim=(1, 3), keepdim=True) - xhat * (dxhat * xhat).mean(dim=(1, 3), keepdim=True))
    return dx.to(x.dtype).view(x.shape), dweight.to(s["weight"].dtype), dbias.to(s["bias"].dtype)


def _product_plain(s):
    c, t = s["case"], s["x"].dtype
    pre = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    y = _act(pre, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (y.to(t), pre.to(t)) if c["train"] else y.to(t)


def _product_grad_plain(s):
    t = s["x"].dtype
    d = s["dy"].float() * _act_grad(s["pre"].float(), s["case"]["act"])
    out = [(d @ s["w"].float()).to(t), (d.t() @ s["x"].float()).to(t)]
    return out + [d.sum(dim=0).to(t)] if s["bias"] is not None else out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if not own:
        return {"norm": _norm_plain, "norm_grad": _norm_grad_plain, "product": _product_plain,
                "product_grad": _product_grad_plain}[c["op"]](state)
    from optimaltextures_amd import ops
    if c["op"] == "norm":
        return ops.group_norm(state["x"], c["groups"], state["weight"], state["bias"], eps=EPS, act=c["act"], want_stats=c["train"])
    if c["op"] == "norm_grad":
        return ops.group_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], c["groups"], state["weight"],
                                       state["bias"], act=c["act"])
    if c["op"] == "product":
        return ops.gemm_bias_act(state["x"], state["w"], state["bias"], act=c["act"], residual=state["residual"],
                                 want_pre=c["train"])
    out = ops.gemm_bias_act_backward(state["dy"], state["x"], state["w"], state["pre"], act=c["act"], want_bias=c["bias"])
    return out if c["bias"] else out[:2]


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"].startswith("norm"):
        e = case["images"] * case["height"] * case["width"] * case["channels"]
        params = 2 * case["channels"] * (case["images"] if case["per_image"] else 1) * size
        stats = 8 * case["images"] * case["groups"]
        if case["op"] == "norm":
            return {"bytes": 2 * e * size + params + (stats if case["train"] else 0), "flops": 12 * e}
        return {"bytes": 3 * e * size + 2 * params + stats, "flops": 24 * e}
    n, k, m = case["rows"], case["inner"], case["outer"]
    bias = m if case["bias"] else 0
    if case["op"] == "product":
        rows = 1 + (1 if case["residual"] else 0) + (1 if case["train"] else 0)
        return {"bytes": size * (n * k + m * k + bias + rows * n * m), "flops": 2 * n * k * m}
    return {"bytes": size * (2 * n * k + 2 * m * k + 2 * n * m + bias), "flops": 4 * n * k * m}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _sigma64(z):
    return torch.special.expit(z)


def _act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp_min(0), "silu": lambda: z * _sigma64(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[act]()


def _slope64(z, act):
    if act == "relu":
        return torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if act == "silu":
        p = _sigma64(z)
        return p + z * p * _sigma64(-z)
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    act = case["act"]
    if case["op"].startswith("norm"):
        b, c, g = case["images"], case["channels"], case["groups"]
        # channels in front: [images, groups, channels of a group, pixels]
        x = d["x"].flatten(1, 2).transpose(1, 2).reshape(b, g, c // g, -1)
        w, off = (p.reshape(-1, g, c // g, 1) for p in (d["weight"], d["bias"]))
        back = lambda v: v.reshape(b, c, -1).transpose(1, 2).reshape(s["x"].shape)  # noqa: E731
        if case["op"] == "norm":
            var, mean = torch.var_mean(x.flatten(2), dim=2, correction=0)
            rstd = (var + EPS) ** -0.5
            y = back(_act64((x - mean[..., None, None]) * (rstd[..., None, None] * w) + off, act))
            return (y, mean, rstd) if case["train"] else y
        rstd = d["rstd"][..., None, None]
        h = (x - d["mean"][..., None, None]) * rstd
        dz = d["dy"].flatten(1, 2).transpose(1, 2).reshape(x.shape) * _slope64(h * w + off, act)
        dw, db = (dz * h).sum(3).reshape(b, c), dz.sum(3).reshape(b, c)
        if not case["per_image"]:
            dw, db = dw.sum(0), db.sum(0)
        e = dz * w
        count = e[0, 0].numel()
        dx = rstd * (e - (e.sum((2, 3), keepdim=True) + h * (e * h).sum((2, 3), keepdim=True)) / count)
        return back(dx), dw, db
    if case["op"] == "product":
        z = torch.mm(d["x"], d["w"].t().contiguous())
        if "bias" in d:
            z += d["bias"]
        y = _act64(z, act)
        if "residual" in d:
            y = y + d["residual"]
        return (y, z) if case["train"] else y
    e = d["dy"] * _slope64(d["pre"], act)
    out = [torch.mm(e, d["w"]), torch.mm(e.t().contiguous(), d["x"])]
    return out + [e.sum(0)] if case["bias"] else out
