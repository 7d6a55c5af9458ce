"""What is measured of the rendering network's operators: group normalisation with an activation, the gate of a gated
convolution, and the two together, all on channels-last images. `listed()` names some cases, `draw()` gives more of the same
ranges, `prepare()` makes what a program has in hand before the call, `run()` is one pass, `work()` is what a pass cannot do
without and `exact()` the same results in 64 bits.

A case is a dict of plain values:
  op      "norm"   y = act(group_norm(x) * weight + bias)                      x [B,C,H,W]
          "gate"   y = act(f) * sigmoid(g)                                     x [B,2C,H,W] = features f, then gates g
          "gated_norm"  y = group_norm(act(f) * sigmoid(g)) * weight + bias    x [B,2C,H,W]
  b, h, w, c, groups, eps; act "none" | "relu" | "elu" | "silu"; dtype of the images, wdtype of weight and bias
  affine  whether there are weight and bias
  train   forward and backward (gradients of x, weight and bias) or the forward pass alone
  slice   x is the leading part of the channels of a wider image, as the two halves of a skip connection are
"""
import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5


def _case(name, op, b, h, w, c, groups=0, dtype="bfloat16", act="elu", wdtype="float32", affine=True, train=False, slice=False):
    return dict(name=name, op=op, b=b, h=h, w=w, c=c, groups=groups, eps=EPS, dtype=dtype, act=act, wdtype=wdtype, affine=affine,
                train=train, slice=slice)


def listed():
    return [
        # The coarsest level of a preview window's network: the launches are all there is.
        _case("norm_coarsest", "norm", 1, 8, 15, 64, 8, "float16", "silu", "float16"),
        # A preview window's finest level in the viewer.
        _case("norm_preview", "norm", 1, 180, 320, 32, 8, "bfloat16", "silu"),
        # The finest level of a 1080p frame in the viewer, sixteen features a pixel.
        _case("norm_1080p", "norm", 1, 1080, 1920, 16, 4, "float16", "relu", "float16"),
        # Training on a batch of 512 x 512 crops.
        _case("norm_train_crops", "norm", 4, 512, 512, 32, 8, "bfloat16", "silu", train=True),
        # The bottom of the network in training: many channels, few pixels, a batch of sixteen views.
        _case("norm_train_deep", "norm", 16, 32, 32, 512, 32, "bfloat16", "silu", train=True),
        # Uneven sizes in full precision, on one half of a skip connection.
        _case("norm_train_skip", "norm", 3, 77, 135, 20, 5, "float32", "elu", train=True, slice=True),
        # The gate of a block without normalisation at a 1080p frame's fourth level, in the viewer.
        _case("gate_preview", "gate", 1, 135, 240, 16, dtype="float16"),
        # The same in training as the reference ships it: full precision, crops, few channels.
        _case("gate_train_crops", "gate", 4, 512, 512, 8, dtype="float32", train=True),
        # The finest level of a 4K frame.
        _case("gate_4k", "gate", 1, 2160, 3840, 8),
        # A gated block with normalisation: a 1080p frame's third level in the viewer, crops in training, and the benchmark's
        # sixteen views at their second level.
        _case("gated_norm_preview", "gated_norm", 1, 270, 480, 16, 4, "float16", wdtype="float16"),
        _case("gated_norm_train_crops", "gated_norm", 4, 512, 512, 16, 4, train=True),
        _case("gated_norm_train_views", "gated_norm", 16, 540, 960, 16, 4, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "gate", "gated_norm"])
    train = rng.random() < 0.6
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
    c = groups * rng.choice([1, 2, 3, 4, 4, 6, 8, 8, 16])
    values = _log_int(rng, 8_000, 60_000_000)  # of x (of the features, for a gated operator)
    pixels = max(12, values // c)
    b = min(_log_int(rng, 1, 16), max(1, pixels // 12))
    w = max(3, min(3840, int(math.sqrt(pixels / b * rng.uniform(1.0, 1.9)))))
    h = max(2, min(2160, pixels // (b * w)))
    # the corner of relu is a border that two correct results may lie on either side of in its derivative
    act = rng.choice(["none", "elu", "silu"] if train else ["none", "relu", "elu", "silu"])
    c_ = _case(None, op, b, h, w, c, groups if op != "gate" else 0, dtype, act, rng.choice(["float32", dtype]),
               op != "gate" and rng.random() < 0.85, train, rng.random() < 0.2)
    del c_["name"]
    return c_


# ---- inputs -------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dtype, wdtype = getattr(torch, case["dtype"]), getattr(torch, case["wdtype"])
    b, h, w, c = case["b"], case["h"], case["w"], case["c"]
    cx = c if case["op"] == "norm" else 2 * c
    wide = 2 * cx if case["slice"] else cx
    # what a convolution puts out: every channel with a mean and a spread of its own
    x = torch.randn((b, h, w, wide), device=DEV, generator=g)
    x.mul_(0.5 + torch.rand(wide, device=DEV, generator=g)).add_(0.5 * torch.randn(wide, device=DEV, generator=g))
    x = x.to(dtype).permute(0, 3, 1, 2)[:, :cx]  # channels last
    s = dict(case=case, x=x, weight=None, bias=None, dy=None)
    if case["op"] != "gate" and case["affine"]:
        s["weight"] = (1 + 0.2 * torch.randn(c, device=DEV, generator=g)).to(wdtype)
        s["bias"] = (0.2 * torch.randn(c, device=DEV, generator=g)).to(wdtype)
    if case["train"]:
        s["dy"] = torch.randn((b, h, w, c), device=DEV, generator=g).to(dtype).permute(0, 3, 1, 2)
        for k in ("x", "weight", "bias"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    ops = _operators()
    case = s["case"]
    if case["op"] == "norm":
        y = ops.group_norm(s["x"], case["groups"], s["weight"], s["bias"], case["eps"], case["act"])
    elif case["op"] == "gate":
        y = ops.gated_activation(s["x"], case["act"])
    else:
        y = ops.gated_group_norm(s["x"], case["groups"], s["weight"], s["bias"], case["eps"], case["act"])
    if not case["train"]:
        return [y]
    leaves = [s[k] for k in ("x", "weight", "bias") if s[k] is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


_loaded = None


def _operators():
    global _loaded
    if _loaded is None:
        from adop_b200 import build
        torch.ops.load_library(build.TORCH_OP_LIB)
        _loaded = torch.ops.adop
    return _loaded


def _act(v, kind):
    if kind == "relu":
        return v.clamp(min=0)
    if kind == "elu":
        return torch.where(v > 0, v, torch.expm1(v))
    return v * torch.sigmoid(v) if kind == "silu" else v


def _act_slope(v, kind):
    if kind == "relu":
        return (v > 0).to(v.dtype)
    if kind == "elu":
        return torch.where(v > 0, torch.ones_like(v), torch.exp(v))
    if kind == "silu":
        s = torch.sigmoid(v)
        return s * (1 + v * (1 - s))
    return torch.ones_like(v)


def _plain(s):
    case = s["case"]
    with torch.no_grad():
        x = s["x"].float()
        b, c, h, w = case["b"], case["c"], case["h"], case["w"]
        norm, act = case["op"] != "gate", case["act"]
        if case["op"] == "norm":
            u = x
        else:
            f, gate = x[:, :c], torch.sigmoid(x[:, c:])
            fa = _act(f, act)
            u = fa * gate
        z = u
        if norm:
            grouped = u.reshape(b, case["groups"], -1)
            mean = grouped.mean(2, keepdim=True)
            rstd = torch.rsqrt((grouped - mean).square().mean(2, keepdim=True) + case["eps"])
            uhat = ((grouped - mean) * rstd).reshape(b, c, h, w)
            weight = s["weight"].float().reshape(1, c, 1, 1) if s["weight"] is not None else 1.0
            z = uhat * weight
            if s["bias"] is not None:
                z = z + s["bias"].float().reshape(1, c, 1, 1)
        y = _act(z, act) if case["op"] == "norm" else z
        out = [y.to(s["x"].dtype)]
        if not case["train"]:
            return out
        du = s["dy"].float()
        if case["op"] == "norm":
            du = du * _act_slope(z, act)
        params = []
        if norm:
            if s["weight"] is not None:
                params = [(du * uhat).sum((0, 2, 3)).to(s["weight"].dtype), du.sum((0, 2, 3)).to(s["bias"].dtype)]
            du = (du * weight).reshape(b, case["groups"], -1)
            uhat = uhat.reshape(b, case["groups"], -1)
            du = rstd * (du - du.mean(2, keepdim=True) - uhat * (du * uhat).mean(2, keepdim=True))
            du = du.reshape(b, c, h, w)
        if case["op"] == "norm":
            dx = du
        else:
            dx = torch.cat([du * gate * _act_slope(f, act), du * fa * gate * (1 - gate)], 1)
        return out + [dx.to(s["x"].dtype)] + params


# ---- what a pass cannot do without, and its results in 64 bits ------------------------------------------------------------
def work(case):
    n = case["b"] * case["h"] * case["w"] * case["c"]
    size = 4 if case["dtype"] == "float32" else 2
    wsize = 4 if case["wdtype"] == "float32" else 2
    per_value = (1 if case["op"] == "norm" else 2) + 1  # x read, y written
    flops = {"norm": 14, "gate": 10, "gated_norm": 20}[case["op"]]
    params = 2 * case["c"] if case["affine"] else 0
    if case["train"]:
        per_value *= 2  # the gradient of y read, that of x written
        flops *= 3
        params *= 2
    return {"bytes": n * per_value * size + params * wsize, "flops": n * flops}


def exact(case, seed):
    """The definitions in 64 bits, the gradients by automatic differentiation."""
    s = prepare(case, seed)
    leaves = {k: s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias") if s[k] is not None}
    functions = {"none": lambda v: v, "relu": torch.relu, "elu": torch.nn.functional.elu, "silu": torch.nn.functional.silu}
    act = functions[case["act"]]
    y = leaves["x"]
    if case["op"] != "norm":
        features, gates = y.chunk(2, 1)
        y = act(features) / (1 + torch.exp(-gates))
    if case["op"] != "gate":
        image = y.unflatten(1, (case["groups"], -1))
        var, mean = torch.var_mean(image, (2, 3, 4), correction=0, keepdim=True)
        y = ((image - mean) / torch.sqrt(var + case["eps"])).flatten(1, 2)
        if "weight" in leaves:
            y = y * leaves["weight"][:, None, None] + leaves["bias"][:, None, None]
        if case["op"] == "norm":
            y = act(y)
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), s["dy"].double())]
