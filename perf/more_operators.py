"""Performance cases of two more operators that train a neural shader over the framework's images.

Each through public entry points:

  layer_norm  layer normalisation of each pixel's channels (or of any rows) with an activation
              (opendressi_amd.ops.layer_norm, layer_norm_bwd): forward alone, or forward and
              backward to the rows, the weight and the bias
  clip        the norm of all gradients of many parameters, and the gradients clipped to it in
              place (opendressi_amd.torch.clip_grad_norm_): the 2-norm or the largest magnitude

With `own` false, `run` computes the same in elementary torch operations in 32 bits (a norm's sum
of squares in 64).
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _decoder(width, layers, features, out):
    """The shapes of a per-pixel decoder: linear layers with a normalisation between them."""
    dims = [features] + [width] * layers
    body = ["%dx%d %d %d %d" % (b, a, b, b, b) for a, b in zip(dims, dims[1:])]
    return " ".join(body + ["%dx%d %d" % (out, width, out)])


def listed():
    return [
        # one latent code on its way through a trained shader: latency is all there is
        {"name": "layer_row_256", "kind": "layer_norm", "direction": "forward", "rows": "1",
         "c": 256, "wide": 256, "type": "bfloat16", "affine": "bfloat16", "activation": "silu"},
        # one frame of a 512 x 512 view: 64 of the 96 channels of an image of features
        {"name": "layer_512x512x64of96", "kind": "layer_norm", "direction": "forward",
         "rows": "1x512x512", "c": 64, "wide": 96, "type": "bfloat16", "affine": "float32",
         "activation": "silu"},
        # the largest: eight 1024 x 1024 views
        {"name": "layer_8x1024x1024x64", "kind": "layer_norm", "direction": "forward",
         "rows": "8x1024x1024", "c": 64, "wide": 64, "type": "bfloat16", "affine": "float32",
         "activation": "silu"},
        # a training step's pass over four 256 x 256 views
        {"name": "layer_train_4x256x256x64", "kind": "layer_norm", "direction": "train",
         "rows": "4x256x256", "c": 64, "wide": 64, "type": "float32", "affine": "float32",
         "activation": "gelu"},
        # the raggedest: odd image, odd channels
        {"name": "layer_train_3x61x97x33", "kind": "layer_norm", "direction": "train",
         "rows": "3x61x97", "c": 33, "wide": 33, "type": "float16", "affine": "float16",
         "activation": "gelu"},
        # few wide rows: the latent codes of a batch of patches
        {"name": "layer_train_1021x4096", "kind": "layer_norm", "direction": "train",
         "rows": "1021", "c": 4096, "wide": 4096, "type": "bfloat16", "affine": "float32",
         "activation": "none"},
        # the largest training pass
        {"name": "layer_train_4x1024x1024x64", "kind": "layer_norm", "direction": "train",
         "rows": "4x1024x1024", "c": 64, "wide": 64, "type": "bfloat16", "affine": "float32",
         "activation": "silu"},
        # the gradients of a small fit: vertices of a 1280-face mesh, an exposure and a background
        # colour; launches and latency are all there is
        {"name": "clip_leaves", "kind": "clip", "tensors": "642x3 1 3", "type": "float32",
         "norm": 2.0, "limit": 0.5},
        # a material fit whose gradients are watched and seldom clipped (not this time): vertices,
        # albedo and metallic-roughness textures and the environment
        {"name": "clip_materials", "kind": "clip",
         "tensors": "10242x3 512x512x3 512x512x3 256x512x3", "type": "float32", "norm": 2.0,
         "limit": 2.0},
        # a decoder network in bfloat16: many tensors, most tiny
        {"name": "clip_decoder", "kind": "clip", "tensors": _decoder(256, 10, 27, 3),
         "type": "bfloat16", "norm": 2.0, "limit": 0.5},
        # vertices in float32 beside networks in both 16-bit types, odd sizes, the largest
        # magnitude's norm
        {"name": "clip_mixed_largest", "kind": "clip",
         "tensors": "10242x3 97x61 97 5023x3 33x97 33 1 31 65x33 65 1x3 3x65 3 12289",
         "type": "mixed", "norm": math.inf, "limit": 0.5},
        # a scene's textures, 16 of 2048 x 2048 x 4: memory traffic is all there is
        {"name": "clip_textures", "kind": "clip", "tensors": " ".join(["2048x2048x4"] * 16),
         "type": "float32", "norm": 2.0, "limit": 0.5},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    if rng.random() < 0.4:
        total, count = _log(rng, 500, 2 ** 28), rng.randint(1, 50)
        parts = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(count)]
        sizes = [max(1, int(total * p / sum(parts))) for p in parts]
        return {"kind": "clip", "tensors": " ".join(str(s) for s in sizes),
                "type": rng.choice(["float32", "bfloat16", "float16", "mixed"]),
                "norm": rng.choice([2.0, 2.0, math.inf]), "limit": rng.choice([0.5, 0.9, 2.0])}
    direction = rng.choice(["forward", "train"])
    c = _log(rng, 8, 16384)
    if rng.random() < 0.5:
        c = -(-c // 8) * 8
    rows = _log(rng, 1, (2 ** 28 if direction == "forward" else 2 ** 27) // c)
    # relu's slope jumps at zero, where a mean's last bit decides on which side a value lies
    smooth = ["none", "silu", "gelu"]
    kind = rng.choice(["float32", "bfloat16", "float16"])
    return {"kind": "layer_norm", "direction": direction, "rows": str(rows), "c": c,
            "wide": c + rng.choice([0, 0, 0, 1, 8, 33]), "type": kind,
            "affine": rng.choice(["float32", kind]),
            "activation": rng.choice(smooth if direction == "train" else smooth + ["relu"])}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

_CTX = []


def _context():
    if not _CTX:
        import opendressi_amd.torch as dr
        _CTX.append(dr.RasterizeHipContext())
    return _CTX[0]


def _sizes(text):
    return tuple(int(d) for d in text.split("x"))


def _types(case):
    """Each tensor's type."""
    n = len(case["tensors"].split())
    if case["type"] != "mixed":
        return [TYPES[case["type"]]] * n
    return [list(TYPES.values())[i % 3] for i in range(n)]


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    if case["kind"] == "layer_norm":
        lead, c, wide = _sizes(case["rows"]), case["c"], case["wide"]
        kind, rows = TYPES[case["type"]], math.prod(lead)
        # features of a layer before: channels differ in size and mean, and so do pixels
        scale, shift = 0.5 + rand(wide), randn(wide)
        x = torch.empty((rows, wide), dtype=kind, device="cuda")
        gy = torch.empty((rows, c), dtype=kind, device="cuda") \
            if case["direction"] == "train" else None
        step = max(1, 2 ** 26 // wide)
        for i in range(0, rows, step):
            n = min(step, rows - i)
            x[i:i + n] = (randn(n, wide) * scale + shift) * (0.2 + rand(n, 1))
            if gy is not None:
                gy[i:i + n] = randn(n, c) * 0.1
        first = (wide - c) // 2
        return {"x": x.view(*lead, wide)[..., first:first + c],
                "gy": None if gy is None else gy.view(*lead, c),
                "weight": (1.0 + 0.1 * randn(c)).to(TYPES[case["affine"]]),
                "bias": (0.1 * randn(c)).to(TYPES[case["affine"]])}
    grads = []
    for shape, kind in zip(map(_sizes, case["tensors"].split()), _types(case)):
        size = 10.0 ** float(rand(1) * 3 - 4)  # tensors differ in their gradients' size
        g = randn(*shape) * size
        g *= rand(*shape) < 0.8  # what no view saw this time has no gradient
        grads.append(g.to(kind))
    largest = case["norm"] == math.inf
    norm = max(float(g.abs().max()) for g in grads) if largest else \
        math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    return {"grads": grads, "max_norm": float("%.3g" % (case["limit"] * norm))}


def prepare(case, seed):
    """What a program has in hand in the midst of a network, or after a backward pass."""
    s = {**_inputs(case, seed), "case": case}
    if case["kind"] == "clip":
        s["params"] = [torch.zeros_like(g) for g in s["grads"]]
        for p, g in zip(s["params"], s["grads"]):
            p.grad = g
    if own:
        s["ctx"] = _context()
    return s


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------

def _act(z, name):
    """(activation, derivative) of z."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _layer_norm(s):
    case, kind = s["case"], s["x"].dtype
    w, b = s["weight"].float(), s["bias"].float()
    d = s["x"].float()
    d = d - d.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    xh = d * rstd
    del d
    y, slope = _act(xh * w + b, case["activation"])
    out = {"y": y.to(kind)}
    if case["direction"] == "train":
        gz = s["gy"].float() * slope
        del y, slope
        c = case["c"]
        out["gb"] = gz.reshape(-1, c).sum(0).to(s["bias"].dtype)
        out["gw"] = (gz * xh).reshape(-1, c).sum(0).to(s["weight"].dtype)
        gz = gz * w
        out["gx"] = (rstd * (gz - gz.mean(-1, keepdim=True)
                             - xh * (gz * xh).mean(-1, keepdim=True))).to(kind)
    return out


def _clip(s):
    grads = s["grads"]
    if s["case"]["norm"] == math.inf:
        norm = torch.stack([g.abs().max().float() for g in grads]).max()
    else:
        norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return {"norm": norm, "grads": [g.copy_(g.float() * coef) for g in grads]}


def run(s):
    case = s["case"]
    if case["kind"] == "clip":
        if own:
            import opendressi_amd.torch as dr
            norm = dr.clip_grad_norm_(s["ctx"], s["params"], s["max_norm"], case["norm"])
            out = {"norm": norm, "grads": s["grads"]}
        else:
            out = _clip(s)
        if case["limit"] < 1.0:
            # clipped gradients would pass the same limit next time: a slowly falling one, so that
            # each pass has what a training step's has to do
            s["max_norm"] *= 0.9999
        return out
    if not own:
        return _layer_norm(s)
    from opendressi_amd import ops as K
    args = dict(weight=s["weight"], bias=s["bias"], activation=case["activation"])
    ctx = s["ctx"]._ctx
    if case["direction"] != "train":
        return {"y": K.layer_norm(ctx, s["x"], eps=EPS, stats=False, **args)[0]}
    y, mean, rstd = K.layer_norm(ctx, s["x"], eps=EPS, **args)
    gx, gw, gb = K.layer_norm_bwd(ctx, s["gy"], s["x"], mean, rstd, **args)
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}


def work(case):
    if case["kind"] == "clip":
        kinds = [2 if t.itemsize == 2 else 4 for t in _types(case)]
        counts = [math.prod(_sizes(t)) for t in case["tensors"].split()]
        read = sum(k * n for k, n in zip(kinds, counts))
        # gradients in, and out again where they are clipped
        return {"bytes": read * (2 if case["limit"] < 1.0 else 1) + 4, "flops": 3 * sum(counts)}
    e = math.prod(_sizes(case["rows"])) * case["c"]
    wide = 4 if case["type"] == "float32" else 2
    train = case["direction"] == "train"
    # x in, y out; x and gy in, y and gx out; weight and bias, and their gradients
    return {"bytes": e * wide * (4 if train else 2)
            + case["c"] * (4 if case["affine"] == "float32" else 2) * (4 if train else 2),
            "flops": e * (32 if train else 14)}


# --------------------------------------------------------------------------
# The definitions, in 64 bits
# --------------------------------------------------------------------------

def _exact_layer(case, d):
    """Forward by the definition, backward by automatic differentiation, some rows at a time:
    64 bits take room."""
    c, train = case["c"], case["direction"] == "train"
    x = d["x"].reshape(-1, c)
    weight = d["weight"].double().requires_grad_(train)
    bias = d["bias"].double().requires_grad_(train)
    f = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
         "gelu": lambda z: z * torch.special.ndtr(z)}[case["activation"]]
    ys, gxs = [], []
    for part, at in zip(x.split(max(1, 2 ** 26 // c)), range(0, len(x), max(1, 2 ** 26 // c))):
        v = part.double().requires_grad_(train)
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        y = f((v - mean) * (var + EPS) ** -0.5 * weight + bias)
        if train:
            y.backward(d["gy"].reshape(-1, c)[at:at + len(part)].double())
            gxs.append(v.grad)
        ys.append(y.detach())
    shape = d["x"].shape
    out = {"y": torch.cat(ys).view(shape)}
    if train:
        out.update(gx=torch.cat(gxs).view(shape), gw=weight.grad, gb=bias.grad)
    return out


def _exact_clip(case, d):
    wide = [g.double() for g in d["grads"]]
    norm = torch.linalg.vector_norm(
        torch.stack([torch.linalg.vector_norm(g, case["norm"]) for g in wide]), case["norm"])
    factor = min(1.0, d["max_norm"] / (float(norm) + 1e-6))
    return {"norm": norm, "grads": [g * factor for g in wide]}


def exact(case, seed):
    d = _inputs(case, seed)
    return _exact_clip(case, d) if case["kind"] == "clip" else _exact_layer(case, d)
