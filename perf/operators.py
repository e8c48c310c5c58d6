"""Performance cases of the operators that train a neural shader over the framework's images.

Two operators, each through public entry points:

  adamw       one AdamW step over all parameter tensors at once (opendressi_amd.torch.AdamW):
              moments in 32 bits or in 8, parameters in float32, or in 16 bits with a float32
              master copy, and the gradients clipped to a global norm where asked
  group_norm  group normalisation of channels-last images with an activation
              (opendressi_amd.ops.group_norm, group_norm_bwd): forward alone, or forward and
              backward to the image, the weight and the bias

With `own` false, `run` computes the same in elementary torch operations in 32 bits.

The moments of all parameters lie in one flat buffer, in the parameters' order, each parameter's
share padded with zeros to a multiple of 32 elements. In 8 bits, 32 neighbours share the largest
exponent field E among them; with f = |x| 2^(T - max(E, T)), T 14 for the first moment and 30 for
the second, the code is (bits of f + r) >> 20 with r a random number below 2^20: a float of 3
mantissa bits whose rounding is right on average. The first moment's sign is the code's top bit.
r comes from a hash of the element's index and the step, so it is the same on both sides.
"""
import math

import torch

own = False

BLOCK = 32
TOP1, TOP2 = 14, 30  # the exponent field of a block's largest value: first, second moment
STEP = 1000          # steps that the resumed training has behind it
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _decoder(width, layers, features, out):
    """The shapes of a per-pixel decoder: linear layers with group norm between them."""
    dims = [features] + [width] * layers
    body = ["%dx%d %d %d %d" % (b, a, b, b, b) for a, b in zip(dims, dims[1:])]
    return " ".join(body + ["%dx%d %d" % (out, width, out)])


def listed():
    return [
        # the leaves of a small fit: vertices of a 1280-face mesh, an exposure and a background
        # colour; launches and latency are all there is
        {"name": "adamw_leaves", "kind": "adamw", "tensors": "642x3 1 3", "type": "float32",
         "bits": 32, "clip": 0.0, "decay": 0.0},
        # a material fit: vertices, albedo and metallic-roughness textures and the environment
        # of the PBR workload, clipped
        {"name": "adamw_materials", "kind": "adamw",
         "tensors": "10242x3 512x512x3 512x512x3 256x512x3", "type": "float32", "bits": 32,
         "clip": 1.0, "decay": 0.01},
        # a decoder network in bfloat16 with a float32 master copy: many tensors, most tiny
        {"name": "adamw_decoder", "kind": "adamw", "tensors": _decoder(256, 10, 27, 3),
         "type": "bfloat16", "bits": 32, "clip": 1.0, "decay": 0.01},
        # the same kind of network in float16 with ragged widths and 8-bit moments
        {"name": "adamw_ragged_8bit", "kind": "adamw",
         "tensors": "97x61 97 33x97 33 1 31 65x33 65 3x65 3 12289", "type": "float16",
         "bits": 8, "clip": 0.0, "decay": 0.01},
        # a scene's textures, 16 of 2048 x 2048 x 4: memory traffic is all there is
        {"name": "adamw_textures", "kind": "adamw",
         "tensors": " ".join(["2048x2048x4"] * 16), "type": "float32", "bits": 32, "clip": 0.0,
         "decay": 0.0},
        # the same with 8-bit moments
        {"name": "adamw_textures_8bit", "kind": "adamw",
         "tensors": " ".join(["2048x2048x4"] * 16), "type": "float32", "bits": 8, "clip": 0.0,
         "decay": 0.0},
        # one small feature image: latency
        {"name": "norm_64x64x32", "kind": "group_norm", "direction": "forward", "n": 1, "h": 64,
         "w": 64, "c": 32, "groups": 8, "type": "float32", "activation": "relu"},
        # one frame of a 512 x 512 view in a trained shader
        {"name": "norm_512x512x64", "kind": "group_norm", "direction": "forward", "n": 1,
         "h": 512, "w": 512, "c": 64, "groups": 8, "type": "bfloat16", "activation": "silu"},
        # the largest: eight 1024 x 1024 views
        {"name": "norm_8x1024x1024x64", "kind": "group_norm", "direction": "forward", "n": 8,
         "h": 1024, "w": 1024, "c": 64, "groups": 16, "type": "bfloat16", "activation": "silu"},
        # a training step's pass over four 256 x 256 views
        {"name": "norm_train_4x256x256x64", "kind": "group_norm", "direction": "train", "n": 4,
         "h": 256, "w": 256, "c": 64, "groups": 8, "type": "float32", "activation": "silu"},
        # the raggedest: odd image, odd channels
        {"name": "norm_train_3x61x97x33", "kind": "group_norm", "direction": "train", "n": 3,
         "h": 61, "w": 97, "c": 33, "groups": 3, "type": "float16", "activation": "gelu"},
        # the largest training pass
        {"name": "norm_train_4x1024x1024x64", "kind": "group_norm", "direction": "train", "n": 4,
         "h": 1024, "w": 1024, "c": 64, "groups": 8, "type": "bfloat16", "activation": "silu"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    if rng.random() < 0.5:
        total, count = _log(rng, 500, 2 ** 27), rng.randint(1, 40)
        parts = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(count)]
        sizes = [max(1, int(total * p / sum(parts))) for p in parts]
        bits = rng.choice([32, 32, 8])
        # a clipped norm's last bit would decide some of the 8-bit roundings one way or the other
        return {"kind": "adamw", "tensors": " ".join(str(s) for s in sizes),
                "type": rng.choice(["float32", "float32", "bfloat16", "float16"]), "bits": bits,
                "clip": rng.choice([0.0, 1.0]) if bits == 32 else 0.0,
                "decay": rng.choice([0.0, 0.01])}
    c, groups = 1024, 1
    while c > 256:
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = groups * rng.choice([1, 2, 3, 4, 5, 8, 11, 16, 32])
    n = rng.randint(1, 8)
    h, w = _log(rng, 8, 1024), _log(rng, 8, 1024)
    while n * h * w * c > 2 ** 27:
        n, h = (n - 1, h) if n > 1 else (1, h // 2)
    direction = rng.choice(["forward", "train"])
    # relu's slope jumps at zero, where a mean's last bit decides on which side a value lies
    smooth = ["none", "silu", "gelu"]
    return {"kind": "group_norm", "direction": direction, "n": n, "h": h, "w": w, "c": c,
            "groups": groups, "type": rng.choice(["float32", "bfloat16", "float16"]),
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


def _shapes(case):
    return [tuple(int(d) for d in t.split("x")) for t in case["tensors"].split()]


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=gen, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    kind = TYPES[case["type"]]
    if case["kind"] == "group_norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        # features of a rendered object before a constant background
        yy = torch.linspace(-1.0, 1.0, h, device="cuda")[:, None, None]
        xx = torch.linspace(-1.0, 1.0, w, device="cuda")[None, :, None]
        seen = (yy * yy + xx * xx < 0.8).float()
        scale, shift = 0.5 + rand(c), randn(c)
        back = 0.5 * randn(c)
        x = torch.empty((n, h, w, c), dtype=kind, device="cuda")
        gy = torch.empty_like(x) if case["direction"] == "train" else None
        for i in range(n):
            x[i] = torch.where(seen > 0, randn(h, w, c) * scale + shift, back)
            if gy is not None:
                gy[i] = randn(h, w, c) * 0.1
        return {"x": x, "gy": gy, "weight": 1.0 + 0.1 * randn(c), "bias": 0.1 * randn(c)}
    shapes = _shapes(case)
    params, grads, ms, vs = [], [], [], []
    for s in shapes:
        n = math.prod(s)
        size = 10.0 ** float(rand(1) * 3 - 5)  # tensors differ in their gradients' size
        g = randn(n) * size
        # what no view saw this time has no gradient, but has its moments
        g *= (rand(n) < 0.8)
        m = 0.3 * size * randn(n)
        v = (size * (0.5 + rand(n))) ** 2
        params.append((randn(n) * 0.1).to(kind).view(s))
        grads.append(g.to(kind).view(s))
        pad = torch.zeros(_padded(n) - n, device="cuda")
        ms += [m, pad]
        vs += [v, pad]
        del g, m, v
    return {"params": params, "grads": grads, "m": torch.cat(ms), "v": torch.cat(vs)}


def prepare(case, seed):
    """What a program resumed from a checkpoint, or one in the midst of an image, has in hand."""
    s = {**_inputs(case, seed), "case": case}
    if case["kind"] == "group_norm":
        if own:
            s["ctx"] = _context()._ctx
        return s
    kept = {"step": [STEP] * len(s["params"])}
    if case["bits"] == 8:
        kept["exp_avg"], kept["exp_avg_scale"] = _encode(s["m"], TOP1, 1 << 19)
        kept["exp_avg_sq"], kept["exp_avg_sq_scale"] = _encode(s["v"], TOP2, 1 << 19)
    else:
        kept["exp_avg"], kept["exp_avg_sq"] = s["m"], s["v"]
    del s["m"], s["v"]
    if case["type"] != "float32":
        kept["master"] = torch.cat([_pad(p.float()) for p in s["params"]])
    if not own:
        # zeros that fill a parameter's share up, one for each
        s["pads"] = [torch.zeros(_padded(p.numel()) - p.numel(), device="cuda")
                     for p in s["params"]]
        s.update(kept, step=STEP)
        return s
    import opendressi_amd.torch as dr
    for p, g in zip(s["params"], s["grads"]):
        p.grad = g
    s["opt"] = dr.AdamW(_context(), s["params"], lr=1e-3, betas=(BETA1, BETA2), eps=EPS,
                        weight_decay=case["decay"], state_bits=case["bits"],
                        max_grad_norm=case["clip"] or None)
    s["opt"].load_state_dict(kept)
    return s


def _pad(t):
    t = t.reshape(-1)
    return torch.cat([t, t.new_zeros(_padded(t.numel()) - t.numel())])


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------

def _encode(x, top, r):
    """(codes, exponents) of flat float32 values, `r` below 2^20 for each or for all."""
    bits = x.abs().view(torch.int32)
    field = (bits >> 23).view(-1, BLOCK).amax(1)
    up = field.clamp(min=top) - top
    # two factors: 2^-(E - T) may not be a float32
    f = x.abs().view(-1, BLOCK) * _two_to(-up.clamp(max=100))[:, None]
    f = f * _two_to(-(up - up.clamp(max=100)))[:, None]
    code = (f.view(-1).view(torch.int32) + r) >> 20
    if top == TOP1:
        code = code | ((x.view(torch.int32) >> 24) & 128)
    else:
        code = torch.where(x > 0, code.clamp(min=1), code)
    return code.to(torch.uint8), field.to(torch.uint8)


def _two_to(e):
    """2^e for whole e of -126 .. 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _decode(code, field, top):
    code = code.to(torch.int32)
    sign = ((code & 128) << 24) if top == TOP1 else 0
    mag = (code & 127) if top == TOP1 else code
    up = field.to(torch.int32).clamp(min=top) - top
    f = (mag << 20).view(torch.float32).view(-1, BLOCK) * _two_to(up.clamp(max=100))[:, None]
    f = (f * _two_to(up - up.clamp(max=100))[:, None]).view(-1)
    return (f.view(torch.int32) | sign).view(torch.float32)


def _noise(n, step):
    """32 random bits for each element of a step."""
    mix = lambda x: x & 0xffffffff  # noqa: E731
    key = (step * 0x9e3779b9 + 0x7f4a7c15) & 0xffffffff  # seed 0
    x = torch.arange(n, device="cuda") ^ key
    x = mix((x ^ (x >> 16)) * 0x7feb352d)
    x = mix((x ^ (x >> 15)) * 0x846ca68b)
    return x ^ (x >> 16)


def _adamw(s):
    case = s["case"]
    s["step"] += 1
    t, lr = s["step"], 1e-3
    both = lambda ts: torch.cat([x for t, z in zip(ts, s["pads"])  # noqa: E731
                                 for x in (t.reshape(-1).float(), z)])
    g = both(s["grads"])
    p = s["master"] if case["type"] != "float32" else both(s["params"])
    out = {}
    if case["clip"]:
        norm = torch.sqrt((g * g).sum())
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0)
        out["grad_norm"] = norm
    if case["bits"] == 8:
        m = _decode(s["exp_avg"], s["exp_avg_scale"], TOP1)
        v = _decode(s["exp_avg_sq"], s["exp_avg_sq_scale"], TOP2)
    else:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    den = torch.sqrt(v) * (1 / math.sqrt(1 - BETA2 ** t)) + EPS
    p = p * (1 - lr * case["decay"]) - (m / den) * (lr / (1 - BETA1 ** t))
    if case["bits"] == 8:
        r = _noise(m.numel(), t)
        low, high = ((r & 0xffff) << 4) + 8, ((r >> 16) << 4) + 8
        s["exp_avg"], s["exp_avg_scale"] = _encode(m, TOP1, low.to(torch.int32))
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = _encode(v, TOP2, high.to(torch.int32))
        # three mantissa bits and an exponent: bfloat16 holds these values as they are
        out["m"] = _decode(s["exp_avg"], s["exp_avg_scale"], TOP1).bfloat16()
        out["v"] = _decode(s["exp_avg_sq"], s["exp_avg_sq_scale"], TOP2).bfloat16()
    else:
        s["exp_avg"], s["exp_avg_sq"] = m, v
        out["m"], out["v"] = m, v
    if case["type"] != "float32":
        s["master"] = out["master"] = p
    sizes = [k for q, z in zip(s["params"], s["pads"]) for k in (q.numel(), z.numel())]
    out["params"] = [q.copy_(x.view(q.shape))
                     for q, x in zip(s["params"], torch.split(p, sizes)[::2])]
    return out


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


def _group_norm(s):
    case, x = s["case"], s["x"]
    n, c, groups = case["n"], case["c"], case["groups"]
    per = (n, case["h"] * case["w"], groups, c // groups)
    w, b = s["weight"].view(per[2:]), s["bias"].view(per[2:])
    xf = x.float().view(per)
    mean = xf.mean((1, 3), keepdim=True)
    d = xf - mean
    del xf
    rstd = 1 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    xh = d * rstd
    del d
    y, slope = _act(xh * w + b, case["activation"])
    out = {"y": y.to(x.dtype).view(x.shape)}
    if case["direction"] == "train":
        gz = s["gy"].float().view(per) * slope
        del y, slope
        out["gb"] = gz.sum((0, 1)).view(c)
        out["gw"] = (gz * xh).sum((0, 1)).view(c)
        gz = gz * w
        gx = rstd * (gz - gz.mean((1, 3), keepdim=True)
                     - xh * (gz * xh).mean((1, 3), keepdim=True))
        out["gx"] = gx.to(x.dtype).view(x.shape)
    return out


def run(s):
    case = s["case"]
    if not own:
        return _adamw(s) if case["kind"] == "adamw" else _group_norm(s)
    if case["kind"] == "adamw":
        opt = s["opt"]
        opt.step()
        m, v = opt.moments()
        out = {"params": s["params"], "m": m, "v": v}
        if case["clip"]:
            out["grad_norm"] = opt.grad_norm
        if case["type"] != "float32":
            out["master"] = opt.master
        return out
    from opendressi_amd import ops as K
    args = dict(groups=case["groups"], weight=s["weight"], bias=s["bias"],
                activation=case["activation"])
    y, mean, rstd = K.group_norm(s["ctx"], s["x"], eps=1e-5, **args)
    if case["direction"] != "train":
        return {"y": y}
    gx, gw, gb = K.group_norm_bwd(s["ctx"], s["gy"], s["x"], mean, rstd, **args)
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}


def work(case):
    if case["kind"] == "adamw":
        e = sum(math.prod(t) for t in _shapes(case))
        wide = 4 if case["type"] == "float32" else 2
        read = 2 * wide if wide == 4 else wide + 4  # gradient and parameter (or its master)
        write = 4 if wide == 4 else 2 + 4
        moments = 16 if case["bits"] == 32 else 2 * (2 + 2 / BLOCK) + 4  # .. and their values
        return {"bytes": e * (read + write + moments), "flops": 15 * e}
    e = case["n"] * case["h"] * case["w"] * case["c"]
    wide = 4 if case["type"] == "float32" else 2
    train = case["direction"] == "train"
    # x in, y out; x and gy in, gx out
    return {"bytes": e * wide * (4 if train else 2) + 16 * case["c"],
            "flops": e * (30 if train else 12)}


# --------------------------------------------------------------------------
# The definitions, in 64 bits
# --------------------------------------------------------------------------

def _exact_norm(case, d):
    """Forward by the definition, backward by automatic differentiation."""
    n, h, w, c = d["x"].shape
    train = case["direction"] == "train"
    out = {"y": []}
    weight = d["weight"].double().requires_grad_(train)
    bias = d["bias"].double().requires_grad_(train)
    f = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
         "gelu": lambda z: z * torch.special.ndtr(z)}[case["activation"]]
    gx = []
    for i in range(n):  # an item at a time: 64 bits take room
        x = d["x"][i].double().requires_grad_(train)
        xg = x.reshape(h * w, case["groups"], -1).transpose(0, 1).reshape(case["groups"], -1)
        var, mean = torch.var_mean(xg, 1, correction=0, keepdim=True)
        z = ((xg - mean) * (var + 1e-5) ** -0.5).view(case["groups"], h * w, -1)
        y = f(z.transpose(0, 1).reshape(h, w, c) * weight + bias)
        if train:
            y.backward(d["gy"][i].double())
            gx.append(x.grad)
        out["y"].append(y.detach())
        del x, xg, z, y
    out["y"] = torch.stack(out["y"])
    if train:
        out.update(gx=torch.stack(gx), gw=weight.grad, gb=bias.grad)
    return out


def _exact_round(x, top, r):
    """x rounded to a code's value: down by its step after r 2^-20 of a step was added."""
    mag = x.abs().view(-1, BLOCK)
    e = torch.frexp(mag.amax(1))[1].clamp(min=top - 126) - 1  # of the block's largest
    low = e - (top - 1)  # of the smallest value that is not subnormal
    own_e = torch.maximum(torch.frexp(mag)[1] - 1, low[:, None])
    step = torch.ldexp(torch.ones_like(mag), own_e - 3)
    q = torch.floor(mag / step + r.view(-1, BLOCK).double() * 2.0 ** -20) * step
    if top == TOP2:
        least = torch.ldexp(torch.ones_like(mag), (low - 3)[:, None])
        q = torch.where(mag > 0, torch.maximum(q, least), q)
    return (q * torch.sign(x).view(-1, BLOCK)).view(-1)


def _exact_adamw(case, d):
    shares = [_padded(p.numel()) for p in d["params"]]
    g = torch.cat([_pad(x).double() for x in d["grads"]])
    p = torch.cat([_pad(x).double() for x in d["params"]])
    out = {}
    if case["clip"]:
        out["grad_norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(out["grad_norm"]) + 1e-6))
    m, v = d["m"], d["v"]
    if case["bits"] == 8:
        half = torch.tensor(1 << 19, device="cuda").expand(m.numel())
        m, v = _exact_round(m.double(), TOP1, half), _exact_round(v.double(), TOP2, half)
    t = STEP + 1
    m = m.double() + (1 - BETA1) * (g - m.double())
    v = v.double() + (1 - BETA2) * (g * g - v.double())
    hat = (v / (1 - BETA2 ** t)).sqrt()
    p = p - 1e-3 * (m / (1 - BETA1 ** t) / (hat + EPS) + case["decay"] * p)
    del g, hat
    if case["bits"] == 8:
        r = _noise(m.numel(), t)
        m = _exact_round(m, TOP1, ((r & 0xffff) << 4) + 8)
        v = _exact_round(v, TOP2, ((r >> 16) << 4) + 8)
    out.update(m=m, v=v)
    if case["type"] != "float32":
        out["master"] = p
    out["params"] = [x[:q.numel()].view(q.shape)
                     for q, x in zip(d["params"], torch.split(p, shares))]
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    return _exact_norm(case, d) if case["kind"] == "group_norm" else _exact_adamw(case, d)
