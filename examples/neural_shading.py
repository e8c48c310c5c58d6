"""A neural shader, trained through the torch surface.

A sphere carries eight learned features a vertex. Each step renders them from some cameras
(rasterize, interpolate), a small decoder turns a pixel's features and position into its colour
(linear layers in bfloat16 with group norm, or layer norm over each pixel's channels, and SiLU
between them), and the images are compared with those of a procedural surface. One AdamW, with
8-bit moments, float32 master weights and a clipped gradient norm, trains the features and the
decoder together; or, with --sgd, torch's SGD does, after the gradients have been clipped.

    python examples/neural_shading.py [--steps 200] [--size 256] [--views 4] [--norm layer] [--sgd]
"""
import argparse
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import opendressi_amd as od  # noqa: E402
import opendressi_amd.torch as dr  # noqa: E402


def cameras(count, angle):
    """Clip matrices of `count` cameras on a ring, turned by `angle`; OpenGL depth."""
    proj = od.perspective_vk(math.radians(45.0), 1.0, 0.1, 10.0).reshape(4, 4)
    out = []
    for i in range(count):
        a = angle + 2.0 * math.pi * i / count
        view = od.look_at([2.6 * math.sin(a), 0.8, 2.6 * math.cos(a)]).reshape(4, 4)
        m = view @ proj  # rows: column-major matrices
        m[:, 2] = 2.0 * m[:, 2] - m[:, 3]
        out.append(m)
    return torch.from_numpy(np.stack(out))


def surface_colour(p):
    """What the shader has to learn: stripes and a soft light over positions [..., 3]."""
    stripes = torch.sin(9.0 * p[..., 0] + 4.0 * torch.sin(5.0 * p[..., 1]))
    light = (p @ p.new_tensor([0.5, 0.7, 0.5])).clamp(min=0.0)
    return torch.stack([0.5 + 0.4 * stripes, 0.3 + 0.6 * light, 0.6 - 0.3 * stripes * light], -1)


class Decoder(torch.nn.Module):
    """Features [N, H, W, C] to colours [N, H, W, 3]."""

    def __init__(self, ctx, features, width=64, layers=3, groups=8, norm="group"):
        super().__init__()
        self.ctx, self.groups, self.norm = ctx, groups, norm
        dims = [features] + [width] * layers
        self.linear = torch.nn.ParameterList(
            torch.randn(b, a) / math.sqrt(a) for a, b in zip(dims, dims[1:] + [3]))
        self.scale = torch.nn.ParameterList(torch.ones(width) for _ in range(layers))
        self.shift = torch.nn.ParameterList(torch.zeros(width) for _ in range(layers))

    def forward(self, x):
        shape = x.shape[:-1]
        for w, scale, shift in zip(self.linear, self.scale, self.shift):
            x = (x.reshape(-1, x.shape[-1]) @ w.t()).view(*shape, w.shape[0])
            if self.norm == "layer":
                x = dr.layer_norm(self.ctx, x, scale, shift, activation="silu")
            else:
                x = dr.group_norm(self.ctx, x, self.groups, scale, shift, activation="silu")
        w = self.linear[-1]
        return torch.sigmoid((x.reshape(-1, x.shape[-1]) @ w.t()).view(*shape, 3).float())


def train(steps=200, size=256, views=4, level=4, lr=1e-2, seed=0, log=None, norm="group",
          sgd=False):
    """The loss of every step."""
    torch.manual_seed(seed)
    ctx = dr.RasterizeHipContext()
    dev = ctx.device
    pos, faces = od.icosphere(level)
    pos = torch.from_numpy(pos).to(dev)
    tri = torch.from_numpy(faces.astype(np.int32)).to(dev)
    hom = torch.cat([pos, torch.ones_like(pos[:, :1])], 1)

    features = [(0.1 * torch.randn(len(pos), 4, device=dev)).requires_grad_() for _ in range(2)]
    decoder = Decoder(ctx, 4 + 4 + 3, norm=norm).to(device=dev)
    params = features + list(decoder.parameters())
    if sgd:  # which keeps no master copies: weights stay in float32
        opt = torch.optim.SGD(params, lr=30 * lr, momentum=0.9)
    else:
        decoder.to(dtype=torch.bfloat16)
        opt = dr.AdamW(ctx, [dict(params=features, weight_decay=0.0),
                             dict(params=decoder.parameters(), lr=0.3 * lr)],
                       lr=lr, weight_decay=1e-3, state_bits=8, max_grad_norm=1.0, seed=seed)
    losses = []
    for step in range(steps):
        clip = hom @ cameras(views, 0.37 * step).to(dev)
        rast, _ = dr.rasterize(ctx, clip, tri, [size, size])
        where, _ = dr.interpolate(pos, rast, tri)
        seen = (rast[..., 3:] > 0).float()
        parts = [dr.interpolate(f, rast, tri)[0] for f in features]
        x = torch.cat(parts + [where], -1).to(decoder.scale[0].dtype)
        image = decoder(x) * seen
        loss = ((image - surface_colour(where) * seen) ** 2).sum() / seen.sum()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        grad_norm = dr.clip_grad_norm_(ctx, params, 0.1) if sgd else None
        opt.step()
        losses.append(loss.detach())
        if log and (step % log == 0 or step + 1 == steps):
            grad_norm = grad_norm if sgd else opt.grad_norm
            print(f"step {step:4d}  loss {float(losses[-1]):.5f}  gradient norm "
                  f"{float(grad_norm):.4f}", flush=True)
    return [float(x) for x in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--size", type=int, default=256)
    ap.add_argument("--views", type=int, default=4)
    ap.add_argument("--norm", choices=("group", "layer"), default="group")
    ap.add_argument("--sgd", action="store_true")
    args = ap.parse_args()
    losses = train(args.steps, args.size, args.views, log=20, norm=args.norm, sgd=args.sgd)
    print(f"loss {losses[0]:.5f} -> {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
