"""A small network beside a frozen cloud that learns how each photograph tints it: exposure and white balance change from
image to image, and splats that share their colours with all images cannot follow.

The head reads each splat's SH coefficients and the image's embedding and adds an offset to the splat's colour: a layer
norm over the coefficients, a linear layer, residual blocks of norm, linear, GELU, linear, and a last norm and linear layer.
Its training step is the framework's operators in the order a program uses them: the colours go through rasterize_fwd, the
image's L1 gradient comes back through rasterize_bwd, the head's backward runs layer_norm's, and AdamW clips the gradients'
norm and steps all tensors at once, with 8-bit moments if wanted. `python appearance_head.py` trains one on a synthetic
scene and prints the loss.
"""
from __future__ import annotations

import argparse
import math

import splatx_torch  # first: its HIP runtime is the process's
import torch

import numpy as np
import scene


class Block(torch.nn.Module):
    def __init__(self, hidden, dtype):
        super().__init__()
        self.norm_weight = torch.nn.Parameter(torch.ones(hidden))
        self.norm_bias = torch.nn.Parameter(torch.zeros(hidden))
        self.up = torch.nn.Linear(hidden, hidden, dtype=dtype)
        self.down = torch.nn.Linear(hidden, hidden, dtype=dtype)

    def forward(self, backend, stream, update):
        """(the residual stream with the last block's update added, this block's update)"""
        if update is None:
            y = splatx_torch.layer_norm(backend, stream, self.norm_weight, self.norm_bias)
        else:
            y, stream = splatx_torch.layer_norm(backend, stream, self.norm_weight, self.norm_bias, residual=update)
        return stream, self.down(torch.nn.functional.gelu(self.up(y)))


class AppearanceHead(torch.nn.Module):
    """Colour offsets [splats, 3] of the splats' features in one image."""

    def __init__(self, backend, features, images, hidden=64, embedding=16, blocks=2, dtype=torch.bfloat16):
        super().__init__()
        self.backend = backend
        self.norm_weight = torch.nn.Parameter(torch.ones(features))
        self.norm_bias = torch.nn.Parameter(torch.zeros(features))
        self.embedding = torch.nn.Parameter(0.1 * torch.randn(images, embedding, dtype=dtype))
        self.enter = torch.nn.Linear(features, hidden, dtype=dtype)
        self.mix = torch.nn.Linear(embedding, hidden, bias=False, dtype=dtype)
        self.blocks = torch.nn.ModuleList(Block(hidden, dtype) for _ in range(blocks))
        self.last_weight = torch.nn.Parameter(torch.ones(hidden))
        self.last_bias = torch.nn.Parameter(torch.zeros(hidden))
        self.leave = torch.nn.Linear(hidden, 3, dtype=dtype)
        torch.nn.init.zeros_(self.leave.weight)
        torch.nn.init.zeros_(self.leave.bias)
        self.to(backend.device)

    def forward(self, features, image):
        x = splatx_torch.layer_norm(self.backend, features, self.norm_weight, self.norm_bias)
        stream, update = self.enter(x) + self.mix(self.embedding[image]), None
        for block in self.blocks:
            stream, update = block(self.backend, stream, update)
        y, _ = splatx_torch.layer_norm(self.backend, stream, self.last_weight, self.last_bias, residual=update)
        return self.leave(y).float()


def optimizer(head, lr=2e-3, state_bits=32, max_norm=1.0):
    """AdamW over a head's parameters; norms and biases do not decay."""
    decays = [p for p in head.parameters() if p.dim() > 1]
    others = [p for p in head.parameters() if p.dim() <= 1]
    return splatx_torch.AdamW(head.backend, [dict(params=decays, weight_decay=0.01), dict(params=others, weight_decay=0.0)],
                              lr=lr, state_bits=state_bits, max_norm=max_norm)


class View:
    """A camera on a frozen cloud: everything of its images but the colours, formed once."""

    def __init__(self, backend, sc: scene.Scene, viewmat):
        p, n, w, h = sc.params, sc.n, sc.width, sc.height
        self.backend = backend
        opacity = 1.0 / (1.0 + np.exp(-p[3]))
        pr = backend.projection_fused_fwd(means=p[0], quats=p[1], scales=np.exp(p[2]), opacities=opacity, viewmats=viewmat, Ks=sc.K,
                                          width=w, height=h)
        valid = (pr["radii"][0].min(-1) > 0).astype(np.uint8)
        dirs = p[0] - (-(viewmat[:3, :3].T @ viewmat[:3, 3])).astype(np.float32)
        coeffs = np.concatenate([p[4][:, None, :], p[5].reshape(n, -1, 3)], 1)
        self.colors = torch.from_numpy(backend.sh_fwd(dirs, coeffs, sc.sh_degree, masks=valid) + np.float32(0.5)).to(backend.device)
        tw, th = (w + 15) // 16, (h + 15) // 16
        it = backend.isect_tiles(pr["means2d"], pr["radii"], pr["depths"], 1, n, tw, th, conics=pr["conics"], opacities=opacity)
        keys, ids = backend.sort_isect(it["isect_ids"], it["flatten_ids"], 32 + it["tile_n_bits"])
        self.raster = dict(means2d=pr["means2d"], conics=pr["conics"], opacities=opacity, flatten_ids=ids, I=1, N=n, n_isects=ids.size,
                           isect_offsets=backend.isect_offset_encode(keys, 1, tw, th), width=w, height=h, tile_width=tw, tile_height=th)

    def render(self, offset=None):
        """(image [H, W, 3], what the backward needs) with colours offset by a head's output."""
        colors = self.colors if offset is None else self.colors + offset.detach()
        host = colors.clamp_min(0.0).cpu().numpy()
        r = self.backend.rasterize_fwd(colors=host, **self.raster)
        return r["render_colors"][0], (r, host, colors > 0)

    def backward(self, kept, v_image):
        """The gradient of the colours' offset."""
        r, host, positive = kept
        g = self.backend.rasterize_bwd(r["render_alphas"], r["last_ids"], v_image[None], np.zeros_like(r["render_alphas"]), colors=host,
                                       **self.raster)
        return torch.from_numpy(g["v_colors"]).to(self.backend.device) * positive


def train_step(head, opt, features, view, image, target):
    """One image's L1 loss and the head's step for it."""
    offset = head(features, image)
    picture, kept = view.render(offset)
    difference = picture - target
    opt.zero_grad()
    offset.backward(view.backward(kept, np.sign(difference).astype(np.float32) / difference.size))
    opt.step()
    return float(np.abs(difference).mean())


def demo(n=20_000, images=6, steps=120, state_bits=8, seed=0, width=320, height=240, sh_degree=3, quiet=False):
    """A head on a synthetic scene whose images are tinted differently; the losses of the steps."""
    torch.manual_seed(seed)
    backend = splatx_torch.TorchBackend(0)
    sc = scene.make_scene(n=n, sh_degree=sh_degree, width=width, height=height, fx=0.9 * width, seed=seed, gt=None)
    rng = np.random.Generator(np.random.PCG64(seed + 1))
    views = [View(backend, sc, scene.jittered_view(rng)) for _ in range(images)]
    targets = [(v.render()[0] * rng.uniform(0.6, 1.4, 3)).astype(np.float32) for v in views]
    features = torch.from_numpy(np.concatenate([sc.params[4], sc.params[5]], 1)).to(backend.device, torch.bfloat16)
    head = AppearanceHead(backend, features.shape[1], images)
    opt = optimizer(head, state_bits=state_bits)
    losses = []
    for step in range(steps):
        k = step % images
        losses.append(train_step(head, opt, features, views[k], k, targets[k]))
        if not quiet and (step + 1) % images == 0 and (step + 1) % (10 * images) == 0:
            print(f"step {step + 1}: L1 {np.mean(losses[-images:]):.5f}", flush=True)
    backend.close()
    return losses


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--splats", type=int, default=20_000)
    p.add_argument("--images", type=int, default=6)
    p.add_argument("--steps", type=int, default=360)
    p.add_argument("--state-bits", type=int, choices=(8, 32), default=8)
    a = p.parse_args()
    losses = demo(a.splats, a.images, a.steps, a.state_bits)
    first, last = (float(np.mean(x)) for x in (losses[:a.images], losses[-a.images:]))
    print(f"L1 over the images: {first:.5f} before, {last:.5f} after ({20 * math.log10(first / max(last, 1e-9)):.1f} dB)")


if __name__ == "__main__":
    main()
