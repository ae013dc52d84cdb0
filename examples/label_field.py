"""A label field: teach a foam's cells the labels that a 2D teacher sees, then ask them.

The foam is a noisy shell around a sphere, the teacher a function that knows the sphere:
per ray it names its best few of many labels (patches of the surface) with their logits, as
a segmenter or a vision-language model would per pixel.  Each cell has a learned row; a
step traces a batch of rays, takes the rows of the cells that they end in, weighted by the
rays' opacity, makes logits of them, and distils the teacher into rows and head:

    trace_forward -> depth_indices -> cell_rows -> head -> distill_loss -> backward

Afterwards the field answers for an image it was not trained on: each pixel's log
probability of the teacher's best label, the entropy, and its own best labels.

    python examples/label_field.py [--points N] [--labels V] [--steps K] ...
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import sdfoam_amd  # noqa: E402

RADIUS = 0.5


def foam(points, gen):
    """Points of a shell in a box, their adjacency, and attributes whose last channel is the
    sphere's signed distance."""
    dev = torch.device("cuda")
    n = points * 4 // 5
    shell = torch.randn((n, 3), generator=gen, device=dev)
    shell = shell / shell.norm(dim=1, keepdim=True)
    shell = shell * (RADIUS + 0.02 * torch.randn((n, 1), generator=gen, device=dev))
    box = 3.0 * torch.rand((points - n, 3), generator=gen, device=dev) - 1.5
    raw = torch.cat([shell, box])
    tri = sdfoam_amd.Triangulation(raw)
    p = raw[tri.permutation().view(torch.int32).long()].contiguous()
    attributes = torch.zeros((points, 4), device=dev)
    attributes[:, 3] = p.norm(dim=1) - RADIUS
    return p, attributes, tri.point_adjacency(), tri.point_adjacency_offsets()


def camera_rays(k, cameras, size):
    """The rays [size * size, 6] of camera k on a ring around the sphere."""
    dev = torch.device("cuda")
    phi, z = 2.0 * math.pi * k / cameras, 0.8 * math.sin(2.4 * k)
    pos = torch.tensor([math.cos(phi), math.sin(phi), z], device=dev)
    pos = 2.0 * pos / pos.norm()
    forward = -pos / 2.0
    right = torch.linalg.cross(forward, torch.tensor([0.0, 0.0, 1.0], device=dev))
    right = right / right.norm()
    up = torch.linalg.cross(right, forward)
    at = (torch.arange(size, device=dev) + 0.5) / size * 2.0 - 1.0
    v, u = torch.meshgrid(-at, at, indexing="ij")
    d = forward + 0.33 * (u[..., None] * right + v[..., None] * up)
    d = (d / d.norm(dim=-1, keepdim=True)).reshape(-1, 3)
    return torch.cat([pos.expand_as(d), d], dim=1)


class Teacher:
    """Labels are patches around directions spread over the sphere; a ray that meets it
    prefers the patches near the point it meets, one that misses it has no label."""

    def __init__(self, labels, top):
        k = torch.arange(labels, device="cuda") + 0.5
        z, phi = 1.0 - 2.0 * k / labels, k * math.pi * (3.0 - math.sqrt(5.0))
        r = (1.0 - z * z).sqrt()
        self.patches = torch.stack([r * phi.cos(), r * phi.sin(), z])
        self.sharpness = 4.0 * labels / 10.0
        self.top = top

    def __call__(self, rays):
        o, d = rays[:, :3], rays[:, 3:]
        b = (o * d).sum(1)
        root = b * b - (o * o).sum(1) + RADIUS * RADIUS
        hit = o + (-b - root.clamp(min=0.0).sqrt())[:, None] * d
        logits, labels = (self.sharpness * (hit / RADIUS) @ self.patches).topk(self.top, dim=1)
        return torch.where((root > 0.0)[:, None], labels, -1), logits


class LabelField(torch.nn.Module):
    """A learned row per cell and a head that makes logits over labels of it."""

    def __init__(self, scene, labels, features):
        super().__init__()
        self.points, self.attributes, self.adjacency, self.offsets = scene
        self.tree = sdfoam_amd.build_aabb_tree(self.points)
        self.pipeline = sdfoam_amd.create_pipeline(0)
        dev = self.points.device
        self.table = torch.nn.Parameter(0.3 * torch.randn(self.points.shape[0], features, device=dev))
        self.head = torch.nn.Linear(features, labels, device=dev)

    def surface(self, rays):
        """The cell that each ray ends in (uint32, 0xffffffff for none) and its opacity."""
        with torch.no_grad():
            start = sdfoam_amd.get_starting_point(rays, self.points, self.tree)
            half = torch.full((rays.shape[0], 1), 0.5, device=rays.device)
            out = self.pipeline.trace_forward(
                self.points, self.attributes, self.adjacency, self.offsets, rays, start,
                depth_quantiles=half, alpha_mode="sdfoam", inv_s=50.0)
        return out["depth_indices"][:, 0].contiguous(), out["rgba"][:, 3].contiguous()

    def forward(self, rays):
        cells, opacity = self.surface(rays)
        return self.head(sdfoam_amd.cell_rows(self.table, cells, weight=opacity))


def main(points=20_000, labels=512, features=32, top=8, size=128, cameras=8, batch=16_384,
         steps=60, seed=0, log=print):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    field = LabelField(foam(points, gen), labels, features)
    teacher = Teacher(labels, top)
    rays = torch.cat([camera_rays(k, cameras, size) for k in range(cameras)])
    fetcher = sdfoam_amd.BatchFetcher(rays.cpu(), batch, True)
    optimizer = torch.optim.Adam(field.parameters(), lr=0.05)
    losses = []
    for step in range(steps):
        some = fetcher.next()
        loss = sdfoam_amd.distill_loss(field(some), *teacher(some))
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if log and (step % 10 == 0 or step + 1 == steps):
            log(f"step {step}: loss {float(losses[-1]):.4f}")
    # a view between two of the training cameras
    view = camera_rays(0.5, cameras, size)
    best, _ = teacher(view)
    with torch.no_grad():
        answer = sdfoam_amd.label_log_probs(field(view), best[:, 0].contiguous(), top=5)
    seen = best[:, 0] >= 0
    result = {
        "loss": [float(x) for x in losses],
        "log_prob": float(answer.log_prob[seen].mean()),
        "entropy": float(answer.entropy[seen].mean()),
        "first": float((answer.top_labels[seen, 0] == best[seen, 0]).float().mean()),
        "in_five": float((answer.top_labels[seen] == best[seen, :1]).any(1).float().mean()),
    }
    if log:
        log(f"unseen view: log probability of the teacher's best label {result['log_prob']:.3f}, "
            f"entropy {result['entropy']:.3f}; it is the field's best label for "
            f"{100 * result['first']:.1f}% of the pixels and among its best five for "
            f"{100 * result['in_five']:.1f}%")
    return result


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("points", 20_000), ("labels", 512), ("features", 32), ("top", 8),
                        ("size", 128), ("cameras", 8), ("batch", 16_384), ("steps", 60),
                        ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    main(**vars(ap.parse_args()))
