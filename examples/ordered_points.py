"""A small generator of point clouds on the attention operators.

    python examples/ordered_points.py [--steps 60] [--points 256]

Spheres and boxes are sampled to a few hundred points each by farthest point
sampling and ordered along a Morton curve.  A transformer reads them in that
order and predicts each next point's cell of a 16 x 16 x 16 grid: queries and
keys are normed and rotated by the point's three coordinates
(``qk_norm_rotate``), and every point sees a window of the order and the first
two (``window_attention``, with a bias learned by buckets of the offset).  The
trained model then continues a cloud point by point over a cache of keys and
values (``window_attention_step``); fed the same points, the steps give the
whole pass's logits.  ``Layer.weights`` shows what a head attends to, from
ordinary products and the dense bias (``relative_bias``).
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn
from torch.nn import functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "mps-pointops_amd"))

import mps_pointops as mp  # noqa: E402
from mps_pointops import attention  # noqa: E402

GRID = 16
WIDTH, HEADS, KEY_HEADS, HEAD = 128, 4, 2, 32
WINDOW, FIRST, BUCKETS, REACH = 64, 2, 16, 64


def morton(cell: Tensor) -> Tensor:
    """Place of (..., 3) cells of the grid along the curve."""
    code = torch.zeros_like(cell[..., 0])
    for bit in range(4):
        for axis in range(3):
            code |= ((cell[..., axis] >> bit) & 1) << (3 * bit + axis)
    return code


def clouds(batch: int, points: int, seed: int) -> Tensor:
    """Spheres and boxes of random size and place in the unit cube, ordered:
    (batch, points) cells as one number each."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    raw = torch.randn(batch, 8 * points, 3, generator=gen, device="cuda")
    sphere = raw / raw.norm(dim=-1, keepdim=True)
    box = raw / raw.abs().amax(-1, keepdim=True)
    shape = torch.where(torch.rand(batch, 1, 1, generator=gen, device="cuda") < 0.5, sphere, box)
    size = 0.2 + 0.25 * torch.rand(batch, 1, 3, generator=gen, device="cuda")
    xyz = 0.5 + size * shape
    chosen = mp.furthest_point_sample(xyz, points)
    xyz = torch.gather(xyz, 1, chosen[..., None].expand(-1, -1, 3))
    cell = (xyz * GRID).long().clamp(0, GRID - 1)
    order = morton(cell).argsort(1)
    cell = torch.gather(cell, 1, order[..., None].expand(-1, -1, 3))
    return (cell[..., 0] * GRID + cell[..., 1]) * GRID + cell[..., 2]


def place(token: Tensor) -> Tensor:
    """Centres of (...) cells, in grid units."""
    return torch.stack([token // (GRID * GRID), token // GRID % GRID, token % GRID], -1).float() + 0.5


def angles(xyz: Tensor) -> tuple[Tensor, Tensor]:
    """cos and sin for (batch, tokens, 3) places: five frequencies an axis."""
    frequency = 4.0 ** -torch.arange(5, device=xyz.device)
    angle = (xyz[..., None] * frequency).flatten(-2)
    return angle.cos(), angle.sin()


class Layer(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm1, self.norm2 = nn.LayerNorm(WIDTH), nn.LayerNorm(WIDTH)
        self.qkv = nn.Linear(WIDTH, (HEADS + 2 * KEY_HEADS) * HEAD, bias=False)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(HEAD)), nn.Parameter(torch.ones(HEAD))
        self.bias = nn.Parameter(torch.zeros(BUCKETS, HEADS))
        self.out = nn.Linear(HEADS * HEAD, WIDTH, bias=False)
        self.mlp = nn.Sequential(nn.Linear(WIDTH, 2 * WIDTH), nn.GELU(), nn.Linear(2 * WIDTH, WIDTH))

    def heads(self, x: Tensor, cos: Tensor, sin: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        packed = self.qkv(self.norm1(x)).unflatten(-1, (HEADS + 2 * KEY_HEADS, HEAD))
        q, k, v = packed.split((HEADS, KEY_HEADS, KEY_HEADS), 2)
        return *attention.qk_norm_rotate(q, k, self.q_weight, self.k_weight, cos, sin), v

    def rest(self, x: Tensor, seen: Tensor) -> Tensor:
        x = x + self.out(seen.flatten(2))
        return x + self.mlp(self.norm2(x))

    def forward(self, x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
        q, k, v = self.heads(x, cos, sin)
        return self.rest(x, attention.window_attention(q, k, v, window=WINDOW, sinks=FIRST, causal=True,
                                                       bias=self.bias, max_distance=REACH))

    def step(self, x: Tensor, cos: Tensor, sin: Tensor, keys: Tensor, values: Tensor, at: int) -> Tensor:
        """One token for each cloud, its key and value written to the cache."""
        q, k, v = self.heads(x, cos, sin)
        keys[:, at:at + 1], values[:, at:at + 1] = k, v
        lengths = torch.full((len(x),), at + 1, dtype=torch.int32, device=x.device)
        return self.rest(x, attention.window_attention_step(q, keys, values, lengths, window=WINDOW, sinks=FIRST,
                                                            bias=self.bias, max_distance=REACH))

    def weights(self, x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
        """(batch, heads, tokens, tokens) weights, for inspection."""
        q, k, _ = self.heads(x, cos, sin)
        n = q.shape[1]
        k = k.repeat_interleave(HEADS // KEY_HEADS, 2).permute(0, 2, 3, 1).contiguous()
        score = q.transpose(1, 2).contiguous() @ k * HEAD ** -0.5
        score = score + attention.relative_bias(self.bias, n, n, max_distance=REACH, causal=True)
        i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)
        return score.masked_fill((j > i) | (i - j >= WINDOW) & (j >= FIRST), -torch.inf).softmax(-1)


class Generator(nn.Module):
    def __init__(self, layers: int = 2):
        super().__init__()
        self.token = nn.Embedding(GRID ** 3, WIDTH)
        self.layers = nn.ModuleList(Layer() for _ in range(layers))
        self.head = nn.Sequential(nn.LayerNorm(WIDTH), nn.Linear(WIDTH, GRID ** 3))

    def forward(self, token: Tensor) -> Tensor:
        x, turn = self.token(token), angles(place(token))
        for layer in self.layers:
            x = layer(x, *turn)
        return self.head(x)

    def cache(self, batch: int, tokens: int) -> list[tuple[Tensor, Tensor]]:
        like = self.token.weight
        return [(like.new_zeros(batch, tokens, KEY_HEADS, HEAD), like.new_zeros(batch, tokens, KEY_HEADS, HEAD))
                for _ in self.layers]

    @torch.no_grad()
    def step(self, token: Tensor, cache: list[tuple[Tensor, Tensor]], at: int) -> Tensor:
        """Logits after the (batch, 1) tokens at place `at` of the cache."""
        x, turn = self.token(token), angles(place(token))
        for layer, (keys, values) in zip(self.layers, cache):
            x = layer.step(x, *turn, keys, values, at)
        return self.head(x)


def train(model: Generator, steps: int, points: int, batch: int = 16) -> list[float]:
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3)
    losses = []
    for n in range(steps):
        token = clouds(batch, points, n)
        loss = F.cross_entropy(model(token[:, :-1]).flatten(0, 1), token[:, 1:].flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(x) for x in torch.stack(losses).tolist()]


@torch.no_grad()
def replay(model: Generator, token: Tensor) -> Tensor:
    """The whole pass's logits, step by step."""
    cache = model.cache(*token.shape)
    return torch.cat([model.step(token[:, n:n + 1], cache, n) for n in range(token.shape[1])], 1)


@torch.no_grad()
def generate(model: Generator, start: Tensor, points: int) -> Tensor:
    """The start continued with the likeliest next cells."""
    cache = model.cache(len(start), points)
    token = start
    for n in range(points):
        logits = model.step(token[:, n:n + 1], cache, n)
        if n + 1 == token.shape[1] and n + 1 < points:
            token = torch.cat([token, logits[:, -1:].argmax(-1)], 1)
    return token


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--points", type=int, default=256)
    args = parser.parse_args()
    torch.manual_seed(0)
    model = Generator().cuda()
    losses = train(model, args.steps, args.points)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {args.steps} steps")
    token = clouds(4, args.points, 10 ** 6)
    with torch.no_grad():
        whole, single = model(token), replay(model, token)
    print(f"whole pass and single steps differ by {(whole - single).norm() / whole.norm():.1e}")
    made = generate(model, token[:, :args.points // 2], args.points)
    kept = (made[:, 1:] != made[:, :-1]).float().mean()
    print(f"continued {tuple(made.shape)} cells; {100 * kept:.0f}% of them move on")


if __name__ == "__main__":
    main()
