"""qk_norm_rotate against its definition in 64 bits, with gradients.

Tolerances, as the 2-norm of the difference over that of the result, u being
half the spacing of the type's values at 1: a 16-bit result carries one
rounding (u at most); a float32 one those of a sum of up to 128 terms in a tree
and of about ten operations, below 16 u.  A weight's gradient is a sum over all
rows: the same of the sum of its terms' magnitudes.  Values below float16's
normal range are spaced evenly (2^-24): half of that for each of them besides."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 16 * 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def definition(x, w, cos, sin, eps, g):
    x, cos, sin, g = (t.detach().cpu().double() for t in (x, cos, sin, g))
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.detach().cpu().double()
    cos, sin = (t.expand(x.shape[0], *t.shape[-2:])[:, :, None] for t in (cos, sin))
    R = 2 * cos.shape[-1]
    unit = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    y = unit * w
    a, b = y[..., :R // 2], y[..., R // 2:R]
    out = torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., R:]], -1)
    a, b = g[..., :R // 2], g[..., R // 2:R]
    dy = torch.cat([a * cos + b * sin, b * cos - a * sin, g[..., R:]], -1)
    dw = (dy * unit).sum((0, 1, 2))
    size = (dy * unit).abs().sum((0, 1, 2))
    along = (dy * w * unit).mean(-1, keepdim=True)
    dx = (dy * w - unit * along) / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return out, dx, dw, size


def close(got, want, size=None):
    got_cpu = got.detach().cpu().double()
    assert got_cpu.shape == want.shape and torch.isfinite(got_cpu).all()
    norm = (want if size is None else size).norm()
    least = 2.0 ** -25 * want.numel() ** 0.5 if got.dtype == torch.float16 else 0.0
    assert (got_cpu - want).norm() <= UNIT[got.dtype] * norm + least, ((got_cpu - want).norm() / norm).item()


def check(q, k, wq, wk, cos, sin, gq, gk, eps=1e-6):
    from mps_pointops.attention import qk_norm_rotate

    print(q.dtype, tuple(q.shape), tuple(k.shape), 2 * cos.shape[-1], flush=True)
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, wq, wk)]
    outs = qk_norm_rotate(*leaves, cos, sin, eps=eps)
    there = [t for t in leaves if t is not None]
    got = dict(zip([n for n, t in enumerate(leaves) if t is not None], torch.autograd.grad(outs, there, (gq, gk))))
    again = torch.autograd.grad(qk_norm_rotate(*leaves, cos, sin, eps=eps), there, (gq, gk))
    assert all(torch.equal(x, y) for x, y in zip(got.values(), again))
    for n, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        out, dx, dw, size = definition(x, w, cos, sin, eps, g)
        assert outs[n].dtype == x.dtype and got[n].dtype == x.dtype
        close(outs[n], out)
        close(got[n], dx)
        if w is not None:
            assert got[2 + n].dtype == w.dtype
            close(got[2 + n], dw, size)


def make(seed, B, N, H, G, D, R, dtype, weight):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    angle = 10 * new(B, N, R // 2)
    return (new(B, N, H, D).to(dtype), new(B, N, G, D).to(dtype), (1 + 0.2 * new(D)).to(weight),
            (1 + 0.2 * new(D)).to(weight), angle.cos(), angle.sin(), new(B, N, H, D).to(dtype), new(B, N, G, D).to(dtype))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("B,N,H,G,D,R", [
    (1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 2, 2), (2, 7, 3, 1, 33, 32), (2, 65, 4, 2, 64, 64), (3, 50, 12, 3, 80, 60),
    (1, 1000, 8, 8, 128, 128), (1, 333, 2, 2, 128, 112), (2, 40, 5, 5, 24, 0), (1, 129, 1, 1, 127, 126),
    (1, 31, 7, 7, 96, 48), (1, 17, 40, 4, 20, 12), (1, 5000, 2, 1, 16, 6),
])
def test_norm(cuda_device, kind, B, N, H, G, D, R):
    dtype = TYPES[kind]
    check(*make(1, B, N, H, G, D, R, dtype, torch.float32))
    q, k, wq, wk, cos, sin, gq, gk = make(2, B, N, H, G, D, R, dtype, dtype)
    check(q, k, wq, wk, cos[0], sin[0], gq, gk)
    check(q, k, None, None, cos, sin, gq, gk)
    check(q, k, wq, None, cos, sin, gq, gk, eps=0.5)


@pytest.mark.parametrize("kind", TYPES)
def test_strides(cuda_device, kind):
    """Views of a packed projection, swapped dimensions, unaligned rows and
    angles, gradients that are one value."""
    from mps_pointops.attention import qk_norm_rotate

    gen = torch.Generator(device="cuda").manual_seed(3)
    _, _, wq, wk, cos, sin, gq, gk = make(4, 2, 45, 4, 2, 64, 48, TYPES[kind], torch.float32)
    flat = torch.randn(2 * 45 * 8 * 64 + 1, generator=gen, device="cuda").to(TYPES[kind])
    for packed in (flat[:-1].view(2, 45, 8, 64), flat[1:].view(2, 45, 8, 64)):
        check(packed[:, :, :4], packed[:, :, 4:6], wq, wk, cos, sin, gq, gk)
        turned = packed.transpose(1, 2).contiguous().transpose(1, 2)
        check(turned[:, :, :4], turned[:, :, 4:6], wq, wk, cos, sin, gq, gk)
        last = packed.transpose(2, 3).contiguous().transpose(2, 3)
        check(last[:, :, :4], last[:, :, 4:6], wq, wk, cos, sin, gq, gk)
    wide = torch.cat([cos[..., :1], cos], -1)
    check(packed[:, :, :4], packed[:, :, 4:6], wq, wk, wide[..., 1:], torch.cat([sin[..., :1], sin], -1)[..., 1:], gq, gk)
    check(packed[:, :, :4], packed[:, :, 4:6], wq[:1].expand(64), wk, cos, sin, gq, gk)
    shared = packed[:1].expand(2, -1, -1, -1)
    check(shared[:, :, :4], shared[:, :, 4:6], wq, wk, cos, sin, gq[:, :1].expand(-1, 45, -1, -1), gk)
    q = packed[:, :, :4].clone().requires_grad_()
    a, b = qk_norm_rotate(q, packed[:, :, 4:6], wq, wk, cos, sin)
    only, = torch.autograd.grad(a.float().sum() + 0 * b.float().sum(), [q])
    both = torch.autograd.grad(qk_norm_rotate(q, packed[:, :, 4:6], wq, wk, cos, sin)[0], [q], torch.ones_like(q))[0]
    assert torch.equal(only, both)


def test_rows_of_zeros_and_one_bad_row(cuda_device):
    """A row of zeros is zeros; a NaN stays in its row."""
    from mps_pointops.attention import qk_norm_rotate

    q, k, wq, wk, cos, sin, gq, gk = make(5, 1, 20, 3, 3, 32, 32, torch.float32, torch.float32)
    q[0, 3, 1] = 0
    k[0, 5, 2, 7] = float("nan")
    a, b = qk_norm_rotate(q, k, wq, wk, cos, sin)
    assert (a[0, 3, 1] == 0).all() and torch.isfinite(a).all()
    bad = ~torch.isfinite(b).all(-1)
    assert bad.nonzero().tolist() == [[0, 5, 2]]


def test_gradient_against_differences(cuda_device):
    """Central differences of a weighted sum of the 32-bit outputs."""
    from mps_pointops.attention import qk_norm_rotate

    q, k, wq, wk, cos, sin, gq, gk = make(6, 1, 9, 2, 1, 16, 12, torch.float32, torch.float32)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(qk_norm_rotate(*leaves, cos, sin), leaves, (gq, gk))
    gen = torch.Generator(device="cuda").manual_seed(7)
    for leaf, grad in zip(leaves, grads):
        way = torch.randn(leaf.shape, generator=gen, device="cuda")
        way /= way.norm()
        value = []
        for sign in (1, -1):
            a, b = qk_norm_rotate(*[t.detach() + (sign * 2.0 ** -6 * way if t is leaf else 0) for t in leaves], cos, sin)
            value.append(((a.double() * gq).sum() + (b.double() * gk).sum()).item())
        slope, along = (value[0] - value[1]) * 2.0 ** 5, (grad.double() * way).sum().item()
        assert abs(slope - along) <= 2e-3 * grad.norm().item()


def test_empty(cuda_device):
    from mps_pointops.attention import qk_norm_rotate

    w = torch.ones(8, device="cuda", requires_grad=True)
    angle = torch.ones(0, 4, device="cuda")
    q = torch.ones(2, 0, 3, 8, device="cuda", requires_grad=True)
    a, b = qk_norm_rotate(q, q, w, w, angle, angle)
    assert a.shape == b.shape == q.shape
    dq, dw = torch.autograd.grad(a.sum() + b.sum(), (q, w))
    assert dq.shape == q.shape and (dw == 0).all()
