"""Workloads of the attention operators, each beside its plain form.

A transformer over clouds whose points are ordered along a curve asks for four
operators: the norm of each head's query and key with the rotation by the
token's position (``norm``), attention within a window of the order with a few
first tokens that every query sees (``attn``), the same for one or a few new
tokens over a cache (``step``), and the bias that is learned by buckets of the
offset in the order, as a dense tensor (``bias``; within attention it is an
argument).  ``run`` computes them by elementary tensor operations in 32 bits,
rounded once at the end, or, where ``own`` is true, by the package's calls.

Shapes: q (B, Q, H, D) and k, v (B, N, G, D), query head h with key head
h // (H // G); the queries are the last Q of the N positions.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
_attention = None


def _package():
    """The package's operators, imported with the first call."""
    global _attention
    if _attention is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mps-pointops_amd"))
        from mps_pointops import attention
        _attention = attention
    return _attention


def listed():
    return [
        # One new token for each of 16 sequences that are being written: its
        # queries' and keys' norm and rotation, where the call's latency counts.
        {"name": "norm_step", "kind": "norm", "type": "bf16", "B": 16, "N": 1, "H": 16, "G": 4,
         "D": 128, "R": 128, "train": False},
        # Training on the benchmark's batch of clouds (32 of 4096 points) in
        # float32, rotated by 3 coordinates of 4 frequencies each.
        {"name": "norm_train", "kind": "norm", "type": "f32", "B": 32, "N": 4096, "H": 4, "G": 4,
         "D": 32, "R": 24, "train": True},
        # Training on one long cloud of odd length, shared key heads.
        {"name": "norm_long", "kind": "norm", "type": "f16", "B": 1, "N": 65537, "H": 12, "G": 3,
         "D": 80, "R": 60, "train": True},
        # A small classifier's layer in float32: 1024 points a cloud, each
        # seeing its neighbours on both sides, with the learned bias.
        {"name": "attn_small", "kind": "attn", "type": "f32", "B": 8, "Q": 1024, "N": 1024, "H": 4,
         "G": 4, "D": 32, "window": 128, "sinks": 0, "causal": False, "buckets": 32, "reach": 128,
         "ragged": False, "train": True},
        # Training a generator of ordered points: causal, first tokens kept
        # visible, two key heads for eight, with the learned bias.
        {"name": "attn_train", "kind": "attn", "type": "bf16", "B": 4, "Q": 4096, "N": 4096, "H": 8,
         "G": 2, "D": 64, "window": 512, "sinks": 4, "causal": True, "buckets": 32, "reach": 128,
         "ragged": False, "train": True},
        # Training on padded clouds of unequal size, one of them empty and one
        # of a single point; odd sizes throughout.
        {"name": "attn_ragged", "kind": "attn", "type": "f16", "B": 13, "Q": 1001, "N": 1001, "H": 6,
         "G": 3, "D": 40, "window": 201, "sinks": 3, "causal": False, "buckets": 0, "reach": 0,
         "ragged": True, "train": True},
        # Training with every earlier token visible.
        {"name": "attn_full", "kind": "attn", "type": "bf16", "B": 2, "Q": 4096, "N": 4096, "H": 8,
         "G": 8, "D": 128, "window": 0, "sinks": 0, "causal": True, "buckets": 0, "reach": 0,
         "ragged": False, "train": True},
        # Reading a long prompt: forward only, a wide window and first tokens.
        {"name": "attn_long", "kind": "attn", "type": "bf16", "B": 1, "Q": 16384, "N": 16384, "H": 8,
         "G": 2, "D": 128, "window": 2048, "sinks": 16, "causal": True, "buckets": 0, "reach": 0,
         "ragged": False, "train": False},
        # Writing the next token of four short sequences.
        {"name": "step_small", "kind": "step", "type": "bf16", "B": 4, "Q": 1, "N": 2048, "H": 8,
         "G": 2, "D": 64, "window": 512, "sinks": 4, "buckets": 32, "reach": 128},
        # The next token of four long sequences, the whole cache visible.
        {"name": "step_long", "kind": "step", "type": "bf16", "B": 4, "Q": 1, "N": 65536, "H": 32,
         "G": 8, "D": 128, "window": 0, "sinks": 0, "buckets": 0, "reach": 0},
        # The bias by itself for a layer that adds it to its own scores.
        {"name": "bias_train", "kind": "bias", "type": "f32", "Q": 2048, "N": 2048, "H": 16,
         "causal": False, "buckets": 32, "reach": 128},
        # A small one of odd sizes: a chunk of queries at the end of its keys.
        {"name": "bias_odd", "kind": "bias", "type": "bf16", "Q": 333, "N": 1001, "H": 6,
         "causal": True, "buckets": 20, "reach": 500},
    ]


def _size(rng, low, high):
    """A whole number of the range, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(("norm", "attn", "attn", "step", "bias"))
    case = {"kind": kind, "type": rng.choice(("f32", "f16", "bf16"))}
    D = rng.choice((16, 20, 24, 32, 40, 48, 64, 80, 96, 128))
    G = rng.choice((1, 2, 3, 4, 8))
    H = G * rng.choice((1, 1, 2, 3, 4))
    reach = _size(rng, 32, 1024)
    if kind == "norm":
        tokens = _size(rng, 1, (1 << 23) // ((H + G) * D))
        B = _size(rng, 1, min(64, tokens))
        return {**case, "B": B, "N": max(1, tokens // B), "H": H, "G": G, "D": D,
                "R": rng.choice((D, D // 2, 2 * (D // 3), 8)), "train": rng.random() < 0.7}
    if kind == "bias":
        Q = _size(rng, 1, 2048)
        causal = rng.random() < 0.5
        return {**case, "Q": Q, "N": max(Q, _size(rng, 64, 4096)), "H": min(H, 8), "causal": causal,
                "buckets": rng.choice((8, 16, 32, 50)), "reach": max(reach, 64)}
    bias = rng.random() < 0.5
    seen = {"window": rng.choice((0, _size(rng, 2, 2048))), "sinks": rng.choice((0, 0, 1, 4, 70)),
            "buckets": rng.choice((8, 16, 32)) if bias else 0, "reach": reach if bias else 0}
    if kind == "step":
        N = _size(rng, 16, 65536)
        B = _size(rng, 1, max(1, min(32, (1 << 26) // (N * G * D))))
        return {**case, "B": B, "Q": rng.choice((1, 1, 2, 5)), "N": N, "H": H, "G": G, "D": D, **seen}
    N = _size(rng, 1, int(math.sqrt(130_000_000 / H)))
    B = _size(rng, 1, max(1, min(32, 130_000_000 // (N * N * H))))
    chunk = rng.random() < 0.25
    causal = chunk or rng.random() < 0.5
    return {**case, "B": B, "Q": max(1, N // rng.choice((2, 3, 7))) if chunk else N, "N": N, "H": H, "G": G,
            "D": D, **seen, "causal": causal, "ragged": rng.random() < 0.3,
            "train": N >= 8 and rng.random() < 0.7}


# ------------------------------------------------------------------ buckets
def _edges(count, reach):
    """Smallest distance of each bucket but the first of one side: single
    distances to count // 2, then even steps of the logarithm to ``reach``."""
    single = count // 2
    edges = list(range(1, single + 1))
    d = single
    for t in range(1, count - single):
        while d ** (count - single) < reach ** t * single ** (count - single - t):
            d += 1
        edges.append(d)
    return edges


def _bucket_list(case):
    """The bucket of every offset from -limit to limit, and the limit, beyond
    which the bucket no longer changes."""
    count = case["buckets"]
    side = count if case.get("causal", True) else count // 2
    edges = _edges(side, case["reach"])
    limit = max(edges)
    past = [sum(e <= d for e in edges) for d in range(limit + 1)]
    future = [0] * (limit + 1) if side == count else [side + b for b in past]
    return future[:0:-1] + past, limit


def _lengths(case):
    """The clouds' lengths: a whole one, an empty one, one point, then any; or
    a cache's, each more than half full."""
    B, N = case["B"], case["N"]
    parts = [(b * 0.6180339887) % 1.0 for b in range(B)]
    if case["kind"] == "step":
        return [N if b == 0 else max(1, N - int(parts[b] * N / 2)) for b in range(B)]
    return [(N, 0, 1)[b] if b < 3 else int(round(parts[b] * N)) for b in range(B)]


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(scale).add_(shift).to(dtype)

    state = {"case": case}
    if case["kind"] == "norm":
        B, N, H, G, D, R = (case[x] for x in ("B", "N", "H", "G", "D", "R"))
        packed = normal(B, N, H + 2 * G, D)  # one projection's output: queries, keys and values
        state["q"], state["k"] = packed[:, :, :H], packed[:, :, H:H + G]
        state["wq"] = normal(D, scale=0.1, shift=1.0, dtype=torch.float32)
        state["wk"] = normal(D, scale=0.1, shift=1.0, dtype=torch.float32)
        place = torch.rand(B, N, 3, generator=gen, device=DEVICE) * 64.0
        which = torch.arange(R // 2, device=DEVICE)
        angle = place[:, :, which % 3] * 10.0 ** (-2.0 * (which // 3) / max(1, R // 6))
        state["cos"], state["sin"] = angle.cos(), angle.sin()
        if case["train"]:
            state["gq"], state["gk"] = normal(B, N, H, D), normal(B, N, G, D)
            for x in ("q", "k", "wq", "wk"):
                state[x].requires_grad_()
        return state
    if case["buckets"]:
        state["table"] = normal(case["buckets"], case["H"], scale=0.5)
        buckets, state["limit"] = _bucket_list(case)
        state["buckets"] = torch.tensor(buckets, device=DEVICE)
    if case["kind"] == "bias":
        state["grad"] = normal(case["H"], case["Q"], case["N"])
        state["table"].requires_grad_()
        return state
    B, Q, N, H, G, D = (case[x] for x in ("B", "Q", "N", "H", "G", "D"))
    if case["kind"] == "step" or Q != N:
        state["q"], state["k"], state["v"] = normal(B, Q, H, D), normal(B, N, G, D), normal(B, N, G, D)
    else:
        packed = normal(B, N, H + 2 * G, D)
        state["q"], state["k"], state["v"] = packed[:, :, :H], packed[:, :, H:H + G], packed[:, :, H + G:]
    if case["kind"] == "step" or case["ragged"]:
        state["lengths"] = torch.tensor(_lengths(case), device=DEVICE)
    if case.get("train"):
        state["grad"] = normal(B, Q, H, D)
        for x in ("q", "k", "v", "table"):
            if x in state:
                state[x].requires_grad_()
    return state


# ---------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "attn": _own_attn, "step": _own_step, "bias": _own_bias}[kind](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "attn": _plain_attn, "step": _plain_attn, "bias": _plain_bias}[kind](state)


def _own_norm(s):
    args = s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"]
    q, k = _package().qk_norm_rotate(*args, eps=EPS)
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    grads = torch.autograd.grad((q, k), args[:4], (s["gq"], s["gk"]))
    return {"q": q, "k": k, **dict(zip(("dq", "dk", "dwq", "dwk"), grads))}


def _own_attn(s):
    case = s["case"]
    out = _package().window_attention(
        s["q"], s["k"], s["v"], window=case["window"] or None, sinks=case["sinks"], causal=case["causal"],
        bias=s.get("table"), max_distance=case["reach"] or None, lengths=s.get("lengths"))
    if not case["train"]:
        return {"out": out}
    names = [x for x in ("q", "k", "v", "table") if x in s]
    grads = torch.autograd.grad(out, [s[x] for x in names], s["grad"])
    return {"out": out, **{"d" + x: g for x, g in zip(names, grads)}}


def _own_step(s):
    case = s["case"]
    return {"out": _package().window_attention_step(
        s["q"], s["k"], s["v"], s["lengths"], window=case["window"] or None, sinks=case["sinks"],
        bias=s.get("table"), max_distance=case["reach"] or None)}


def _own_bias(s):
    case = s["case"]
    out = _package().relative_bias(s["table"], case["Q"], case["N"], max_distance=case["reach"],
                                   causal=case["causal"])
    grad, = torch.autograd.grad(out, [s["table"]], s["grad"])
    return {"out": out, "dtable": grad}


def _plain_norm(s):
    case = s["case"]
    half = case["R"] // 2
    cos, sin = s["cos"][:, :, None], s["sin"][:, :, None]

    def turn(x, sin):
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)

    out = {}
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        value, weight = s[x].float(), s[w].float()
        inverse = torch.rsqrt((value * value).mean(-1, keepdim=True) + EPS)
        unit = value * inverse
        out[x] = turn(unit * weight, sin).to(s[x].dtype)
        if case["train"]:
            back = turn(s[g].float(), -sin)
            out["d" + w] = (back * unit).sum((0, 1, 2)).to(s[w].dtype)
            back = back * weight
            out["d" + x] = (inverse * (back - unit * (back * unit).mean(-1, keepdim=True))).to(s[x].dtype)
    return out


def _offset_bias(s, Q, N):
    """(H, Q, N) of the offsets (query's place less key's), from one row of
    the offsets from -(N - 1) to N - 1 that each query reads one place on."""
    limit = s["limit"]
    row = s["buckets"][torch.arange(N - 1, -N, -1, device=DEVICE).clamp(-limit, limit) + limit]
    row = s["table"].float()[row].t().contiguous()  # (H, 2N - 1), falling offsets
    place = torch.arange(N - Q, N, device=DEVICE)[:, None]
    return row[:, (N - 1) - place + torch.arange(N, device=DEVICE)]


def _offset_sums(s, g):
    """The table's gradient from that of the (H, Q, N) bias: the diagonals'
    sums, then the buckets'.  Rows padded to N + Q and cut anew at one more
    bring each diagonal (key less query row = c, or c - N - Q - 1) into one
    column c."""
    H, Q, N = g.shape
    wide = torch.zeros(H, Q * (N + Q + 1), device=DEVICE)
    wide[:, :Q * (N + Q)].view(H, Q, N + Q)[:, :, :N] = g
    sums = wide.view(H, Q, N + Q + 1).sum(1)
    c = torch.arange(N + Q + 1, device=DEVICE)
    offset = (N - Q) - torch.where(c < N, c, c - (N + Q + 1))
    limit = s["limit"]
    bucket = s["buckets"][offset.clamp(-limit, limit) + limit]
    grad = torch.zeros(s["table"].shape, device=DEVICE)
    return grad.index_add_(0, bucket, sums.t()).to(s["table"].dtype)


def _plain_bias(s):
    case = s["case"]
    out = _offset_bias(s, case["Q"], case["N"]).to(s["table"].dtype)
    return {"out": out, "dtable": _offset_sums(s, s["grad"].float())}


def _seen(s):
    """Which keys each query sees: (Q, N), or (B, 1, Q, N) with lengths."""
    case = s["case"]
    Q, N = case["Q"], case["N"]
    key = torch.arange(N, device=DEVICE)
    place = torch.arange(N - Q, N, device=DEVICE)[:, None]
    if case["kind"] == "step":
        length = s["lengths"][:, None, None, None]
        place = place - N + length
    causal = case.get("causal", True)
    seen = torch.ones(1, 1, dtype=torch.bool, device=DEVICE)
    if case["window"]:
        seen = (key > place - case["window"]) & (key < place + case["window"]) | (key < case["sinks"])
    if causal:
        seen = seen & (key <= place)
    if "lengths" in s:
        length = s["lengths"][:, None, None, None]
        seen = seen & (key < length) & (place < length) & (place >= 0)
    return seen


def _plain_attn(s):
    case = s["case"]
    B, Q, N, H, G, D = (case[x] for x in ("B", "Q", "N", "H", "G", "D"))
    scale = D ** -0.5
    q = s["q"].float().reshape(B, Q, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    k, v = (s[x].float().transpose(1, 2).contiguous() for x in ("k", "v"))
    q = q * scale
    p = (q @ k.transpose(2, 3)).reshape(B, H, Q, N)
    if "table" in s:
        if case["kind"] == "step":
            place = s["lengths"][:, None, None] - Q + torch.arange(Q, device=DEVICE)[:, None]
            offset = (place - torch.arange(N, device=DEVICE)).clamp(-s["limit"], s["limit"]) + s["limit"]
            p += s["table"].float()[s["buckets"][offset]].permute(0, 3, 1, 2)
        else:
            p += _offset_bias(s, Q, N)
    seen = _seen(s)
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0)).reshape(B, G, -1, N)

    def whole(x):  # (B, G, rows, D) back to (B, Q, H, D)
        return x.reshape(B, G, H // G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, H, D)

    o = p @ v
    out = {"out": whole(o).to(s["q"].dtype)}
    if not case.get("train"):
        return out
    g = s["grad"].float().reshape(B, Q, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    dv = p.transpose(2, 3) @ g
    ds = (g @ v.transpose(2, 3)).sub_((g * o).sum(-1, keepdim=True)).mul_(p)
    out["dq"] = whole(ds @ k).mul_(scale).to(s["q"].dtype)
    out["dk"] = (ds.transpose(2, 3) @ q).transpose(1, 2).to(s["k"].dtype)
    out["dv"] = dv.transpose(1, 2).to(s["v"].dtype)
    if "table" in s:
        out["dtable"] = _offset_sums(s, ds.reshape(B, H, Q, N).sum(0))
    return out


# --------------------------------------------------------------------- work
def _pairs(case):
    """Query-key pairs that are seen, of one head over all clouds."""
    Q, N, total = case["Q"], case["N"], 0
    step = case["kind"] == "step"
    lengths = _lengths(case) if step or case["ragged"] else [N] * case["B"]
    causal, sinks = case.get("causal", True), case["sinks"]
    window = case["window"] or N + 1
    for length in lengths:
        first = length - Q if step else N - Q
        for place in range(max(0, first), min(first + Q, length)):
            low = max(0, place - window + 1)
            high = min(length, place + 1 if causal else place + window)
            more = min(sinks, place + 1 if causal else length)
            total += high - low + min(more, low) + max(0, more - high)
    return total


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "norm":
        values = case["B"] * case["N"] * (case["H"] + case["G"]) * case["D"]
        tables = case["B"] * case["N"] * case["R"] * 4
        if case["train"]:
            return {"bytes": 4 * values * size + tables, "flops": 20 * values}
        return {"bytes": 2 * values * size + tables, "flops": 6 * values}
    if case["kind"] == "bias":
        values = case["H"] * case["Q"] * case["N"]
        return {"bytes": 2 * values * size, "flops": values}
    B, Q, N, H, G, D = (case[x] for x in ("B", "Q", "N", "H", "G", "D"))
    pairs = _pairs(case) * H
    rows, keys = B * Q * H * D, B * N * G * D
    if case["kind"] == "step":
        window = min(N, (case["window"] + case["sinks"] + Q - 1) if case["window"] else N)
        keys = sum(min(window, length) for length in _lengths(case)) * G * D
    if case.get("train"):
        return {"bytes": (4 * rows + 4 * keys) * size, "flops": 14 * pairs * D}
    return {"bytes": (2 * rows + 2 * keys) * size, "flops": 4 * pairs * D}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, one head of one cloud at a time."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "bias": _exact_bias}.get(case["kind"], _exact_attn)(s, case)


def _exact_norm(s, case):
    half, out = case["R"] // 2, {}
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        value, weight = s[x].double(), s[w].double()
        heads = value.shape[2]
        D = value.shape[3]
        root = ((value ** 2).sum(-1) / D + EPS).sqrt()
        y = value / root[..., None] * weight
        # The rotation as a complex product.
        turn = torch.complex(s["cos"].double(), s["sin"].double())[:, :, None]
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
        out[x] = torch.cat((z.real, z.imag, y[..., 2 * half:]), -1)
        if not case["train"]:
            continue
        grad = s[g].double()
        z = torch.complex(grad[..., :half], grad[..., half:2 * half]) * turn.conj()
        dy = torch.cat((z.real, z.imag, grad[..., 2 * half:]), -1)
        out["d" + w] = torch.stack([(dy[:, :, h] * value[:, :, h] / root[:, :, h, None]).sum((0, 1))
                                    for h in range(heads)]).sum(0)
        dx = dy * weight / root[..., None]
        along = (dy * weight * value).sum(-1) / (D * root ** 3)
        out["d" + x] = dx - value * along[..., None]
    names = ("q", "k", "dq", "dk", "dwq", "dwk") if case["train"] else ("q", "k")
    return {n: out[n] for n in names}


def _exact_buckets(case, offset):
    """The bucket of each offset, by counting the edges that it reaches."""
    count = case["buckets"]
    side = count if case.get("causal", True) else count // 2
    bucket = torch.zeros_like(offset)
    away = offset.clamp(min=0) if side == count else offset.abs()
    for e in _edges(side, case["reach"]):
        bucket += away >= e
    return bucket if side == count else bucket + side * (offset < 0)


def _exact_bias(s, case):
    Q, N = case["Q"], case["N"]
    offset = torch.arange(N - Q, N, device=DEVICE)[:, None] - torch.arange(N, device=DEVICE)
    bucket = _exact_buckets(case, offset)
    table, grad = s["table"].double(), s["grad"].double()
    out = torch.stack([table[:, h][bucket] for h in range(case["H"])])
    dtable = torch.stack([(grad * (bucket == b)).sum((1, 2)) for b in range(case["buckets"])])
    return {"out": out, "dtable": dtable}


def _exact_attn(s, case):
    B, Q, N, H, G, D = (case[x] for x in ("B", "Q", "N", "H", "G", "D"))
    train = case.get("train", False)
    step = case["kind"] == "step"
    lengths = _lengths(case) if step or case["ragged"] else [N] * B
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=DEVICE)  # noqa: E731
    out, dq, dk, dv = new(B, Q, H, D), new(B, Q, H, D), new(B, N, G, D), new(B, N, G, D)
    table = s["table"].double() if "table" in s else None
    dtable = new(case["buckets"], H)
    key = torch.arange(N, device=DEVICE)
    for b in range(B):
        first = lengths[b] - Q if step else N - Q
        place = torch.arange(first, first + Q, device=DEVICE)[:, None]
        offset = place - key
        seen = (key < lengths[b]) & (place >= 0) & (place < lengths[b])
        if case["window"]:
            seen = seen & ((offset.abs() < case["window"]) | (key < case["sinks"]))
        if case.get("causal", True):
            seen = seen & (offset >= 0)
        bucket = _exact_buckets(case, offset) if table is not None else None
        for h in range(H):
            x, y, z = s["q"][b, :, h].double(), s["k"][b, :, h // (H // G)].double(), s["v"][b, :, h // (H // G)].double()
            score = x @ y.t() / math.sqrt(D)
            if table is not None:
                score = score + table[:, h][bucket]
            score = torch.where(seen, score, -math.inf)
            lse = torch.logsumexp(score, -1, keepdim=True)
            p = torch.where(seen, torch.exp(score - torch.where(seen.any(-1, keepdim=True), lse, 0.0)), 0.0)
            out[b, :, h] = p @ z
            if not train:
                continue
            g = s["grad"][b, :, h].double()
            dv[b, :, h // (H // G)] += p.t() @ g
            dp = g @ z.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            dq[b, :, h] = ds @ y / math.sqrt(D)
            dk[b, :, h // (H // G)] += ds.t() @ x / math.sqrt(D)
            if table is not None:
                dtable[:, h] += torch.stack([ds[bucket == c].sum() for c in range(case["buckets"])])
    if not train:
        return {"out": out}
    grads = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    return grads if table is None else {**grads, "dtable": dtable}
