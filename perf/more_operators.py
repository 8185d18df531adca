"""Workloads of the quantised cache and the shared prefix, each beside its plain form.

A transformer that writes clouds point by point keeps the keys and values of
all points before.  In 8 or 4 bits a value they take a half or a quarter of the
memory and of the time that a new token spends reading them: ``cache`` writes
new tokens to such a cache and reads the whole back, ``step`` is the attention
of one or a few new tokens over it, and ``prefix`` that of a batch whose
sequences continue one common start, which is held and read once for all, in the
tokens' type or quantised.  ``run`` computes them by elementary tensor operations in 32 bits,
rounded once at the end, or, where ``own`` is true, by the package's calls.

Shapes: q (B, Q, H, D), keys and values (B, N, G, D), of the common start (P, G, D);
query head h reads key head h // (H // G).  The start's tokens stand before the
sequence's own, of which there are ``lengths``; the queries stand at the last Q.

A quantised row has a scale 2 ** x for each 32 values (the last group may be
shorter): the smallest one, x >= -127, with which the group's largest magnitude
is at most 448 (8 bits) or 6 (4 bits) times it.  The quotients are rounded to the
nearest value of the type (even codes at ties): 8 bits, 3 of them after the point,
exponents from -6 to 8 and even steps of 2 ** -9 below; 4 bits, the values
0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
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
        # The newest token of 16 short sequences is written and all that they
        # hold read back: the smallest call, where latency counts.
        {"name": "cache_token", "kind": "cache", "type": "bf16", "bits": 8, "B": 16, "T": 1, "N": 128, "G": 4,
         "D": 128, "padded": False},
        # A long prompt comes in chunks: one is written to a cache of 4 bits, and
        # what is there so far read back for the chunk's attention.
        {"name": "cache_chunk", "kind": "cache", "type": "bf16", "bits": 4, "B": 4, "T": 2048, "N": 8192, "G": 8,
         "D": 128, "padded": False},
        # Prompts of unequal length, padded to the longest, from a float32 model;
        # odd sizes throughout.
        {"name": "cache_padded", "kind": "cache", "type": "f32", "bits": 8, "B": 7, "T": 333, "N": 1001, "G": 3,
         "D": 40, "padded": True},
        # Eight whole prompts at once.
        {"name": "cache_prompt", "kind": "cache", "type": "f16", "bits": 8, "B": 8, "T": 16384, "N": 16384, "G": 8,
         "D": 128, "padded": False},
        # The next token of four short sequences: a window, first tokens, the bias.
        {"name": "step_small", "kind": "step", "type": "bf16", "bits": 8, "B": 4, "Q": 1, "N": 2048, "H": 8,
         "G": 2, "D": 64, "window": 512, "sinks": 4, "buckets": 32, "reach": 128},
        # The next token of four long sequences, the whole cache visible, 8 bits.
        {"name": "step_long", "kind": "step", "type": "bf16", "bits": 8, "B": 4, "Q": 1, "N": 65536, "H": 32,
         "G": 8, "D": 128, "window": 0, "sinks": 0, "buckets": 0, "reach": 0},
        # The next token of a batch of unequal sequences, 4 bits.
        {"name": "step_batch", "kind": "step", "type": "f16", "bits": 4, "B": 32, "Q": 1, "N": 8192, "H": 32,
         "G": 8, "D": 128, "window": 0, "sinks": 0, "buckets": 0, "reach": 0},
        # Three new tokens at once (a guess to be checked) in float32, odd sizes.
        {"name": "step_odd", "kind": "step", "type": "f32", "bits": 4, "B": 5, "Q": 3, "N": 3001, "H": 6,
         "G": 3, "D": 80, "window": 1000, "sinks": 2, "buckets": 0, "reach": 0},
        # Eight continuations of one small cloud, with a window and the bias.
        {"name": "prefix_small", "kind": "prefix", "type": "bf16", "bits": 16, "B": 8, "Q": 1, "P": 1024, "N": 128,
         "H": 8, "G": 2, "D": 64, "window": 512, "sinks": 4, "buckets": 32, "reach": 128},
        # Many continuations of one long start, where the products count.
        {"name": "prefix_many", "kind": "prefix", "type": "bf16", "bits": 16, "B": 64, "Q": 1, "P": 16384, "N": 512,
         "H": 32, "G": 8, "D": 128, "window": 0, "sinks": 0, "buckets": 0, "reach": 0},
        # Sixteen continuations of a longer one, both quantised.
        {"name": "prefix_coded", "kind": "prefix", "type": "f16", "bits": 8, "B": 16, "Q": 1, "P": 32768, "N": 2048,
         "H": 32, "G": 8, "D": 128, "window": 0, "sinks": 0, "buckets": 0, "reach": 0},
        # Two new tokens each in float32, a window that ends within the start.
        {"name": "prefix_odd", "kind": "prefix", "type": "f32", "bits": 32, "B": 9, "Q": 2, "P": 1537, "N": 300,
         "H": 6, "G": 2, "D": 40, "window": 700, "sinks": 3, "buckets": 20, "reach": 300},
    ]


def _size(rng, low, high):
    """A whole number of the range, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(("cache", "step", "prefix"))
    case = {"kind": kind, "type": rng.choice(("f32", "f16", "bf16"))}
    D = rng.choice((16, 20, 24, 32, 40, 48, 64, 80, 96, 128))
    G = rng.choice((1, 2, 3, 4, 8))
    if kind == "cache":
        N = _size(rng, 1, 16384)
        B = _size(rng, 1, max(1, min(64, (1 << 26) // (N * G * D))))
        return {**case, "bits": rng.choice((8, 4)), "B": B, "T": _size(rng, 1, N), "N": N, "G": G, "D": D,
                "padded": rng.random() < 0.3}
    H = G * rng.choice((1, 1, 2, 3, 4, 8))
    bias = rng.random() < 0.4
    seen = {"window": rng.choice((0, 0, _size(rng, 2, 4096))), "sinks": rng.choice((0, 0, 1, 4, 70)),
            "buckets": rng.choice((8, 16, 32)) if bias else 0, "reach": _size(rng, 32, 1024) if bias else 0}
    Q = rng.choice((1, 1, 1, 2, 5))
    if kind == "step":
        N = _size(rng, 16, 65536)
        B = _size(rng, 1, max(1, min(64, (1 << 27) // (N * G * D * Q))))
        return {**case, "bits": rng.choice((8, 4)), "B": B, "Q": Q, "N": N, "H": H, "G": G, "D": D, **seen}
    coded = rng.random() < 0.5
    P = _size(rng, 16, 32768)
    pairs = (1 << 30) // D // (4 if case["type"] == "f32" else 1)
    B = _size(rng, 1, max(1, min(64, pairs // (P * H * Q))))
    N = _size(rng, 8, max(8, min(2048, (1 << 26) // (B * G * D))))
    return {**case, "bits": rng.choice((8, 4)) if coded else 32 if case["type"] == "f32" else 16, "B": B, "Q": Q,
            "P": P, "N": N, "H": H, "G": G, "D": D, **seen}


# ------------------------------------------------------------------ buckets
def _edges(count, reach):
    """Smallest distance of each bucket but the first: single distances to
    count // 2, then even steps of the logarithm to ``reach``."""
    single = count // 2
    edges = list(range(1, single + 1))
    d = single
    for t in range(1, count - single):
        while d ** (count - single) < reach ** t * single ** (count - single - t):
            d += 1
        edges.append(d)
    return edges


def _lengths(case):
    """Each sequence's own tokens: more than half of the places, or (behind a
    common start) any number from the queries' on."""
    B, N = case["B"], case["N"]
    parts = [(b * 0.6180339887) % 1.0 for b in range(B)]
    if case["kind"] == "prefix":
        low = min(N, case["Q"])
        return [N - int(parts[b] * (N - low)) for b in range(B)]
    if case["kind"] == "cache" and case["padded"]:
        return [min(N, max(1, case["T"] - int(parts[b] * case["T"]))) for b in range(B)]
    return [N if b == 0 else max(1, N - int(parts[b] * N / 2)) for b in range(B)]


# ----------------------------------------------------------- the plain cache
def _power(x):
    """2 ** x of whole numbers in [-126, 127], exactly."""
    return ((x.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, bits):
    """The codes (as the numbers they stand for, in a type of their own) and
    the scales' exponents of (..., D) values."""
    D = x.shape[-1]
    groups = torch.nn.functional.pad(x.float(), (0, -D % 32)).unflatten(-1, (-1, 32))
    most, exponent = torch.frexp(groups.abs().amax(-1))
    exponent = exponent - 9 + (most > 0.875) if bits == 8 else exponent - 3 + (most > 0.75)
    exponent = exponent.clamp(min=-127)
    y = groups * _power(-exponent)[..., None]
    low, digits = (-6, 3) if bits == 8 else (0, 1)
    place = (torch.frexp(y)[1] - 1).clamp(min=low) - digits
    y = torch.round(y * _power(-place)) * _power(place)
    y = y.flatten(-2)[..., :D]
    codes = y.to(torch.float8_e4m3fn) if bits == 8 else (2 * y).to(torch.int8)
    return codes, exponent.to(torch.int16)


def _values(codes, exponent, bits):
    """What the codes stand for, in 32 bits."""
    y = codes.float() if bits == 8 else codes.float() * 0.5
    scale = _power(exponent.clamp(min=-126)) * torch.where(exponent < -126, 0.5, 1.0)
    return y * scale.repeat_interleave(32, -1)[..., :y.shape[-1]]


# ------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """What is drawn, before anything is laid out or quantised."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    B, N, G, D = (case[x] for x in ("B", "N", "G", "D"))
    spread = normal(G, D).mul_(0.5).exp_()  # some of the keys' columns are larger than others
    given = {"lengths": torch.tensor(_lengths(case), device=DEVICE)}
    given["k"], given["v"] = normal(B, N, G, D).mul_(spread).to(dtype), normal(B, N, G, D).to(dtype)
    if case["kind"] == "cache":
        packed = normal(B, case["T"], 2 * G, D)  # one projection's output: keys and values
        packed[:, :, :G] *= spread
        packed = packed.to(dtype)
        given["k_new"], given["v_new"] = packed[:, :, :G], packed[:, :, G:]
        return given
    given["q"] = normal(B, case["Q"], case["H"], D).to(dtype)
    if case["buckets"]:
        given["table"] = (0.5 * normal(case["buckets"], case["H"])).to(dtype)
    if case["kind"] == "prefix":
        P = case["P"]
        given["pk"], given["pv"] = normal(P, G, D).mul_(spread).to(dtype), normal(P, G, D).to(dtype)
    return given


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    bits = case["bits"]
    if case.get("buckets"):
        edges = torch.tensor(_edges(case["buckets"], case["reach"]), device=DEVICE)
        state["limit"] = int(edges[-1])
        state["bucket"] = (torch.arange(state["limit"] + 1, device=DEVICE)[:, None] >= edges).sum(1)
    if case["kind"] == "cache":
        # A padded prompt starts an empty cache; new tokens go behind the old ones.
        state["starts"] = torch.zeros_like(state["lengths"]) if case["padded"] else state["lengths"] - case["T"]
    if bits > 8:
        return state
    for name in ("cache", "prefix"):
        k, v = ("k", "v") if name == "cache" else ("pk", "pv")
        if k not in state:
            continue
        k, v = state.pop(k), state.pop(v)
        if name == "prefix":
            k, v = k[None], v[None]
        if own:
            a = _package()
            state[name] = a.QuantizedCache(k.shape[0], k.shape[1], k.shape[2], k.shape[3], bits=bits, device=DEVICE)
            a.cache_write(state[name], k, v)
        else:
            state[name] = *_quantise(k, bits), *_quantise(v, bits)
    return state


# ---------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    with torch.no_grad():
        if own:
            return {"cache": _own_cache, "step": _own_step, "prefix": _own_prefix}[kind](state)
        return _plain_cache(state) if kind == "cache" else _plain_attn(state)


def _own_cache(s):
    a = _package()
    if s["case"]["padded"]:
        a.cache_write(s["cache"], s["k_new"], s["v_new"], s["lengths"], starts=s["starts"])
    else:
        a.cache_write(s["cache"], s["k_new"], s["v_new"], s["lengths"])
    k, v = a.cache_read(s["cache"], dtype=s["k_new"].dtype)
    return {"k": k, "v": v}


def _how(s):
    case = s["case"]
    return dict(window=case["window"] or None, sinks=case["sinks"], bias=s.get("table"),
                max_distance=case["reach"] or None)


def _own_step(s):
    return {"out": _package().quantized_attention_step(s["q"], s["cache"], s["lengths"], **_how(s))}


def _own_prefix(s):
    coded = s["case"]["bits"] <= 8
    prefix = s["prefix"] if coded else (s["pk"], s["pv"])
    cache = s["cache"] if coded else (s["k"], s["v"])
    return {"out": _package().prefix_attention_step(s["q"], prefix, cache, s["lengths"], **_how(s))}


def _plain_cache(s):
    case, out = s["case"], {}
    B, N, T, bits = case["B"], case["N"], case["T"], case["bits"]
    place = torch.arange(N, device=DEVICE)
    token = place - s["starts"][:, None]  # which new token stands at each place
    new = ((token >= 0) & (token < T) & (place < s["lengths"][:, None]))[:, :, None, None]
    token = token.clamp(0, T - 1)
    rows = torch.arange(B, device=DEVICE)[:, None]
    for i, name in enumerate(("k", "v")):
        codes, exponent = s["cache"][2 * i], s["cache"][2 * i + 1]
        fresh, scale = _quantise(s[name + "_new"], bits)
        # 8-bit values are chosen as the bytes that they are.
        held = codes.view(torch.int8)
        held.copy_(torch.where(new, fresh.view(torch.int8)[rows, token], held))
        exponent.copy_(torch.where(new, scale[rows, token], exponent))
        out[name] = _values(codes, exponent, bits).to(s["k_new"].dtype)
    return out


def _plain_attn(s):
    case = s["case"]
    B, Q, N, H, G, D = (case[x] for x in ("B", "Q", "N", "H", "G", "D"))
    P, rep = case.get("P", 0), H // G
    if case["bits"] > 8:
        (k, v), (pk, pv) = ((s[x].float() for x in names) for names in (("k", "v"), ("pk", "pv")))
    else:
        k, v = (_values(*s["cache"][i:i + 2], case["bits"]) for i in (0, 2))
        if P:
            pk, pv = (_values(*s["prefix"][i:i + 2], case["bits"])[0] for i in (0, 2))
    k, v = (x.transpose(1, 2).contiguous() for x in (k, v))  # (B, G, N, D)
    q = (s["q"].float() * D ** -0.5).reshape(B, Q, G, rep, D).permute(0, 2, 3, 1, 4)  # (B, G, rep, Q, D)
    scores = (q.reshape(B, G, rep * Q, D) @ k.transpose(2, 3)).reshape(B, H, Q, N)
    if P:  # the start once for all sequences
        pk, pv = (x.transpose(0, 1).contiguous() for x in (pk, pv))  # (G, P, D)
        flat = q.permute(1, 0, 2, 3, 4).reshape(G, B * rep * Q, D)
        before = (flat @ pk.transpose(1, 2)).reshape(G, B, rep, Q, P).transpose(0, 1).reshape(B, H, Q, P)
        scores = torch.cat((before, scores), -1)
    key = torch.arange(P + N, device=DEVICE)
    length = P + s["lengths"][:, None, None]
    place = length - Q + torch.arange(Q, device=DEVICE)[:, None]  # (B, Q, 1)
    if "table" in s:
        bucket = s["bucket"][(place - key).clamp(0, s["limit"])]
        scores += s["table"].float()[bucket].permute(0, 3, 1, 2)
    seen = (key <= place) & (key < length) & (place >= 0)
    if case["window"]:
        seen = seen & ((key > place - case["window"]) | (key < case["sinks"]))
    scores = scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    out = (p[..., P:].reshape(B, G, rep * Q, N) @ v).reshape(B, G, rep, Q, D)
    if P:
        flat = p[..., :P].reshape(B, G, rep * Q, P).transpose(0, 1).reshape(G, B * rep * Q, P)
        out = out + (flat @ pv).reshape(G, B, rep, Q, D).transpose(0, 1)
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(B, Q, H, D).to(s["q"].dtype)}


# --------------------------------------------------------------------- work
def _seen(case, length):
    """Of one sequence: the keys of the start and its own that any query sees,
    and the pairs seen."""
    P, Q = case.get("P", 0), case["Q"]
    window = case["window"] or P + case["N"] + 1
    first, pairs = P + length, 0
    for i in range(Q):
        place = P + length - Q + i
        if place < 0:
            continue
        low = max(0, place - window + 1)
        first = min(first, low)
        pairs += place + 1 - low + min(case["sinks"], low)
    sinks = min(case["sinks"], first)
    return max(0, P - first) + min(sinks, P), P + length - max(first, P) + max(0, sinks - P), pairs


def work(case):
    size = 4 if case["type"] == "f32" else 2
    B, N, G, D, bits = (case[x] for x in ("B", "N", "G", "D", "bits"))
    row = 2 * G * (D * bits / 8 + (-(-D // 32) if bits <= 8 else 0))  # a token's keys and values as they are held
    if case["kind"] == "cache":
        starts = [0] * B if case["padded"] else [length - case["T"] for length in _lengths(case)]
        tokens = sum(min(start + case["T"], length) - max(start, 0) for start, length in zip(starts, _lengths(case)))
        return {"bytes": 2 * (tokens + B * N) * G * D * size + (tokens + B * N) * row, "flops": 4 * (tokens + B * N) * G * D}
    seen = [_seen(case, length) for length in _lengths(case)]
    keys = max(x[0] for x in seen) + sum(x[1] for x in seen)
    return {"bytes": 2 * B * case["Q"] * case["H"] * D * size + keys * row, "flops": 4 * case["H"] * D * sum(x[2] for x in seen)}


# -------------------------------------------------------------------- exact
def _representable(bits):
    """The type's values from zero up, in the order of their codes."""
    if bits == 4:
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [m / 512 for m in range(8)] + [2.0 ** e * (1 + m / 8) for e in range(-6, 9) for m in range(8)][:-1]


def _rounded(x, bits):
    """Values in 64 bits as a cache of so many bits holds them, by a search
    among the type's values."""
    table = torch.tensor(_representable(bits), dtype=torch.float64, device=x.device)
    x = x.double()
    two = lambda n: ((n.long() + 1023) << 52).view(torch.float64)  # noqa: E731  2 ** n (a power may miss its last bit)
    out = torch.empty_like(x)
    for first in range(0, x.shape[-1], 32):
        group = x[..., first:first + 32]
        share = group.abs().amax(-1, keepdim=True) / table[-1]
        power = torch.log2(share.clamp(min=2.0 ** -127)).floor()
        power = torch.where(share > two(power), power + 1, power)  # (floor and logarithm may miss by one)
        power = torch.where(share <= two(power - 1), power - 1, power).clamp(min=-127)
        part = (group / two(power)).abs()
        middle = (table[1:] + table[:-1]) / 2
        code = torch.searchsorted(middle, part.contiguous())  # ties: the lower code
        tie = (part == middle[code.clamp(max=len(middle) - 1)]) & (code < len(middle))
        code = code + (tie & (code % 2 == 1))
        out[..., first:first + 32] = torch.copysign(table[code], group) * two(power)
    return out


def exact(case, seed):
    """The definitions in 64 bits, one head of one sequence at a time."""
    with torch.no_grad():
        s = _inputs(case, seed)
        return _exact_cache(s, case) if case["kind"] == "cache" else _exact_attn(s, case)


def _exact_cache(s, case):
    out, T = {}, case["T"]
    for name in ("k", "v"):
        held = torch.stack([_rounded(s[name][b], case["bits"]) for b in range(case["B"])])
        for b, length in enumerate(_lengths(case)):
            start = 0 if case["padded"] else length - T
            low, high = max(start, 0), min(start + T, length)
            held[b, low:high] = _rounded(s[name + "_new"][b, low - start:high - start], case["bits"])
        out[name] = held
    return out


def _exact_attn(s, case):
    B, Q, H, G, D, bits = (case[x] for x in ("B", "Q", "H", "G", "D", "bits"))
    hold = (lambda x: _rounded(x, bits)) if bits <= 8 else (lambda x: x.double())
    P = case.get("P", 0)
    out = torch.zeros(B, Q, H, D, dtype=torch.float64, device=DEVICE)
    table = s["table"].double() if "table" in s else None
    edges = torch.tensor(_edges(case["buckets"], case["reach"]), device=DEVICE) if table is not None else None
    start = [[hold(s[x][:, g]) for x in ("pk", "pv")] for g in range(G)] if P else None
    for b, length in enumerate(_lengths(case)):
        place = P + length - Q + torch.arange(Q, device=DEVICE)[:, None]
        offset = place - torch.arange(P + length, device=DEVICE)
        seen = (offset >= 0) & (place >= 0)
        if case["window"]:
            seen = seen & ((offset < case["window"]) | (place - offset < case["sinks"]))
        bucket = torch.bucketize(offset, edges, right=True) if table is not None else None
        for g in range(G):
            k, v = (hold(s[x][b, :length, g]) for x in ("k", "v"))
            if P:
                k, v = torch.cat((start[g][0], k)), torch.cat((start[g][1], v))
            for h in range(g * (H // G), (g + 1) * (H // G)):
                score = s["q"][b, :, h].double() @ k.t() / math.sqrt(D)
                if table is not None:
                    score = score + table[:, h][bucket]
                score = torch.where(seen, score, -math.inf)
                lse = torch.logsumexp(score, -1, keepdim=True)
                weight = torch.exp(score - torch.where(seen.any(-1, keepdim=True), lse, 0.0))
                out[b, :, h] = torch.where(seen, weight, 0.0) @ v
    return {"out": out}
