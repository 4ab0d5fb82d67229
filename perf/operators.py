"""Timed cases of the operators that a model needs around its 2-simplicial layers: rotary positions on the
projected heads, and the ordinary causal attention of the layers in between, over whole prompts, packed
sequences of different lengths, chunks of a prompt and single tokens.

`own = False` computes them with elementary torch operations in 32 bits (angles in 64), `own = True` makes
the calls of this library's users.  `exact()` has the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# What a case may say; what it leaves out has these values.
DEFAULTS = dict(
    kind="attend",      # rotate / rotate_step, attend / attend_step: forward call, or forward and gradients
    dtype="bf16",
    S=1,                # sequences
    N=512,              # queries of the longest sequence
    M=0,                # its keys; 0: as many as queries
    H=4, Hkv=0,         # query heads and K/V heads; 0: as many as query heads
    D=64,
    packed=False,       # sequences of different lengths behind one another, [T, H, D]; else [S, N, H, D]
    lens_seed=1,        # their lengths
    layout="bnhd",      # bnhd; bhnd: head-major storage passed as a transposed view; fused: views of one projection's output
    simplicial=False,   # rotate: three tensors (Q, K1, K2) instead of two (Q, K)
    rd=0,               # rotated elements of a head; 0: all
    interleaved=False,  # pairs (2i, 2i + 1) instead of (i, i + rd / 2)
    base=10000.0,
    factor=1.0,         # > 1: low frequencies are interpolated by it
    original=4096,      # ... with respect to this length
    first=0,            # positions count from here
)


def listed():
    return [
        # Eight sequences decode one token each, far into their contexts: a call that is all latency.
        dict(name="rotate_tokens", kind="rotate", S=8, N=1, H=16, Hkv=4, D=64, first=100000),
        # A training step's rotation in a 2-simplicial layer: Q, K1, K2 out of one fused projection, default head size.
        dict(name="rotate_step_layer", kind="rotate_step", S=4, N=2048, H=16, Hkv=8, D=64, simplicial=True, layout="fused"),
        # A long prompt, grouped heads, half of every head rotated in interleaved pairs, frequencies scaled for the length.
        dict(name="rotate_prompt_16k", kind="rotate", dtype="fp16", N=16384, H=32, Hkv=2, D=128, rd=64, interleaved=True, factor=8.0),
        # fp32 and packed, an odd part of the head: a careful small run.
        dict(name="rotate_step_packed_fp32", kind="rotate_step", dtype="fp32", S=5, N=777, H=6, Hkv=3, D=64, rd=24, packed=True),
        # One token of one sequence: the smallest serving call.
        dict(name="attend_token", N=1, M=2001, H=16, Hkv=4, D=64),
        # A batch of sequences of different lengths decodes a token each.
        dict(name="attend_tokens_16k", S=16, N=1, M=16384, H=32, Hkv=2, D=128, packed=True),
        # A chunk of a long prompt over the keys before it.
        dict(name="attend_chunk", N=500, M=16384, H=16, Hkv=2, D=128, layout="fused"),
        # Prefill / evaluation of 8 K tokens, head-major storage.
        dict(name="attend_prompt_8k", S=2, N=8192, H=8, D=128, layout="bhnd"),
        # A training step of a toy model.
        dict(name="attend_step_tiny", kind="attend_step", S=2, N=512, H=4, D=64),
        # fp32: the numerically careful small run (gradient checks, debugging against a reference).
        dict(name="attend_step_fp32", kind="attend_step", dtype="fp32", S=1, N=256, H=2, D=64),
        # Packed training sequences of different lengths in fp16, grouped heads.
        dict(name="attend_step_packed_fp16", kind="attend_step", dtype="fp16", S=9, N=1999, H=16, Hkv=4, D=64, packed=True),
        # A training step at the benchmark's length and heads.
        dict(name="attend_step_8k", kind="attend_step", S=2, N=8192, H=16, Hkv=4, D=128),
    ]


def _full(case):
    c = dict(DEFAULTS, **{k: v for k, v in case.items() if k != "name"})
    c["Hkv"] = c["Hkv"] or c["H"]
    c["M"] = c["M"] or c["N"]
    c["rd"] = c["rd"] or c["D"]
    return c


def _lengths(c):
    """(queries, keys) of every sequence: the first is the longest, packed ones are down to an eighth of it."""
    if not c["packed"]:
        return [(c["N"], c["M"])] * c["S"]
    rng = random.Random(c["lens_seed"])
    out = [(c["N"], c["M"])]
    for _ in range(c["S"] - 1):
        m = rng.randint(max(1, c["M"] // 8), c["M"])
        out.append((m if c["N"] == c["M"] else min(m, rng.randint(max(1, c["N"] // 8), c["N"])), m))
    return out


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["rotate", "rotate_step", "attend", "attend_step"], [20, 20, 35, 25])[0]
    dtype = rng.choices(["bf16", "fp16", "fp32"], [60, 25, 15])[0]
    Hkv = rng.choice([1, 2, 3, 4, 8, 16])
    H = Hkv * rng.choice([1, 1, 2, 4, 8])
    c = dict(kind=kind, dtype=dtype, H=H, Hkv=Hkv, lens_seed=rng.randrange(1 << 30), packed=rng.random() < 0.4)
    if kind.startswith("rotate"):
        D = rng.choice([64, 64, 128, 128, 32, 80, 256])
        c.update(D=D, S=_log_int(rng, 1, 16), N=rng.choice([1, _log_int(rng, 16, 16384)]), interleaved=rng.random() < 0.4,
                 rd=rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), simplicial=rng.random() < 0.4,
                 factor=rng.choice([1.0, 1.0, 4.0, 16.0]), base=rng.choice([10000.0, 500000.0]),
                 first=rng.choice([0, 0, _log_int(rng, 100, 1000000)]))
        if not c["packed"]:
            c["layout"] = rng.choice(["bnhd", "bhnd", "fused"])
        while c["S"] * c["N"] * (H + Hkv) * D > 2e8:
            c["S"], c["N"] = max(1, c["S"] // 2), max(1, int(c["N"] * 0.7))
        return c
    D = rng.choices([64, 128, 32, 80, 256], [40, 45, 5, 5, 5])[0]
    small = dtype == "fp32" or D not in (64, 128)       # what users run at toy sizes
    N = M = _log_int(rng, 17, 1024 if small else 8192)
    if kind == "attend":
        shape = rng.choice(["prompt", "tokens", "chunk"])
        if shape == "tokens":
            N, M = rng.choice([1, 1, 1, 2, 4, 7]), _log_int(rng, 60, 1024 if small else 32768)
        if shape == "chunk":
            M = _log_int(rng, 300, 1024 if small else 16384)
            N = _log_int(rng, 16, min(M, 2048))
    c.update(D=D, N=N, M=M, S=_log_int(rng, 1, 32))
    if not c["packed"]:
        c["layout"] = rng.choice(["bnhd", "bhnd", "fused"])
    # No case beyond the largest listed one (toy sizes for the types used at toy sizes), in scores, and in keys to read.
    most = 1 << 26 if small else 2 * 16 * 8192 * 8192
    while c["S"] * H * c["N"] * c["M"] > most or c["S"] * c["M"] * Hkv * D > 1 << 27:
        if c["S"] > 1:
            c["S"] = max(1, int(c["S"] * 0.7))
        elif c["N"] == c["M"]:
            c["N"] = c["M"] = int(c["N"] * 0.8)
        elif c["N"] > 8:
            c["N"] = int(c["N"] * 0.8)
        else:
            c["M"] = int(c["M"] * 0.8)
    return c


def _randn(g, c, rows, heads, dtype):
    """Tensors of `rows[i]` rows and `heads[i]` heads in the case's layout."""
    D, S = c["D"], c["S"]
    if c["packed"]:
        return [torch.randn(r, h, D, generator=g, device="cuda", dtype=dtype) for r, h in zip(rows, heads)]
    if c["layout"] == "bhnd":
        return [torch.randn(S, h, r, D, generator=g, device="cuda", dtype=dtype).transpose(1, 2) for r, h in zip(rows, heads)]
    if c["layout"] == "fused":
        # every group of tensors with equally many rows is cut out of one buffer
        out = [None] * len(rows)
        for r in sorted(set(rows)):
            of = [i for i, n in enumerate(rows) if n == r]
            buf = torch.randn(S, r, sum(heads[i] for i in of), D, generator=g, device="cuda", dtype=dtype)
            for i, t in zip(of, buf.split([heads[i] for i in of], dim=2)):
                out[i] = t
        return out
    return [torch.randn(S, r, h, D, generator=g, device="cuda", dtype=dtype) for r, h in zip(rows, heads)]


def _starts(lens):
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = _full(case)
    dtype = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lengths(c)
    s = dict(c=c)
    step = c["kind"].endswith("step")
    if c["kind"].startswith("rotate"):
        heads = [c["H"]] + [c["Hkv"]] * (2 if c["simplicial"] else 1)
        rows = sum(n for n, _ in lens) if c["packed"] else c["N"]
        s["inputs"] = [t.detach().requires_grad_(step) for t in _randn(g, c, [rows] * len(heads), heads, dtype)]
        if step:
            s["grads"] = _randn(g, dict(c, layout="bnhd"), [rows] * len(heads), heads, dtype)
        # frequencies in radians a position, low ones interpolated: a frequency with fewer than one turn in the original
        # length is divided by the factor, one with more than 32 stays, in between the share grows with the turns
        f = c["base"] ** (-torch.arange(0, c["rd"], 2, dtype=torch.float64, device="cuda") / c["rd"])
        keep = ((f * c["original"] / (2 * math.pi) - 1) / 31).clamp(0, 1)
        s["frequencies"] = f * (keep + (1 - keep) / c["factor"])
        s["magnitude"] = 1.0 if c["factor"] == 1 else 0.1 * math.log(c["factor"]) + 1
        # positions: sequences of a packed batch start anew; sequences in a batch are at different places
        if c["packed"]:
            s["positions"] = torch.cat([torch.arange(n, device="cuda") + c["first"] for n, _ in lens])
        else:
            at = torch.randint(0, c["first"] + 1, (c["S"], 1), generator=g, device="cuda")
            s["positions"] = at + torch.arange(c["N"], device="cuda")
        return s
    if c["packed"]:
        rows = (sum(n for n, _ in lens), sum(m for _, m in lens))
        s["cu_q"], s["cu_k"] = _starts([n for n, _ in lens]), _starts([m for _, m in lens])
    else:
        rows = (c["N"], c["M"])
    q, k, v = _randn(g, c, (rows[0], rows[1], rows[1]), (c["H"], c["Hkv"], c["Hkv"]), dtype)
    s["inputs"] = [t.detach().requires_grad_(step) for t in (q, k, v)]
    if step:
        s["d_o"] = _randn(g, dict(c, layout="bnhd"), [rows[0]], [c["H"]], dtype)[0]
    return s


# ---- plain forms

def _turn(x, cos, sin, c, inverse=False):
    """x with the first rd elements of every head rotated pair by pair (or back)."""
    rd = c["rd"]
    y = x.float()
    if inverse:
        sin = -sin
    a, b = (y[..., 0:rd:2], y[..., 1:rd:2]) if c["interleaved"] else (y[..., : rd // 2], y[..., rd // 2: rd])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((p, q), -1).flatten(-2) if c["interleaved"] else torch.cat((p, q), -1)
    return torch.cat((turned, y[..., rd:]), -1).to(x.dtype)


def _rotate(s):
    c = s["c"]
    angle = s["positions"].double()[..., None, None] * s["frequencies"]          # [..., 1, rd / 2]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    out = tuple(_turn(x.detach(), cos, sin, c) for x in s["inputs"])
    if c["kind"] == "rotate":
        return out
    return out + tuple(_turn(d, cos, sin, c, inverse=True) for d in s["grads"])


def _padded(x, cu, n):
    """[T, heads, D] -> [S, n, heads, D] of the sequences that start at cu."""
    at = (cu[:-1, None] + torch.arange(n, device=x.device)).clamp(max=x.shape[0] - 1)
    return x[at]


def _unpadded(x, cu, rows):
    """The rows of the sequences behind one another again."""
    at = torch.arange(rows, device=x.device)
    seq = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    return x[seq, at - cu[seq]]


def _by_kv_head(x, Hkv):
    """[S, n, H, D] -> [S, Hkv, G n, D]: the query heads of a K/V head as one list of rows."""
    S, n, H, D = x.shape
    return x.permute(0, 2, 1, 3).reshape(S, Hkv, H // Hkv * n, D)


def _attend(s):
    c = s["c"]
    q, k, v = (t.detach().float() for t in s["inputs"])
    d_o = s["d_o"].float() if "d_o" in s else None
    Hkv, G, N, M = c["Hkv"], c["H"] // c["Hkv"], c["N"], c["M"]
    if c["packed"]:
        rows_q, rows_k = q.shape[0], k.shape[0]
        len_q, len_k = s["cu_q"].diff(), s["cu_k"].diff()
        q, k, v = _padded(q, s["cu_q"], N), _padded(k, s["cu_k"], M), _padded(v, s["cu_k"], M)
        if d_o is not None:
            d_o = _padded(d_o, s["cu_q"], N)
    else:
        len_q = torch.full((c["S"],), N, device="cuda")
        len_k = torch.full((c["S"],), M, device="cuda")
    scale = c["D"] ** -0.5
    i, j = torch.arange(N, device="cuda"), torch.arange(M, device="cuda")
    # query i of n sees the keys up to i + (m - n)
    seen = (j <= i[:, None] + (len_k - len_q)[:, None, None]) & (i < len_q[:, None])[:, :, None]          # [S, N, M]
    seen = seen.repeat(1, G, 1)[:, None]
    qh, kh, vh = _by_kv_head(q, Hkv), k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    logits = (qh @ kh.transpose(2, 3) * scale).masked_fill_(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = (logits - top).exp_()
    p = p / p.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = p @ vh

    def rows_of(x, heads, n):
        return x.reshape(c["S"], heads, n, c["D"]).permute(0, 2, 1, 3)

    out = [rows_of(o, c["H"], N)]
    if d_o is not None:
        dh = _by_kv_head(d_o, Hkv).masked_fill(~seen.any(-1, keepdim=True), 0.0)
        delta = (dh * o).sum(-1, keepdim=True)
        ds = p * (dh @ vh.transpose(2, 3) - delta) * scale
        out += [rows_of(ds @ kh, c["H"], N), rows_of(ds.transpose(2, 3) @ qh, Hkv, M), rows_of(p.transpose(2, 3) @ dh, Hkv, M)]
    if c["packed"]:
        of = [("cu_q", rows_q), ("cu_q", rows_q), ("cu_k", rows_k), ("cu_k", rows_k)]
        out = [_unpadded(x, s[cu], rows) for x, (cu, rows) in zip(out, of)]
    return tuple(x.to(t.dtype).contiguous() for x, t in zip(out, [s["inputs"][0]] + s["inputs"]))


# ---- the library's calls

def _rotate_own(s):
    from simplical_attn_b200 import rotary_positions
    c = s["c"]
    out = rotary_positions(s["inputs"], s["frequencies"], s["positions"], interleaved=c["interleaved"], magnitude=s["magnitude"])
    if c["kind"] == "rotate":
        return out
    return out + torch.autograd.grad(out, s["inputs"], s["grads"])


def _attend_own(s):
    from simplical_attn_b200 import causal_attention
    c = s["c"]
    if c["packed"]:
        o = causal_attention(*s["inputs"], cu_q=s["cu_q"], cu_k=s["cu_k"], max_q=c["N"], max_k=c["M"])
    else:
        o = causal_attention(*s["inputs"])
    if c["kind"] == "attend":
        return (o,)
    return (o,) + torch.autograd.grad(o, s["inputs"], s["d_o"])


def run(state):
    rotate = state["c"]["kind"].startswith("rotate")
    if own:
        return _rotate_own(state) if rotate else _attend_own(state)
    return _rotate(state) if rotate else _attend(state)


def work(case):
    c = _full(case)
    size = 4 if c["dtype"] == "fp32" else 2
    lens = _lengths(c)
    rows_q, rows_k = sum(n for n, _ in lens), sum(m for _, m in lens)
    step = c["kind"].endswith("step")
    if c["kind"].startswith("rotate"):
        heads = c["H"] + c["Hkv"] * (2 if c["simplicial"] else 1)
        passes = 2 if step else 1
        return {"bytes": passes * (2 * rows_q * heads * c["D"] * size + 8 * rows_q) + 4 * c["rd"],
                "flops": passes * 3.0 * rows_q * heads * c["rd"]}
    pairs = sum(n * (m - n) + n * (n + 1) // 2 if m >= n else m * (m + 1) // 2 for n, m in lens)
    unit = 2.0 * pairs * c["H"] * c["D"]                # one product: forward has two of them, backward five (the scores again)
    q, kv = rows_q * c["H"] * c["D"] * size, rows_k * c["Hkv"] * c["D"] * size
    if not step:
        return {"bytes": 2 * q + 2 * kv, "flops": 2 * unit}
    return {"bytes": 4 * q + 4 * kv, "flops": 7 * unit}          # q, k, v, d_o read, o and the gradients written


# ---- definitions in 64 bits

def _exact_rotate(c, s):
    out = []
    n = c["rd"] // 2
    first, second = (range(0, 2 * n, 2), range(1, 2 * n, 2)) if c["interleaved"] else (range(n), range(n, 2 * n))
    for sign, tensors in ((1, s["inputs"]), (-1, s.get("grads", []))):
        w = torch.polar(torch.full((), float(s["magnitude"]), dtype=torch.float64, device="cuda"),
                        sign * s["positions"].to(torch.float64).unsqueeze(-1) * s["frequencies"]).unsqueeze(-2)
        for x in tensors:
            y = x.detach().to(torch.float64).clone()
            z = torch.complex(y[..., list(first)], y[..., list(second)]) * w
            y[..., list(first)], y[..., list(second)] = z.real, z.imag
            out.append(y)
    return tuple(out)


def _exact_attend(c, s):
    q, k, v = (t.detach() for t in s["inputs"])
    step = "d_o" in s
    res = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in ((q, q, k, v) if step else (q,))]
    G = c["H"] // c["Hkv"]
    q0 = k0 = 0
    for b, (n, m) in enumerate(_lengths(c)):
        rq, rk = ((slice(q0, q0 + n),), (slice(k0, k0 + m),)) if c["packed"] else ((b, slice(0, n)), (b, slice(0, m)))
        q0, k0 = q0 + n, k0 + m
        for h in range(c["H"]):
            qi, ki, vi = q[rq + (h,)].double(), k[rk + (h // G,)].double(), v[rk + (h // G,)].double()
            x = torch.einsum("id,jd->ij", qi, ki).div_(math.sqrt(c["D"]))
            x.masked_fill_(torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1), -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)
            o = p @ vi
            res[0][rq + (h,)] = o
            if step:
                d = s["d_o"][rq + (h,)].double()
                res[3][rk + (h // G,)] += p.T @ d
                g = torch.einsum("id,jd->ij", d, vi)
                g = (g - (g * p).sum(-1, keepdim=True)) * p / math.sqrt(c["D"])
                res[1][rq + (h,)] = g @ ki
                res[2][rk + (h // G,)] += g.T @ qi
    return tuple(res)


def exact(case, seed):
    c = _full(case)
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_rotate(c, s) if c["kind"].startswith("rotate") else _exact_attend(c, s)
