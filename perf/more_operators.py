"""The operators of a token layer with 4-bit weights and a state of fixed size, and the calls that are timed of them.

Three kinds of case, each one pass through the package's entry points:

  linear   `kernels.linear_q4`: rows times a weight held in 4 bits with one scale and zero point a group
  rotate   `kernels.qk_norm_rope`: norms of the query and key heads and the rotation by position, in one pass
  decay    `kernels.linear_attention`: S_t = e^g_t S_(t-1) + k_t v_t^T, o_t = scale q_t S_t over packed sequences, the
           states S read and written

The 4-bit weights: W[n, k] = scale * (code - zero), code and zero 0..15, scale a bf16 number, one scale and zero for
`group` neighbouring k of a row. They lie in tiles of 16 rows and 128 columns, in the order in which a wavefront's
lanes read them (`_lay_out`); a tile's missing rows and columns have code 0. A group's 32 bits are its scale's as fp32
with the zero in the lowest four.
"""

from __future__ import annotations

import math
import random
from typing import Any

import numpy as np
import torch

own = False

DEV = "cuda"
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
DTYPES = {"bf16": BF16, "f32": F32}
# The decoder shapes' attention heads: 9B (16/8 heads of 256) and 27B (32/16 heads of 128).
HEADS_9B = dict(hq=16, hkv=8, d=256)
HEADS_27B = dict(hq=32, hkv=16, d=128)
# A layer with states of fixed size at those shapes' widths: key heads, heads, state rows and columns.
STATE_9B = dict(hk=8, h=16, dk=256, dv=256)
STATE_27B = dict(hk=16, h=32, dk=128, dv=128)
CHUNK = 64


def listed() -> list[dict[str, Any]]:
    return [
        # One token through the 9B shape's o projection: latency counts.
        dict(name="linear-1-o", kind="linear", rows=1, n=3584, k=4096, group=128, out="bf16"),
        # One token through its gate and up projections, the widest of a layer.
        dict(name="linear-1-gate-up", kind="linear", rows=1, n=28672, k=3584, group=128, out="bf16"),
        # Answers of a small batch through an odd number of outputs, small groups, the longest sums.
        dict(name="linear-13-odd", kind="linear", rows=13, n=3585, k=14336, group=32, out="bf16"),
        # The logits of four answers in flight.
        dict(name="linear-4-vocab", kind="linear", rows=4, n=256000, k=3584, group=128, out="f32"),
        # A question's rows through the q | k | v projection of the 9B shape.
        dict(name="linear-611-qkv", kind="linear", rows=611, n=8192, k=3584, group=64, out="bf16"),
        # The newest token of each of 48 answers, full rotation, no norms: what a Gemma-2 layer asks for.
        dict(name="rotate-48", kind="rotate", dtype="bf16", **HEADS_9B, rows=48, rot=256, layout="half", norm=False,
             far=9000, stretch=1.0),
        # The serving batch of states: all rows of one layer, norms and a rotation of a quarter of the head.
        dict(name="rotate-70471", kind="rotate", dtype="bf16", **HEADS_9B, rows=70471, rot=64, layout="half", norm=True,
             far=16384, stretch=1.0),
        # Full precision rows of small heads, interleaved pairs, positions far beyond the trained range.
        dict(name="rotate-3001-far", kind="rotate", dtype="f32", hq=12, hkv=4, d=64, rows=3001, rot=32,
             layout="interleaved", norm=True, far=1000000, stretch=32.0),
        # The newest token of each of 48 answers: the states' bytes are what it costs.
        dict(name="decay-48x1", kind="decay", dtype="bf16", **STATE_27B, seqs=48, lo=1, hi=1),
        # One question over its state: few sequences, the work has to be split along the tokens.
        dict(name="decay-1x2111", kind="decay", dtype="bf16", **STATE_9B, seqs=1, lo=2111, hi=2111),
        # A batch of states is read, ragged lengths.
        dict(name="decay-12-states", kind="decay", dtype="bf16", **STATE_27B, seqs=12, lo=517, hi=16384),
        # Full precision, small heads, a few tokens at a time.
        dict(name="decay-f32-5x37", kind="decay", dtype="f32", hk=4, h=4, dk=64, dv=64, seqs=5, lo=3, hi=37),
    ]


def draw(rng: random.Random) -> dict[str, Any]:
    def log(lo: int, hi: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["linear", "linear", "rotate", "decay", "decay"])
    if kind == "linear":
        group, rows = rng.choice([32, 64, 128]), rng.choice([1, log(1, 16), log(16, 900)])
        return dict(kind=kind, rows=rows, n=log(100, 30000 if rows <= 16 else 6000),
                    k=group * log(256 // group, (14336 if rows <= 16 else 5000) // group), group=group,
                    out=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "rotate":
        d = rng.choice([64, 128, 256])
        hkv = rng.choice([1, 2, 5, 8])
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f32"]), hq=hkv * rng.choice([1, 2, 3]), hkv=hkv, d=d,
                    rows=log(1, 20000), rot=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["half", "interleaved"]),
                    norm=rng.random() < 0.6, far=log(100, 2000000), stretch=rng.choice([1.0, 1.0, 8.0]))
    hk, dk, dv = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256]), rng.choice([64, 128, 128, 256])
    long = log(1, min(9000, (1 << 28) // (dk * dv)))
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]), hk=hk, h=hk * rng.choice([1, 2, 3]), dk=dk, dv=dv,
                seqs=rng.randint(1, 32 if long < 200 else 6), lo=max(1, int(long * rng.uniform(0.2, 1.0))), hi=long)


# ------------------------------------------------------------------------------------------ inputs


def _normal(g: torch.Generator, shape: tuple[int, ...], std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=F32, device=DEV).normal_(0.0, std, generator=g)


def _i32(values: Any) -> torch.Tensor:
    return torch.as_tensor(np.asarray(values, np.int32)).to(DEV)


def _lengths(case: dict[str, Any]) -> list[int]:
    """Lengths of a case: part of its size, so the same for every seed; the first is the longest."""
    if case["hi"] <= case["lo"]:
        return [case["lo"]] * case["seqs"]
    r = np.random.Generator(np.random.PCG64(3))
    return [case["hi"]] + [int(round(math.exp(x))) for x in
                           r.uniform(math.log(case["lo"]), math.log(case["hi"]), case["seqs"] - 1)]


def _lay_out(code: torch.Tensor) -> torch.Tensor:
    """Codes [16 a, 128 b] uint8 -> [a, b, 64, 16] bytes: lane 16 q + r of a tile holds row r; its bytes 4 j .. 4 j + 3
    hold the columns 32 j + 8 q + (0, 2 | 4, 6 | 1, 3 | 5, 7), the first of a byte in its low half."""
    a, b = code.shape[0] // 16, code.shape[1] // 128
    t = code.view(a, 16, b, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)  # [a, b, q, r, j, column]
    return (t[..., [0, 4, 1, 5]] | (t[..., [2, 6, 3, 7]] << 4)).reshape(a, b, 64, 16)


def _prepare_linear(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    n, k, group = case["n"], case["k"], case["group"]
    # activations after a norm: some channels are several times as large as others
    x = (_normal(g, (case["rows"], k)) * _normal(g, (k,), 0.7).exp_()).to(BF16)
    rows, cols = -(-n // 16) * 16, -(-k // 128) * 128
    code = torch.empty((rows, cols), dtype=torch.uint8, device=DEV).random_(0, 256, generator=g)
    code = (code & 15).add_(code >> 4).add_(1).div_(2, rounding_mode="floor")  # more of the middle codes, as weights have
    code[n:], code[:, k:] = 0, 0
    scale = (_normal(g, (rows, k // group), 0.3).exp_() * (0.4 / math.sqrt(k))).to(BF16)
    zero = torch.randint(5, 11, (rows, k // group), generator=g, device=DEV, dtype=torch.int32)
    scale[n:], zero[n:] = 0, 0
    groups = (scale.to(F32).view(torch.int32) | zero).view(rows // 16, 16, k // group).transpose(1, 2).contiguous()
    return dict(case=case, x=x, codes=_lay_out(code), groups=groups)


def _prepare_rotate(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    hq, hkv, d, rows = case["hq"], case["hkv"], case["d"], case["rows"]
    t = DTYPES[case["dtype"]]
    # q | k | v rows as the projection leaves them; v is not touched
    x = (_normal(g, (rows, (hq + 2 * hkv) * d), 2.0) * _normal(g, ((hq + 2 * hkv) * d,), 0.3).exp_()).to(t)
    pair = torch.arange(case["rot"] // 2, dtype=F64, device=DEV)
    inv_freq = 10000.0 ** (-2.0 * pair / case["rot"])
    low = 2 * math.pi / inv_freq > 4096  # what has not turned once in the trained length is stretched
    inv_freq = torch.where(low, inv_freq / case["stretch"], inv_freq)
    s = dict(case=case, x=x, inv_freq=inv_freq, factor=0.1 * math.log(case["stretch"]) + 1.0,
             positions=torch.randint(0, case["far"], (rows,), generator=g, device=DEV, dtype=torch.int32),
             out=torch.empty((rows, (hq + hkv) * d), dtype=t, device=DEV))
    s["q_norm"], s["k_norm"] = (_normal(g, (d,), 0.3).to(t) if case["norm"] else None for _ in "qk")
    return s


def _prepare_decay(case: dict[str, Any], g: torch.Generator) -> dict[str, Any]:
    hk, h, dk, dv = case["hk"], case["h"], case["dk"], case["dv"]
    lengths, t = _lengths(case), DTYPES[case["dtype"]]
    rows = sum(lengths)
    k = _normal(g, (rows, hk, dk))
    k = k / k.square().sum(-1, keepdim=True).sqrt()  # unit keys, as such layers have them
    qkv = torch.cat([_normal(g, (rows, hk * dk)), k.flatten(1), _normal(g, (rows, h * dv))], 1).to(t)
    # heads that forget within a token or two next to heads that hold thousands, varying with the token
    rate = torch.empty((h,), device=DEV).uniform_(math.log(2e-4), math.log(2.0), generator=g).exp_()
    decay = -rate * torch.nn.functional.softplus(_normal(g, (rows, h)))
    slots = case["seqs"] + 3
    index = torch.randperm(slots, generator=g, device=DEV)[:case["seqs"]].int()
    state = _normal(g, (slots, h, dk, dv), 0.2)
    return dict(case=case, qkv=qkv, decay=decay, state=state, state_out=state.clone(), index=index, rows=rows,
                lengths=_i32(lengths), starts=_i32([0, *np.cumsum(lengths)[:-1].tolist()]), longest=max(lengths))


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"linear": _prepare_linear, "rotate": _prepare_rotate, "decay": _prepare_decay}[case["kind"]](case, g)


# ------------------------------------------------------------------------------------------ one pass


def run(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    return {"linear": _linear, "rotate": _rotate, "decay": _decay}[s["case"]["kind"]](s)


def _linear(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    if own:
        from deciax_amd import kernels

        weight = kernels.Q4Weight(s["codes"], s["groups"], n, k)
        return (kernels.linear_q4(s["x"], weight, out_dtype=DTYPES[c["out"]]),)
    a, b = s["codes"].shape[:2]
    byte = s["codes"].view(a, b, 4, 16, 4, 4).permute(0, 3, 1, 4, 2, 5)        # [a, r, b, j, q, byte]
    lo, hi = byte & 15, byte >> 4
    code = torch.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]], -1)
    code = code.reshape(16 * a, 128 * b)[:n, :k].unflatten(1, (-1, group))
    word = s["groups"].transpose(1, 2).reshape(16 * a, -1, 1)[:n]
    w = (code.to(F32) - (word & 15)) * (word & -16).view(F32)
    return ((s["x"].to(F32) @ w.flatten(1).T).to(DTYPES[c["out"]]),)


def _rotate(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hq, hkv, d, rot = c["hq"], c["hkv"], c["d"], c["rot"]
    if own:
        from deciax_amd import kernels

        return (kernels.qk_norm_rope(s["x"], s["positions"], s["inv_freq"], num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, layout=c["layout"],
                                     attention_factor=s["factor"], out=s["out"]),)
    x = s["x"][:, :(hq + hkv) * d].to(F32).unflatten(1, (hq + hkv, d))
    if c["norm"]:
        w = torch.cat([s["q_norm"].expand(hq, d), s["k_norm"].expand(hkv, d)]).to(F32)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + w)
    angle = s["positions"].to(F64).unsqueeze(1) * s["inv_freq"]                # in 64 bits: far positions
    cos, sin = ((f(angle) * s["factor"]).to(F32).unsqueeze(1) for f in (torch.cos, torch.sin))
    if c["layout"] == "half":
        p, q = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([p * cos - q * sin, q * cos + p * sin], -1)
    else:
        p, q = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([p * cos - q * sin, q * cos + p * sin], -1).flatten(-2)
    return (torch.cat([turned, x[..., rot:]], -1).flatten(1).to(s["x"].dtype),)


def _decay(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hk, h, dk, dv = c["hk"], c["h"], c["dk"], c["dv"]
    q, k, v = s["qkv"].split([hk * dk, hk * dk, h * dv], 1)
    if own:
        from deciax_amd import kernels

        out = kernels.linear_attention(q, k, v, s["decay"], s["state"], s["starts"], s["lengths"], s["longest"],
                                       num_k_heads=hk, num_heads=h, k_dim=dk, v_dim=dv, scale=dk ** -0.5,
                                       state_index=s["index"], state_out=s["state_out"])
        return out, s["state_out"]
    chunks = -(-s["longest"] // CHUNK)
    i = torch.arange(chunks * CHUNK, device=DEV)
    real = i < s["lengths"].unsqueeze(1)                                       # [seqs, tokens]
    at = (s["starts"].unsqueeze(1) + i).clamp(max=s["rows"] - 1).long()

    def rows(x: torch.Tensor, heads: int) -> torch.Tensor:
        """[seqs, heads, chunks, CHUNK, values] in 32 bits, zeros behind a sequence's end."""
        x = x[at].to(F32).masked_fill(~real.unsqueeze(-1), 0.0).view(c["seqs"], chunks, CHUNK, heads, -1)
        return x.permute(0, 3, 1, 2, 4).repeat_interleave(h // heads, 1)

    q, k, v = rows(q, hk), rows(k, hk), rows(v, h)
    g = rows(s["decay"], h).squeeze(-1).to(F64).cumsum(-1)                     # in 64 bits: long sums
    ends = torch.nn.functional.pad(g[..., -1].cumsum(-1), (1, 0))              # [seqs, h, chunks + 1]

    def between(x: torch.Tensor) -> torch.Tensor:
        """e^(x_i - x_j) for j <= i, else 0."""
        gap = x.unsqueeze(-1) - x.unsqueeze(-2)
        return torch.exp(gap.to(F32)).tril()

    added = (k * torch.exp((g[..., -1:] - g).to(F32)).unsqueeze(-1)).transpose(-1, -2) @ v
    sources = torch.cat([s["state"][s["index"].long()].unsqueeze(2), added], 2).flatten(3)
    states = (between(ends) @ sources).unflatten(3, (dk, dv))                  # before each chunk, and at the end
    o = ((q @ k.transpose(-1, -2)) * between(g)) @ v + (q * torch.exp(g.to(F32)).unsqueeze(-1)) @ states[:, :, :-1]
    out = (o * dk ** -0.5).permute(0, 2, 3, 1, 4).reshape(c["seqs"], -1, h * dv)[real].to(s["qkv"].dtype)
    state = s["state"].clone()
    state[s["index"].long()] = states[:, :, -1]
    return out, state


# ------------------------------------------------------------------------------------------ costs


def work(case: dict[str, Any]) -> dict[str, float]:
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        # half a byte a weight, a bf16 scale and a 4-bit zero a group
        return {"bytes": n * k * (0.5 + 2.5 / case["group"]) + 2 * m * k + m * n * (2 if case["out"] == "bf16" else 4),
                "flops": 2.0 * m * n * k}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "rotate":
        values = case["rows"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * size * values + 4 * case["rows"], "flops": (7.0 if case["norm"] else 3.0) * values}
    hk, h, dk, dv = case["hk"], case["h"], case["dk"], case["dv"]
    rows = sum(_lengths(case))
    return {"bytes": rows * (size * (2 * hk * dk + 2 * h * dv) + 4 * h) + case["seqs"] * 8 * h * dk * dv,
            "flops": 4.0 * rows * h * dk * dv}


# ------------------------------------------------------------------------------------------ in 64 bits


def exact(case: dict[str, Any], seed: int) -> tuple[torch.Tensor, ...]:
    s = prepare(case, seed)
    return {"linear": _linear64, "rotate": _rotate64, "decay": _decay64}[case["kind"]](s)


def _linear64(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    n, k, group = c["n"], c["k"], c["group"]
    x = s["x"].to(F64)
    out = torch.empty((c["rows"], n), dtype=F64, device=DEV)
    column = torch.arange(k, device=DEV)
    # where a column's code is: its tile, the quarter of the lanes, the byte, the half of it
    tile, j, quarter, e = column // 128, column % 128 // 32, column % 32 // 8, column % 8
    byte = 4 * j + 2 * (e % 2) + e // 4
    shift = 4 * (e % 4 // 2)
    step = 1024
    for r0 in range(0, n, step):
        row = torch.arange(r0, min(n, r0 + step), device=DEV).unsqueeze(1)
        code = (s["codes"][row // 16, tile, 16 * quarter + row % 16, byte] >> shift) & 15
        word = s["groups"][row // 16, column // group, row % 16]
        w = (code.to(F64) - (word % 16).to(F64)) * (word - word % 16).view(F32).to(F64)
        out[:, r0:r0 + step] = x @ w.T
    return (out,)


def _rotate64(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hq, hkv, d, rot = c["hq"], c["hkv"], c["d"], c["rot"]
    out = torch.empty((c["rows"], hq + hkv, d), dtype=F64, device=DEV)
    first = torch.arange(rot // 2, device=DEV) * (1 if c["layout"] == "half" else 2)
    second = first + (rot // 2 if c["layout"] == "half" else 1)
    for r in range(0, c["rows"], 4096):
        x = s["x"][r:r + 4096, :(hq + hkv) * d].to(F64).unflatten(1, (hq + hkv, d))
        if c["norm"]:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + 1e-6)
            x = torch.cat([x[:, :hq] * (1.0 + s["q_norm"].to(F64)), x[:, hq:] * (1.0 + s["k_norm"].to(F64))], 1)
        turn = torch.polar(torch.full((1,), s["factor"], dtype=F64, device=DEV),
                           s["positions"][r:r + 4096].to(F64).view(-1, 1, 1) * s["inv_freq"])
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out[r:r + 4096] = x
    return (out.flatten(1),)


def _decay64(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hk, h, dk, dv = c["hk"], c["h"], c["dk"], c["dv"]
    lengths, index = _lengths(c), s["index"].long()
    out = torch.empty((s["rows"], h, dv), dtype=F64, device=DEV)
    state = s["state"].to(F64)
    S = state[index]
    start = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    order = sorted(range(len(lengths)), key=lambda b: -lengths[b])             # the longest first: a prefix is still running
    S = S[order]
    first = _i32(start[order]).long()
    running = [sum(n > t for n in lengths) for t in range(max(lengths))]
    for t, n in enumerate(running):
        row = first[:n] + t
        x = s["qkv"][row].to(F64)
        q, k = (x[:, i * hk * dk:(i + 1) * hk * dk].view(n, hk, dk).repeat_interleave(h // hk, 1) for i in (0, 1))
        v = x[:, 2 * hk * dk:].view(n, h, 1, dv)
        now = S[:n]
        now.mul_(torch.exp(s["decay"][row].to(F64)).view(n, h, 1, 1)).addcmul_(k.unsqueeze(-1), v)
        out[row] = (q.unsqueeze(2) @ now).squeeze(2) * dk ** -0.5
    back = torch.empty_like(S)
    back[order] = S
    state[index] = back
    return out.flatten(1), state
