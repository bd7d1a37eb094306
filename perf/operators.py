"""The operators for answers over a state that was read before, and the calls that are timed of them.

A state's keys and values stay in a paged cache of 4-bit values; later tokens (a question, an answer) attend to it,
a long state gives up the keys that nothing attended to, and given answers are scored by their tokens' log
probabilities. Four kinds of case, each one pass through the package's entry points:

  append   `kernels.kv4_append` of new rows, then `kernels.kv4_read`: the rows as the cache holds them
  attend   `kernels.attention_kv4`: the newest tokens over the cache, with or without the accumulated weights
  evict    `kernels.kv4_evict` to fresh pages, then `kernels.kv4_read` of what was kept
  score    `kernels.token_logprobs`: log probabilities of given tokens, entropy, the best alternatives

The 4-bit format: 32 neighbouring values of a head share a scale 2^e, e the smallest integer with amax <= 6 2^e (kept
in [-119, 125]), stored as the byte e + 127; a value is a sign and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to
the even code) times the scale, two to a byte, the even one in the low half.
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
# The decoder shapes' attention: 9B (16/8 heads of 256, query scale 1/16) and 27B (32/16 heads of 128, 1/12).
HEADS_9B = dict(hq=16, hkv=8, d=256, scale=1 / 16)
HEADS_27B = dict(hq=32, hkv=16, d=128, scale=1 / 12)


def listed() -> list[dict[str, Any]]:
    return [
        # One token of each of 48 answers in flight: the call a decoding loop makes once a layer and step.
        dict(name="append-48x1", kind="append", dtype="bf16", **HEADS_9B, seqs=48, new_lo=1, new_hi=1, ctx_lo=300,
             ctx_hi=9000, page=64),
        # A batch of states is read: all rows of one layer of the serving batch's size, ragged lengths.
        dict(name="append-12-states", kind="append", dtype="bf16", **HEADS_9B, seqs=12, new_lo=517, new_hi=16384,
             ctx_lo=0, ctx_hi=0, page=256),
        # One answer over one state of ordinary length, a global layer: latency counts.
        dict(name="attend-1x2111", kind="attend", dtype="bf16", **HEADS_9B, seqs=1, new_lo=1, new_hi=1, ctx_lo=2111,
             ctx_hi=2111, cap=50.0, window=0, weights=False, page=64),
        # Decoding for a batch of long states, a global layer: the cache's bytes are what it costs.
        dict(name="attend-32x16384", kind="attend", dtype="bf16", **HEADS_9B, seqs=32, new_lo=1, new_hi=1, ctx_lo=9000,
             ctx_hi=16384, cap=50.0, window=0, weights=False, page=256),
        # The same step of the larger shape's sliding layers, with the weights that eviction goes by.
        dict(name="attend-24-window", kind="attend", dtype="bf16", **HEADS_27B, seqs=24, new_lo=1, new_hi=1, ctx_lo=700,
             ctx_hi=12000, cap=50.0, window=4096, weights=True, page=64),
        # Questions of some hundred tokens over their states, weights accumulated.
        dict(name="attend-6-questions", kind="attend", dtype="bf16", **HEADS_9B, seqs=6, new_lo=40, new_hi=611,
             ctx_lo=1500, ctx_hi=8192, cap=50.0, window=0, weights=True, page=64),
        # Full precision queries, small heads, no soft-cap, a few tokens at a time.
        dict(name="attend-f32-5x3", kind="attend", dtype="f32", hq=12, hkv=4, d=64, scale=1 / 8, seqs=5, new_lo=3,
             new_hi=3, ctx_lo=97, ctx_hi=2500, cap=0.0, window=0, weights=True, page=64),
        # One state is cut to a third.
        dict(name="evict-1x2900", kind="evict", **HEADS_9B, seqs=1, ctx_lo=2900, ctx_hi=2900, keep=1000, recent=128,
             page=64),
        # A batch of long states is cut to the sliding layers' length.
        dict(name="evict-12-long", kind="evict", **HEADS_9B, seqs=12, ctx_lo=3000, ctx_hi=16384, keep=4096, recent=512,
             page=256),
        # One decoding step's logits, soft-capped, with alternatives.
        dict(name="score-1", kind="score", dtype="f32", rows=1, vocab=256000, cap=30.0, top=8, banned=0),
        # Answers' tokens over an odd vocabulary, no cap, some tokens banned.
        dict(name="score-301-odd", kind="score", dtype="f32", rows=301, vocab=50257, cap=0.0, top=5, banned=40),
        # All answers of a batch at once.
        dict(name="score-1500", kind="score", dtype="bf16", rows=1500, vocab=256000, cap=30.0, top=4, banned=0),
    ]


def draw(rng: random.Random) -> dict[str, Any]:
    def log(lo: int, hi: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def heads() -> dict[str, Any]:
        if rng.random() < 0.5:
            return dict(rng.choice([HEADS_9B, HEADS_27B]))
        d, hkv = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8])
        return dict(hq=hkv * rng.choice([1, 2, 3, 4, 8]), hkv=hkv, d=d, scale=d ** -0.5)

    kind = rng.choice(["append", "attend", "attend", "attend", "evict", "score", "score"])
    page = rng.choice([64, 64, 128, 256])
    if kind == "append":
        new = log(1, 4000)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f32"]), **heads(), seqs=rng.randint(1, 12), new_lo=new,
                    new_hi=int(new * rng.uniform(1.0, 2.0)), ctx_lo=0, ctx_hi=rng.choice([0, 900]), page=page)
    if kind == "attend":
        new, ctx = rng.choice([1, 1, 1, log(2, 16), log(16, 400)]), log(33, 12000)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f32"]), **heads(), seqs=rng.randint(1, 16 if new < 17 else 4),
                    new_lo=new, new_hi=int(new * rng.uniform(1.0, 1.5)), ctx_lo=ctx, ctx_hi=int(ctx * rng.uniform(1.0, 1.3)),
                    cap=rng.choice([0.0, 50.0]), window=rng.choice([0, 0, 128, 4096]), weights=rng.random() < 0.5, page=page)
    if kind == "evict":
        ctx = log(200, 12000)
        keep = max(2, int(ctx * rng.uniform(0.1, 0.9)))
        return dict(kind=kind, **heads(), seqs=rng.randint(1, 8), ctx_lo=ctx, ctx_hi=int(ctx * rng.uniform(1.0, 1.3)),
                    keep=keep, recent=rng.choice([0, 1, min(keep, 64), keep // 2]), page=page)
    rows, vocab = log(1, 700), rng.choice([1024, 32001, 50257, 151936, 256000])
    return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), rows=rows, vocab=vocab, cap=rng.choice([0.0, 30.0]),
                top=rng.choice([0, 1, 5, 20]), banned=rng.choice([0, 0, 30]))


# ------------------------------------------------------------------------------------------ inputs


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _lengths(case: dict[str, Any], lo: str, hi: str, salt: int) -> list[int]:
    """Lengths of a case: part of its size, so the same for every seed; the first is the longest."""
    if case[hi] <= case[lo]:
        return [case[lo]] * case["seqs"]
    r = np.random.Generator(np.random.PCG64(salt))
    a, b = math.log(max(case[lo], 1)), math.log(case[hi])
    return [case[hi]] + [int(round(math.exp(x))) for x in r.uniform(a, b, case["seqs"] - 1)]


def _shapes(case: dict[str, Any]) -> tuple[list[int], list[int]]:
    """(new tokens, cached tokens with them) of every sequence."""
    old = _lengths(case, "ctx_lo", "ctx_hi", 1)
    if "new_lo" not in case:
        return [0] * case["seqs"], old
    new = _lengths(case, "new_lo", "new_hi", 2)
    return new, [a + b for a, b in zip(new, old)]


def _i32(values: Any) -> torch.Tensor:
    return torch.as_tensor(np.asarray(values, np.int32)).to(DEV)


def _starts(lengths: list[int]) -> list[int]:
    return [0, *np.cumsum(lengths)[:-1].tolist()]


def _normal(g: torch.Generator, shape: tuple[int, ...], std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=F32, device=DEV).normal_(0.0, std, generator=g)


def _keys(g: torch.Generator, rows: int, hkv: int, d: int) -> torch.Tensor:
    """Keys as projections give them: some channels of a head are several times as large as others."""
    channel = _normal(g, (hkv, d), 0.5).exp_()
    return _normal(g, (rows, hkv, d)) * (channel / channel.square().mean(1, keepdim=True).sqrt())


def _codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] -> (codes 0..15 [..., d] uint8, scale bytes [..., d / 32] uint8), in 32 bits: every step is exact."""
    b = x.to(F32).unflatten(-1, (-1, 32))
    bits = b.abs().amax(-1).view(torch.int32)
    e = ((bits >> 23) - 127 - 2 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp(-119, 125)
    r = b * ((127 - e) << 23).view(F32).unsqueeze(-1)  # times 2^-e
    a = r.abs()
    code = (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + \
        (a >= 3.5).byte() + (a > 5.0).byte()
    return (code + 8 * torch.signbit(r).byte()).flatten(-2), (e + 127).byte()


def _bytes(code: torch.Tensor) -> torch.Tensor:
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(packed: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """What the stored bytes [..., d / 2] and scales [..., d / 32] stand for, [..., d] in 32 bits."""
    half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    one = torch.cat([half, -half])
    table = torch.stack([one.repeat(16), one.repeat_interleave(16)], 1)
    return (table[packed.int()].flatten(-2).unflatten(-1, (-1, 32)) *
            (scale.int() << 23).view(F32).unsqueeze(-1)).flatten(-2)


def _pages(case: dict[str, Any], lengths: list[int], g: torch.Generator, first: int = 0) -> tuple[torch.Tensor, int]:
    """Page table [seqs, most] of shuffled pages from `first` on (-1 behind a sequence's last), and how many there are."""
    counts = [-(-n // case["page"]) for n in lengths]
    order = torch.randperm(sum(counts), generator=g, device=DEV).cpu().numpy() + first
    table = np.full((len(counts), max(max(counts), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return _i32(table), at


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = _gen(seed)
    if case["kind"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.empty((rows, vocab), dtype=DTYPES[case["dtype"]], device=DEV).normal_(0.0, 3.0, generator=g)
        targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
        if case["banned"]:
            gone = torch.randint(0, vocab, (case["banned"],), generator=g, device=DEV)
            targets = torch.where(torch.isin(targets, gone), -1, targets).int()  # a banned token is no target
            logits[:, gone] = -math.inf
        # the likely token: most targets are ahead of the field, as a trained model has them
        ahead = (targets >= 0) & (torch.rand(rows, generator=g, device=DEV) < 0.7)
        at = torch.nonzero(ahead).flatten()
        logits[at, targets[at].long()] += 12.0
        return dict(case=case, logits=logits, targets=targets)

    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    new, ctx = _shapes(case)
    seqs, rows = case["seqs"], sum(new)
    table, pages = _pages(case, ctx, g)
    s = dict(case=case, table=table, ctx=_i32(ctx), ctx_host=ctx, max_ctx=max(ctx), new=_i32(new), starts=_i32(_starts(new)),
             rows=rows, max_new=max(new))
    total = pages
    if case["kind"] == "evict":
        kept = [min(n, case["keep"]) for n in ctx]
        s["out_table"], more = _pages(case, kept, g, pages)
        s["kept_rows"], s["kept_starts"], s["pages"], total = sum(kept), _i32(_starts(kept)), pages, pages + more
        # accumulated attention: heavy-tailed, and nothing at all for some keys
        w = _normal(g, (seqs, hkv, max(ctx)), 2.0).exp_() * 0.01
        s["weights"] = w * (torch.rand(w.shape, generator=g, device=DEV) > 0.1)
    shape = (total, hkv, page)
    s["positions"] = torch.zeros(shape, dtype=torch.int32, device=DEV)
    if case["kind"] != "append":
        slot = torch.arange(table.shape[1] * page, device=DEV, dtype=torch.int32).view(1, -1, 1, page)
        used = table >= 0
        s["positions"][table[used].long()] = slot.expand(seqs, -1, hkv, -1)[used]
    for name in ("k", "v"):
        s[name] = torch.zeros((*shape, d // 2), dtype=torch.uint8, device=DEV)
        s[name + "_scale"] = torch.zeros((*shape, d // 32), dtype=torch.uint8, device=DEV)
        if case["kind"] == "append":
            continue
        for p in range(0, pages, 256):  # some pages at a time: the 32-bit values of all of them are eight times the cache
            n = min(256, pages - p) * page
            x = (_keys(g, n, hkv, d) if name == "k" else _normal(g, (n, hkv, d))).unflatten(0, (-1, page)).transpose(1, 2)
            code, scale = _codes(x)
            s[name][p:p + len(x)], s[name + "_scale"][p:p + len(x)] = _bytes(code), scale
    if rows:
        # q | k | v rows as the projection leaves them; the operators take slices of its columns
        s["qkv"] = torch.cat([_normal(g, (rows, hq * d), 2.5), _keys(g, rows, hkv, d).flatten(1),
                              _normal(g, (rows, hkv * d))], 1).to(DTYPES[case["dtype"]])
        where = np.concatenate([np.arange(c - n, c) for n, c in zip(new, ctx)])
        s["where"] = _i32(where)
    if case.get("weights"):
        s["weights"] = _normal(g, (seqs, hkv, max(ctx)), 2.0).exp_() * 0.01
        s["weights_out"] = torch.zeros_like(s["weights"])
    return s


# ------------------------------------------------------------------------------------------ one pass


def run(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    return {"append": _append, "attend": _attend, "evict": _evict, "score": _score}[s["case"]["kind"]](s)


def _append(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    qd, kd = c["hq"] * c["d"], c["hkv"] * c["d"]
    k, v = s["qkv"][:, qd:qd + kd], s["qkv"][:, qd + kd:]
    if own:
        from deciax_amd import kernels

        cache = kernels.KV4Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["positions"])
        kernels.kv4_append(cache, k, v, s["where"], s["table"], s["starts"], s["new"], s["ctx"], s["max_new"])
        held = kernels.kv4_read(cache, s["table"], s["starts"], s["new"], s["ctx"], s["max_new"], rows=s["rows"])
        return (*held, s["positions"])
    held = []
    for x in (k, v):
        code, scale = _codes(x)
        held.append(_values(_bytes(code), scale).to(BF16))
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), s["new"], output_size=s["rows"])
    slot = (s["ctx"] - s["new"] - s["starts"])[seq].long() + torch.arange(s["rows"], device=DEV)
    page = s["table"][seq, slot // c["page"]].long()
    positions = s["positions"].clone()
    positions[page, :, slot % c["page"]] = s["where"].unsqueeze(1).expand(-1, c["hkv"])
    return (*held, positions)


def _cached(s: dict[str, Any], name: str) -> torch.Tensor:
    """[seqs, hkv, slots, d] values of every sequence's pages, in 32 bits."""
    pages = s["table"].clamp(min=0).long()
    return _values(s[name][pages], s[name + "_scale"][pages]).transpose(1, 2).flatten(2, 3)


def _attend(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    q = s["qkv"][:, :hq * d]
    if own:
        from deciax_amd import kernels

        cache = kernels.KV4Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["positions"])
        out = kernels.attention_kv4(q, cache, s["table"], s["starts"], s["new"], s["ctx"], s["max_new"], s["max_ctx"],
                                    num_q_heads=hq, scale=c["scale"], softcap=c["cap"], window=c["window"],
                                    weights=s.get("weights"), weights_out=s.get("weights_out"))
        return (out, s["weights_out"]) if c["weights"] else (out,)
    seqs, n, group = c["seqs"], s["max_new"], hq // hkv
    i = torch.arange(n, device=DEV)
    real = i < s["new"].unsqueeze(1)                                           # [seqs, n]
    at = (s["starts"].unsqueeze(1) + i).clamp(max=s["rows"] - 1).long()
    rows = q[at].to(F32).view(seqs, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * n, d)
    scores = (rows @ _cached(s, "k").transpose(-1, -2) * c["scale"]).view(seqs, hkv, group, n, -1)
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    slot = torch.arange(scores.shape[-1], device=DEV)
    last = (s["ctx"] - s["new"]).unsqueeze(1) + i                              # the query's own slot
    seen = (slot <= last.unsqueeze(-1)) & real.unsqueeze(-1)                   # [seqs, n, slots]
    if c["window"]:
        seen &= slot > (last - c["window"]).unsqueeze(-1)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p.view(seqs, hkv, group * n, -1) @ _cached(s, "v")
    o = o.view(seqs, hkv, group, n, d).permute(0, 3, 1, 2, 4).reshape(seqs, n, hq * d)
    out = o[real].to(q.dtype)
    if not c["weights"]:
        return (out,)
    slot = slot[:s["max_ctx"]]
    old = s["weights"].masked_fill((slot >= (s["ctx"] - s["new"]).unsqueeze(1)).unsqueeze(1), 0.0)
    total = old + p.sum((2, 3))[..., :s["max_ctx"]]
    return out, total.masked_fill((slot >= s["ctx"].unsqueeze(1)).unsqueeze(1), 0.0)


def _evict(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    keep = c["keep"]
    if own:
        from deciax_amd import kernels

        cache = kernels.KV4Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["positions"])
        weights, length = kernels.kv4_evict(cache, s["weights"], s["table"], s["ctx"], s["max_ctx"], s["out_table"],
                                            keep=keep, recent=c["recent"])
        held = kernels.kv4_read(cache, s["out_table"], s["kept_starts"], length, length, keep, rows=s["kept_rows"])
        return (*held, weights, length, s["positions"][s["pages"]:])
    slot = torch.arange(s["max_ctx"], device=DEV)
    ctx = s["ctx"].view(-1, 1, 1)
    rank = s["weights"].masked_fill(slot >= ctx - c["recent"], math.inf).masked_fill(slot >= ctx, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    length = s["ctx"].clamp(max=keep)
    there = torch.arange(order.shape[-1], device=DEV) < length.view(-1, 1, 1)  # [seqs, 1, keep]
    order = order.masked_fill(~there, s["max_ctx"]).sort(-1).values            # in slot order, the missing ones last
    weights = torch.zeros((c["seqs"], c["hkv"], keep), dtype=F32, device=DEV)
    found = s["weights"].gather(-1, order.clamp(max=s["max_ctx"] - 1)).masked_fill(~there, 0.0)
    weights[..., :order.shape[-1]] = found
    order = order.clamp(max=s["max_ctx"] - 1)
    page = s["table"][torch.arange(c["seqs"], device=DEV).view(-1, 1, 1), order // c["page"]].clamp(min=0).long()
    place = (page, torch.arange(c["hkv"], device=DEV).view(1, -1, 1), order % c["page"])
    real = there.squeeze(1)
    held = [_values(s[n][place], s[n + "_scale"][place]).transpose(1, 2)[real].flatten(1).to(BF16) for n in ("k", "v")]
    positions = torch.zeros_like(s["positions"][s["pages"]:])
    out_slot = torch.arange(order.shape[-1], device=DEV)
    out_page = s["out_table"][:, out_slot // c["page"]].long() - s["pages"]
    positions[out_page[real], :, (out_slot % c["page"]).expand(c["seqs"], -1)[real]] = s["positions"][place].transpose(1, 2)[real]
    return (*held, weights, length, positions)


def _score(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    if own:
        from deciax_amd import kernels

        return kernels.token_logprobs(s["logits"], s["targets"], top=c["top"], softcap=c["cap"])
    x = s["logits"].to(F32)
    t = x
    if c["cap"]:
        t = (c["cap"] * torch.tanh(x / c["cap"])).masked_fill(x == -math.inf, -math.inf)
    u = t - t.amax(-1, keepdim=True)
    p = torch.exp(u)
    total = p.sum(-1, keepdim=True)
    norm = torch.log(total)
    u = u - norm                                             # log probabilities
    entropy = norm.squeeze(1) - (p * (u + norm).clamp(min=-1e30)).sum(-1) / total.squeeze(1)
    logprobs = u.gather(1, s["targets"].clamp(min=0).long().unsqueeze(1)).squeeze(1).masked_fill(s["targets"] < 0, 0.0)
    # one whole number orders the alternatives: the logit first, then the lower token
    bits = x.view(torch.int32).long()
    rank = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32) - torch.arange(c["vocab"], device=DEV)
    ids = torch.topk(rank, c["top"], dim=-1).indices
    return logprobs, entropy, ids.int(), u.gather(1, ids)


# ------------------------------------------------------------------------------------------ costs


def work(case: dict[str, Any]) -> dict[str, float]:
    if case["kind"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["rows"] * (12 + 8 * case["top"]), "flops": 6.0 * n}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new, ctx = _shapes(case)
    slot = 2 * hkv * (d // 2 + d // 32)  # K and V of one slot
    size = 2 if case.get("dtype") != "f32" else 4
    if case["kind"] == "append":
        rows = sum(new)
        # rows in, the cache written and read, the values out
        return {"bytes": rows * (2 * hkv * d * (size + 2) + 2 * slot + 4 + 4 * hkv), "flops": 6.0 * rows * 2 * hkv * d}
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in ctx)
        # all weights in; what is kept: cache in and out and in again, weights, positions, values out
        return {"bytes": 4 * hkv * sum(ctx) + kept * (3 * slot + 12 * hkv + 4 * hkv * d), "flops": 4.0 * hkv * sum(ctx)}
    w = case["window"]
    cached, pairs = 0, 0
    for n, c in zip(new, ctx):
        cached += min(c, w + n - 1) if w else c
        seen = [min(c - n + i + 1, w) if w else c - n + i + 1 for i in range(n)]
        pairs += sum(seen)
    total = cached * (slot + (4 * hkv if w else 0)) + sum(new) * hq * d * 2 * size
    if case["weights"]:
        total += 8 * hkv * sum(ctx)
    return {"bytes": total, "flops": 4.0 * d * hq * pairs}


# ------------------------------------------------------------------------------------------ in 64 bits


def exact(case: dict[str, Any], seed: int) -> tuple[torch.Tensor | None, ...] | None:
    s = prepare(case, seed)
    if case["kind"] == "score":
        parts = [_score64(s, r, min(r + 64, case["rows"])) for r in range(0, case["rows"], 64)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), None, torch.cat([p[2] for p in parts])
    if case["kind"] == "append":
        qd, kd = case["hq"] * case["d"], case["hkv"] * case["d"]
        return _nearest64(s["qkv"][:, qd:qd + kd]), _nearest64(s["qkv"][:, qd + kd:]), None
    if case["kind"] == "evict":
        return _evict64(s)
    return _attend64(s)


def _score64(s: dict[str, Any], r0: int, r1: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    c = s["case"]
    x = s["logits"][r0:r1].to(F64)
    t = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
    t = torch.where(torch.isinf(x), x, t)
    logp = t - torch.logsumexp(t, 1, keepdim=True)
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    target = s["targets"][r0:r1].long()
    mine = torch.where(target >= 0, logp[torch.arange(r1 - r0, device=DEV), target.clamp(min=0)], torch.zeros_like(entropy))
    return mine, entropy, torch.sort(logp, 1, descending=True).values[:, :c["top"]]


def _power64(n: torch.Tensor) -> torch.Tensor:
    return ((n.long() + 1023) << 52).view(F64)  # 2^n, from its bits


def _nearest64(x: torch.Tensor) -> torch.Tensor:
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64, device=DEV)
    out = torch.empty(x.shape, dtype=F64, device=DEV)
    for r in range(0, len(x), 2048):
        b = x[r:r + 2048].to(F64).unflatten(-1, (-1, 32))
        top = b.abs().amax(-1, keepdim=True)
        unit = _power64(torch.ceil(torch.log2(top / 6.0)).clamp(-119, 125))
        a = (b.abs() / unit).clamp(max=6.0)
        hi = torch.searchsorted(grid, a).clamp(min=1)                          # grid[hi - 1] <= a <= grid[hi]
        below, above = a - grid[hi - 1], grid[hi] - a
        up = (above < below) | ((above == below) & (hi % 2 == 0))              # a tie goes to the even code
        out[r:r + 2048] = (torch.copysign(grid[hi - 1 + up.long()] * unit, b)).flatten(-2)
    return out


def _held64(s: dict[str, Any], name: str, pages: torch.Tensor) -> torch.Tensor:
    """[hkv, slots, d] in 64 bits, decoded from the bits."""
    raw = s[name][pages].transpose(0, 1).flatten(1, 2)
    scale = s[name + "_scale"][pages].transpose(0, 1).flatten(1, 2)
    code = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)
    power, odd = (code >> 1) & 3, (code & 1).to(F64)
    size = torch.where(power > 0, (1.0 + 0.5 * odd) * _power64(power.long() - 1), 0.5 * odd)
    return torch.where(code > 7, -size, size) * torch.repeat_interleave(_power64(scale.long() - 127), 32, -1)


def _attend64(s: dict[str, Any]) -> tuple[torch.Tensor, ...]:
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    new, ctx = _shapes(c)
    out = torch.empty((sum(new), hq * d), dtype=F64, device=DEV)
    total = torch.zeros((c["seqs"], hkv, max(ctx)), dtype=F64, device=DEV)
    row = 0
    for b, (n, m) in enumerate(zip(new, ctx)):
        pages = s["table"][b, :-(-m // page)].long()
        k, v = (_held64(s, name, pages)[:, :m] for name in ("k", "v"))
        if c["weights"]:
            total[b, :, :m - n] = s["weights"][b, :, :m - n].to(F64)
        for i0 in range(0, n, 64):
            i1 = min(n, i0 + 64)
            q = s["qkv"][row + i0:row + i1, :hq * d].to(F64).view(i1 - i0, hkv, hq // hkv, d)
            at = torch.arange(m - n + i0, m - n + i1, device=DEV).unsqueeze(1)
            j = torch.arange(m, device=DEV)
            hidden = j > at
            if c["window"]:
                hidden |= j <= at - c["window"]
            for h in range(hq):
                t = q[:, h * hkv // hq, h % (hq // hkv)] @ k[h * hkv // hq].T * c["scale"]
                t = c["cap"] * torch.tanh(t / c["cap"]) if c["cap"] else t
                p = torch.softmax(t.masked_fill(hidden, -math.inf), 1)
                out[row + i0:row + i1, h * d:(h + 1) * d] = p @ v[h * hkv // hq]
                total[b, h * hkv // hq, :m] += p.sum(0)
        row += n
    return (out, total) if c["weights"] else (out,)


def _evict64(s: dict[str, Any]) -> tuple[torch.Tensor | None, ...]:
    c = s["case"]
    hkv, d, page, keep = c["hkv"], c["d"], c["page"], c["keep"]
    _, ctx = _shapes(c)
    held = {"k": [], "v": []}
    weights = torch.zeros((c["seqs"], hkv, keep), dtype=F64, device=DEV)
    for b, m in enumerate(ctx):
        w = s["weights"][b, :, :m].cpu().numpy().astype(np.float64)
        n = min(m, keep)
        w[:, max(m - c["recent"], 0):] = np.inf
        slots = np.stack([np.sort(np.lexsort((np.arange(m), -w[h]))[:n]) for h in range(hkv)])
        at = torch.from_numpy(slots).to(DEV)
        weights[b, :, :n] = s["weights"][b].gather(1, at).to(F64)
        for name, rows in held.items():
            x = _held64(s, name, s["table"][b, :-(-m // page)].long())
            rows.append(x.gather(1, at.unsqueeze(-1).expand(-1, -1, d)).transpose(0, 1).flatten(1))
    return torch.cat(held["k"]), torch.cat(held["v"]), weights, None, None
