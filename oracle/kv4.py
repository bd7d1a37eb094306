"""The 4-bit cache, attention over it, eviction and token log probabilities, in 64 bits on the CPU.

The cache format restates `include/deciax_hip.h`; attention is `blocked.attention`'s causal form
(src/deciax/kernels/attention/blocked.py:9-32) with soft-cap and window over one sequence's slots.
"""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """x [..., d] -> (codes 0..15 [..., d], scale bytes [..., d / 32])."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    _, e = np.frexp(np.where(top > 0, top / 6.0, 1e-300))  # top / 6 = f 2^e, f in [0.5, 1): 2^e is at least that
    e = np.where(np.ldexp(1.0, e - 1) >= top / 6.0, e - 1, e)
    e = np.clip(e, -119, 125)
    a = np.abs(b) / np.ldexp(1.0, e)[..., None]
    # midpoints, and which neighbour takes a tie: the even code
    mid = (GRID[1:] + GRID[:-1]) / 2
    code = np.zeros(a.shape, np.int64)
    for i, m in enumerate(mid):
        code += (a > m) if i % 2 == 0 else (a >= m)
    code += 8 * np.signbit(b)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code: np.ndarray, scale: np.ndarray) -> np.ndarray:
    v = GRID[code & 7] * np.where(code > 7, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return (v.reshape(*scale.shape, 32) * s[..., None]).reshape(code.shape)


def pack(code: np.ndarray) -> np.ndarray:
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(b: np.ndarray) -> np.ndarray:
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], 2 * b.shape[-1])


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, positions: np.ndarray, *, scale: float, softcap: float,
              window: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """q [n, Hq, D] newest tokens, k and v [Hkv, ctx, D], positions [Hkv, ctx] -> (out [n, Hq, D], summed weights
    [Hkv, ctx], sum_j p_j |v_j| [n, Hq, D]). Values of slots that a row does not see do not reach it."""
    n, hq, d = q.shape
    hkv, ctx, _ = k.shape
    out, mass = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    weights = np.zeros((hkv, ctx))
    slot = np.arange(ctx)
    for i in range(n):
        own = ctx - n + i
        for h in range(hq):
            g = h // (hq // hkv)
            see = slot <= own
            if window > 0 and own >= 0:
                see &= (slot > own - window) & (positions[g] > positions[g][own] - window)
            if not see.any():
                continue
            with np.errstate(invalid="ignore"):
                t = k[g][see] @ q[i, h] * scale
                if softcap > 0:
                    t = softcap * np.tanh(t / softcap)
                p = np.exp(t - t.max())
                p /= p.sum()
                out[i, h] = p @ v[g][see]
                mass[i, h] = p @ np.abs(v[g][see])
                weights[g][see] += p
    return out, weights, mass


def evict(weights: np.ndarray, keep: int, recent: int) -> np.ndarray:
    """Slots kept of weights [ctx], ascending."""
    ctx = len(weights)
    if ctx <= keep:
        return np.arange(ctx)
    rank = np.where(np.isnan(weights), np.inf, weights.astype(np.float64))
    nan = np.isnan(weights)
    protected = np.arange(ctx) >= ctx - recent
    # protected first, then NaN, then by weight, then the lower slot
    order = np.lexsort((np.arange(ctx), -rank, ~nan, ~protected))
    return np.sort(order[:keep])


def token_logprobs(x: np.ndarray, target: int, top: int, softcap: float) -> tuple[float, float, np.ndarray, np.ndarray]:
    """One row: (log probability of the target, entropy, best tokens, their log probabilities)."""
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or (softcap == 0 and (x == np.inf).any()):
        lp = 0.0 if target == -1 else np.nan
        return lp, np.nan, np.full(top, -1), np.full(top, np.nan)
    t = np.where(x == -np.inf, -np.inf, softcap * np.tanh(x / softcap)) if softcap > 0 else x
    ids, tops = np.full(top, -1), np.full(top, -np.inf)
    if not (x > -np.inf).any():
        lp, ent = -np.inf, 0.0
        logp = t
    else:
        m = t.max()
        logp = (t - m) - np.log(np.exp(t - m).sum())
        p = np.exp(logp)
        ent = float(-(p[p > 0] * logp[p > 0]).sum())
        lp = logp[target] if 0 <= target < len(x) else np.nan
        best = np.lexsort((np.arange(len(x)), -x))[:top]
        best = best[x[best] > -np.inf]
        ids[:len(best)], tops[:len(best)] = best, logp[best]
    if target == -1:
        lp = 0.0
    elif not 0 <= target < len(x):
        lp = np.nan
    return float(lp), ent, ids, tops
