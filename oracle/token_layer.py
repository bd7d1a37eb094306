"""Products with 4-bit weights, head norms with rotation and linear attention with decay, in 64 bits on the CPU.

The weight format restates `include/deciax_hip.h`. The norms and the partial rotation are those of
src/deciax/models/qwen3_5/text.py:25-28,75-91 and `apply_rope` (src/deciax/nn.py:35-44); the recurrence is
src/deciax/kernels/gdn/reference.py:24-37 without the delta rule.
"""

from __future__ import annotations

import numpy as np

from oracle.numerics import bf16

NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]  # the columns of a 32-bit word, from its lowest four bits up


def quantise_q4(w: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """w [n, k] (bf16 numbers) -> codes [n, k], scales and zeros [n, k / group]; a group that holds an infinity or a NaN
    has the scale NaN."""
    g = np.asarray(w, np.float32).reshape(w.shape[0], -1, group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], np.float32(0), g)
    lo, hi = np.minimum(g.min(-1), np.float32(0)), np.maximum(g.max(-1), np.float32(0))
    scale = bf16(hi / np.float32(15) - lo / np.float32(15))
    some = scale > 0
    by = np.where(some, scale, np.float32(1))
    zero = np.where(some, np.minimum(np.rint(-lo / by), 15), 0).astype(np.float32)
    code = np.where(some[..., None], np.clip(np.rint(g / by[..., None]) + zero[..., None], 0, 15), 0)
    return code.reshape(w.shape).astype(np.uint8), np.where(bad, np.float32(np.nan), scale), zero.astype(np.uint8)


def q4_values(code: np.ndarray, scale: np.ndarray, zero: np.ndarray) -> np.ndarray:
    n, groups = scale.shape
    c = code.reshape(n, groups, -1).astype(np.float64) - zero[..., None]
    return (c * scale.astype(np.float64)[..., None]).reshape(n, -1)


def lay_out(code: np.ndarray, scale: np.ndarray, zero: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, groups) as a weight holds them, written element by element."""
    n, k = code.shape
    groups = scale.shape[1]
    tiles = -(-n // 16)
    words = np.zeros((tiles, -(-k // 128), 64, 4), np.uint64)
    for col in range(k):
        lane, word, nibble = 16 * (col % 32 // 8), col % 128 // 32, NIBBLES.index(col % 8)
        for row in range(n):
            words[row // 16, col // 128, lane + row % 16, word] |= np.uint64(int(code[row, col]) << (4 * nibble))
    out = np.zeros((tiles, groups, 16), np.uint32)
    for row in range(n):
        out[row // 16, :, row % 16] = (scale[row].astype(np.float32).view(np.uint32) & np.uint32(0xFFFFFFF0)) | zero[row]
    return words.astype("<u4").view(np.uint8), out.view(np.int32)


def qk_norm_rope(x: np.ndarray, positions: np.ndarray, inv_freq: np.ndarray, q_norm: np.ndarray | None,
                 k_norm: np.ndarray | None, *, heads: tuple[int, int], d: int, eps: float, interleaved: bool,
                 factor: float) -> np.ndarray:
    """x [rows, (Hq + Hkv) d] -> the same heads, normed and turned."""
    rows, n = len(x), sum(heads)
    u = np.asarray(x, np.float64).reshape(rows, n, d)
    if q_norm is not None:
        w = np.concatenate([np.repeat(np.asarray(q_norm, np.float64)[None], heads[0], 0),
                            np.repeat(np.asarray(k_norm, np.float64)[None], heads[1], 0)])
        u = u / np.sqrt((u * u).mean(-1, keepdims=True) + eps) * (1.0 + w)
    out = u.copy()
    pairs = len(inv_freq)
    for j in range(pairs):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        angle = np.asarray(positions, np.float64) * inv_freq[j]
        c, s = (factor * np.cos(angle))[:, None], (factor * np.sin(angle))[:, None]
        out[..., a] = u[..., a] * c - u[..., b] * s
        out[..., b] = u[..., b] * c + u[..., a] * s
    return out.reshape(rows, n * d)


def linear_attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, decay: np.ndarray, state: np.ndarray,
                     scale: float) -> tuple[np.ndarray, np.ndarray]:
    """q, k [n, Hk, DK], v [n, H, DV], decay [n, H], state [H, DK, DV] -> (out [n, H, DV], the state at the end)."""
    group = v.shape[1] // k.shape[1]
    s = np.asarray(state, np.float64).copy()
    out = np.zeros(v.shape)
    q, k, v, d = (np.asarray(t, np.float64) for t in (q, k, v, np.exp(np.asarray(decay, np.float64))))
    for t in range(len(q)):
        s *= d[t][:, None, None]
        s += np.repeat(k[t], group, 0)[:, :, None] * v[t][:, None, :]
        out[t] = scale * (np.repeat(q[t], group, 0)[:, None, :] @ s)[:, 0]
    return out, s
