"""The oracle of 4-bit weights, head norms with rotation and linear attention against closed forms."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import token_layer as oracle
from tests.conftest import bf16_np, rng


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_values_are_within_half_a_step(group: int) -> None:
    w = bf16_np(rng(group).normal(size=(5, 2 * group)))
    code, scale, zero = oracle.quantise_q4(w, group)
    off = np.abs(oracle.q4_values(code, scale, zero) - w).reshape(5, 2, group)
    # half a step, and where the rounded scale is too small for the range what is cut at its ends: 15 2^-9 of a step, and
    # the zero's own rounding half a step
    assert (off <= scale[..., None] * (0.5 + 0.5 + 15 * 2.0 ** -9)).all()
    assert code.min() == 0 and code.max() == 15


def test_quantise_special_groups() -> None:
    w = np.zeros((4, 64), np.float32)
    w[1, 3] = np.inf
    w[2, 40] = np.nan
    w[3] = -2.0
    code, scale, zero = oracle.quantise_q4(w, 32)
    v = oracle.q4_values(code, scale, zero)
    assert (v[0] == 0).all() and np.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all() and np.isnan(v[2, 32:]).all()
    assert (code[3] == 0).all() and (zero[3] == 15).all() and abs(v[3, 0] + 2.0) < 2.0 * 2.0 ** -8


def test_layout_words() -> None:
    code = np.zeros((17, 160), np.uint8)
    code[16, 130] = 9   # second tile of rows, second of columns, first word, column 2 of 8: the second nibble
    codes, groups = oracle.lay_out(code, np.full((17, 5), 0.5, np.float32), np.full((17, 5), 3, np.uint8))
    assert codes.shape == (2, 2, 64, 16) and groups.shape == (2, 5, 16)
    assert codes[1, 1, 0, 0] == 9 << 4 and codes.astype(int).sum() == 9 << 4
    assert groups[1, 4, 0] == 0x3F000003 and (groups[1, :, 1:] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_products_of_equal_distance(interleaved: bool) -> None:
    r = rng(1)
    freq = 100.0 ** (-np.arange(8) / 8.0)
    x = np.repeat(r.normal(size=(1, 32)), 4, 0)
    kw = dict(heads=(1, 0), d=32, eps=0.0, interleaved=interleaved, factor=1.0)
    y = oracle.qk_norm_rope(x, np.array([0, 5, 7, 12]), freq, None, None, **kw)
    assert np.allclose(y[0], x[0]) and np.allclose(y[1] @ y[0], y[3] @ y[2])
    assert np.allclose((y ** 2).sum(1), (x ** 2).sum(1)) and (y[:, 16:] == x[:, 16:]).all()


def test_norms_are_one() -> None:
    x = rng(2).normal(size=(3, 64)) * 7
    y = oracle.qk_norm_rope(x, np.zeros(3), np.zeros(0), np.zeros(32), np.ones(32), heads=(1, 1), d=32, eps=0.0,
                            interleaved=False, factor=1.0)
    assert np.allclose((y[:, :32] ** 2).mean(1), 1.0) and np.allclose((y[:, 32:] ** 2).mean(1), 4.0)


def test_recurrence_is_the_weighted_sum() -> None:
    r = rng(3)
    n, h, dk, dv = 9, 2, 4, 3
    q, k, v, g = r.normal(size=(n, 1, dk)), r.normal(size=(n, 1, dk)), r.normal(size=(n, h, dv)), -r.random((n, h))
    s0 = r.normal(size=(h, dk, dv))
    out, s = oracle.linear_attention(q, k, v, g, s0, 0.5)
    for x in range(h):
        total = np.cumsum(g[:, x])
        for i in range(n):
            want = math.exp(total[i]) * q[i, 0] @ s0[x]
            for j in range(i + 1):
                want = want + math.exp(total[i] - total[j]) * (q[i, 0] @ k[j, 0]) * v[j, x]
            assert np.allclose(out[i, x], 0.5 * want)
    first, s1 = oracle.linear_attention(q[:4], k[:4], v[:4], g[:4], s0, 0.5)
    second, s2 = oracle.linear_attention(q[4:], k[4:], v[4:], g[4:], s1, 0.5)
    assert np.allclose(np.concatenate([first, second]), out) and np.allclose(s2, s)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_only_cut_codes_are_further_than_half_a_step(group: int) -> None:
    """A code between 0 and 15 is the nearest one, up to the division's rounding to fp32. One that is cut to 15: range and zero
    together pass 15 by the scale's rounding, 15 2^-8 / (1 - 2^-8) of a step, and by the zero's, half a step."""
    w = bf16_np(rng(group + 1).normal(size=(400, 2 * group)) * np.exp(rng(group + 2).normal(size=(400, 1))))
    code, scale, zero = oracle.quantise_q4(w, group)
    steps = w.reshape(400, 2, group) / scale[..., None].astype(np.float64)
    off = np.abs(code.reshape(steps.shape) - zero[..., None].astype(np.float64) - steps)
    whole = np.rint(steps) + zero[..., None]
    cut = (whole < 0) | (whole > 15)
    assert (off[~cut] <= 0.5 + 16 * 2.0 ** -24).all() and (off[cut] <= 0.5 + 15 / 255 + 16 * 2.0 ** -24).all()
    assert cut.any() and off[~cut].max() > 0.49
