"""The 4-bit oracle against brute force: nearest values, ties to the even code, scale choice, eviction order."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4
from tests.conftest import rng


def test_values_are_the_nearest_with_ties_to_the_even_code() -> None:
    x = np.concatenate([np.linspace(-6.5, 6.5, 1041), [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -5.0, -0.0]])
    x = np.concatenate([x, np.zeros(-len(x) % 31)]).reshape(-1, 31)
    x = np.concatenate([x, np.full((len(x), 1), 6.0)], 1)  # amax 6 or a little above
    code, scale = kv4.quantise(x)
    got = kv4.values(code, scale)
    assert set(np.unique(scale)) <= {127, 128}
    for i in range(x.shape[0]):
        unit = 2.0 ** (int(scale[i, 0]) - 127)
        assert (np.abs(x[i]).max() <= 6 * unit) and (np.abs(x[i]).max() > 3 * unit)
        for j in range(32):
            d = np.abs(kv4.GRID * unit - abs(x[i, j]))
            near = np.flatnonzero(d == d.min())
            want = near[0] if len(near) == 1 else near[near % 2 == 0][0]
            assert code[i, j] & 7 == want and bool(code[i, j] & 8) == bool(np.signbit(x[i, j]))
            assert got[i, j] == np.copysign(kv4.GRID[want] * unit, x[i, j])


@pytest.mark.parametrize("amax,byte", [(0.0, 8), (1e-38, 8), (6.0, 127), (6.000001, 128), (3.0, 126), (3e38, 252),
                                       (np.inf, 255), (np.nan, 255)])
def test_scale_byte(amax: float, byte: int) -> None:
    x = np.zeros((1, 32))
    x[0, 7] = amax
    code, scale = kv4.quantise(x)
    assert scale[0, 0] == byte
    v = kv4.values(code, scale)
    assert np.isnan(v).all() if byte == 255 else np.isfinite(v).all()


def test_pack_round_trip() -> None:
    code = rng(1).integers(0, 16, (3, 64)).astype(np.uint8)
    assert (kv4.unpack(kv4.pack(code)) == code).all()


def test_evict_keeps_recent_then_heavy_then_low_slots() -> None:
    w = np.array([0.5, 0.0, 2.0, 0.5, np.nan, 0.5, 0.0, 0.1])
    assert kv4.evict(w, 4, 1).tolist() == [0, 2, 4, 7]
    assert kv4.evict(w, 8, 1).tolist() == list(range(8))
    assert kv4.evict(w, 2, 2).tolist() == [6, 7]


def test_log_probabilities_far_from_zero() -> None:
    """A common shift changes nothing, however large it is beside the differences."""
    for x in (np.full(35, -3.4e38), np.full(35, 1e300), np.arange(35.0) + 2.0 ** 50):
        lp, ent, ids, tops = kv4.token_logprobs(x, 3, 2, 0.0)
        want = kv4.token_logprobs(x - x[0], 3, 2, 0.0)
        assert abs(lp - want[0]) < 1e-12 and abs(ent - want[1]) < 1e-12
        assert ids.tolist() == want[2].tolist() and np.abs(tops - want[3]).max() < 1e-12
    assert abs(kv4.token_logprobs(np.full(35, -3.4e38), 3, 2, 0.0)[0] + np.log(35)) < 1e-12
