"""Refusals of the entry points of 4-bit weights, head norms with rotation and linear attention, on the CPU: every call
here is rejected (or is empty) before the library touches the device."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from deciax_amd import _lib
from deciax_amd import kernels as K

P = ctypes.c_void_p(0x10000)  # an aligned, non-null stand-in; never dereferenced by these calls
OTHER = ctypes.c_void_p(0x20000)
ODD, BYTE = ctypes.c_void_p(0x10008), ctypes.c_void_p(0x10001)
F = ctypes.c_float
INVALID, UNSUPPORTED, OK = _lib.DX_ERR_INVALID, _lib.DX_ERR_UNSUPPORTED, _lib.DX_OK
BIG = 1 << 40


def quantize(w=P, ldw=256, codes=P, groups=P, n=8, k=256, group=128):
    return "dx_q4_quantize", (w, ldw, codes, groups, n, k, group, None)


def pack(code=P, scales=P, half=0, zeros=None, codes=P, groups=P, n=8, k=256, group=128):
    return "dx_q4_pack", (code, scales, half, zeros, codes, groups, n, k, group, None)


def values(codes=P, groups=P, w=P, ldw=256, n=8, k=256, group=128):
    return "dx_q4_values", (codes, groups, w, ldw, n, k, group, None)


def linear(x=P, codes=P, groups=P, y=P, m=0, n=8, k=256, group=128, ldx=256, ldy=8, dtype=_lib.DX_BF16):
    return "dx_linear_q4", (x, codes, groups, y, m, n, k, group, ldx, ldy, dtype, None)


def turn(x=P, out=P, pos=P, freq=P, qn=None, kn=None, rows=0, hq=4, hkv=2, d=64, rot=64, xs=512, os=384, eps=1e-6,
         factor=1.0, inter=0, dtype=_lib.DX_BF16):
    return "dx_qk_norm_rope", (x, out, pos, freq, qn, kn, rows, hq, hkv, d, rot, xs, os, F(eps), F(factor), inter, dtype,
                               None)


def attend(q=P, k=P, v=P, decay=P, out=OTHER, s_in=P, s_out=P, start=P, length=P, index=None, seqs=0, most=100, states=4,
           rows=100, hk=2, h=4, dk=128, dv=64, qs=256, ks=256, vs=256, ds=4, os=256, scale=0.1, dtype=_lib.DX_BF16, ws=P,
           ws_bytes=BIG):
    return "dx_linear_attn", (q, k, v, decay, out, s_in, s_out, start, length, index, seqs, most, states, rows, hk, h, dk,
                              dv, qs, ks, vs, ds, os, F(scale), dtype, ws, ws_bytes, None)


def check(call, want: int) -> None:
    name, args = call
    got = getattr(_lib.lib(), name)(*args)
    assert got == want, (name, got, want, _lib.lib().dx_last_error())
    if want != OK:
        assert name.removeprefix("dx_").encode() in _lib.lib().dx_last_error()


@pytest.mark.parametrize("make", [quantize, pack, values, linear], ids=lambda f: f.__name__)
@pytest.mark.parametrize("bad,want", [
    (dict(codes=None), INVALID), (dict(groups=None), INVALID), (dict(codes=ODD), INVALID), (dict(groups=ODD), INVALID),
    (dict(n=0), INVALID), (dict(n=-3), INVALID), (dict(k=0), INVALID), (dict(group=16), UNSUPPORTED),
    (dict(group=0), UNSUPPORTED), (dict(group=256), UNSUPPORTED), (dict(k=192), UNSUPPORTED),
    (dict(n=(1 << 24) + 1), UNSUPPORTED), (dict(k=1 << 25), UNSUPPORTED), (dict(n=1 << 24, k=1 << 17), UNSUPPORTED),
    (dict(n=1 << 23, k=1 << 14), UNSUPPORTED)])
def test_malformed_weights_are_refused(make, bad, want) -> None:
    check(make(**bad), want)


@pytest.mark.parametrize("call,want", [
    (quantize(w=None), INVALID), (quantize(w=ODD), INVALID), (quantize(ldw=248), INVALID), (quantize(ldw=260), INVALID),
    (pack(code=None), INVALID), (pack(scales=None), INVALID), (pack(scales=BYTE), INVALID),
    (values(w=None), INVALID), (values(w=BYTE), INVALID), (values(ldw=255), INVALID),
    (linear(x=None), INVALID), (linear(y=None), INVALID), (linear(x=ODD), INVALID), (linear(y=BYTE), INVALID),
    (linear(m=-1), INVALID), (linear(m=(1 << 20) + 1), UNSUPPORTED), (linear(ldx=248), INVALID),
    (linear(ldx=260), INVALID), (linear(ldx=1 << 24), UNSUPPORTED), (linear(ldy=7), INVALID), (linear(dtype=5), INVALID), (linear(), OK)])
def test_q4(call, want) -> None:
    check(call, want)


@pytest.mark.parametrize("bad,want", [
    (dict(x=None), INVALID), (dict(out=None), INVALID), (dict(pos=None), INVALID), (dict(freq=None), INVALID),
    (dict(qn=P), INVALID), (dict(kn=P), INVALID), (dict(rows=-1), INVALID), (dict(hq=-1), INVALID),
    (dict(hkv=-1), INVALID), (dict(dtype=2), INVALID), (dict(d=96, rot=32), UNSUPPORTED), (dict(rot=72), UNSUPPORTED),
    (dict(rot=8), UNSUPPORTED), (dict(rot=128), UNSUPPORTED), (dict(xs=376), INVALID), (dict(os=376), INVALID),
    (dict(xs=388), INVALID), (dict(os=388), INVALID), (dict(x=ODD), INVALID), (dict(out=ODD), INVALID),
    (dict(qn=ODD, kn=P), INVALID), (dict(freq=ctypes.c_void_p(0x10004)), INVALID), (dict(qn=P, kn=P, eps=-1.0), INVALID),
    (dict(qn=P, kn=P, eps=math.nan), INVALID), (dict(rows=(1 << 31) + 1), UNSUPPORTED), (dict(rows=1 << 24), UNSUPPORTED), (dict(), OK),
    (dict(rows=5, hq=0, hkv=0), OK), (dict(xs=388, os=388, dtype=_lib.DX_F32), OK)])
def test_qk_norm_rope(bad, want) -> None:
    check(turn(**bad), want)


@pytest.mark.parametrize("bad,want", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(decay=None), INVALID),
    (dict(out=None), INVALID), (dict(s_in=None), INVALID), (dict(s_out=None), INVALID), (dict(start=None), INVALID),
    (dict(length=None), INVALID), (dict(seqs=-1), INVALID), (dict(most=-1), INVALID), (dict(states=-1), INVALID),
    (dict(rows=-1), INVALID), (dict(hk=0), INVALID), (dict(h=0), INVALID), (dict(h=3), INVALID), (dict(dtype=9), INVALID),
    (dict(dk=96), UNSUPPORTED), (dict(dv=32), UNSUPPORTED), (dict(dk=512), UNSUPPORTED), (dict(seqs=65536), UNSUPPORTED),
    (dict(h=65536), UNSUPPORTED), (dict(most=(1 << 30) + 1), UNSUPPORTED), (dict(scale=0.0), INVALID),
    (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID), (dict(seqs=5), INVALID), (dict(qs=248), INVALID),
    (dict(ks=260), INVALID), (dict(vs=248), INVALID), (dict(os=252), INVALID), (dict(ds=3), INVALID),
    (dict(ds=-4), INVALID), (dict(qs=1 << 24), UNSUPPORTED), (dict(ks=1 << 24), UNSUPPORTED),
    (dict(vs=1 << 24), UNSUPPORTED), (dict(os=1 << 24), UNSUPPORTED), (dict(ds=1 << 22), UNSUPPORTED), (dict(q=ODD), INVALID), (dict(s_in=ODD), INVALID), (dict(s_out=ODD), INVALID),
    (dict(out=P), INVALID), (dict(seqs=3, most=2000, ws_bytes=1000), INVALID), (dict(seqs=3, most=2000, ws=None), INVALID),
    (dict(seqs=3, most=2000, ws=ODD), INVALID), (dict(), OK), (dict(ds=0), OK), (dict(ws=None, ws_bytes=0), OK)])
def test_linear_attention(bad, want) -> None:
    check(attend(**bad), want)


def test_linear_attention_workspace() -> None:
    size = _lib.lib().dx_linear_attn_workspace
    assert size(0, 1000, 4, 64, 64) == 0 and size(3, 512, 4, 64, 64) == 0 and size(3, -1, 4, 64, 64) == 0
    assert size(3, 769, 4, 128, 64) >= 3 * 3 * 4 * (128 * 64 * 4 + 8)  # segments of 320 tokens at least
    assert size(65535, 1 << 30, 65535, 128, 256) >= 65535 * 16 * 65535 * 128 * 256 * 4
    assert size(65535, 1 << 30, 65535, 256, 256) >= 65535 * 8 * 65535 * 256 * 256 * 4
    assert size(2 ** 31 - 1, 1 << 30, 2 ** 31 - 1, 2 ** 31 - 1, 256) == 2 ** 63 - 1


def test_weights_of_other_shapes_are_refused() -> None:
    codes, groups = torch.zeros((2, 3, 64, 16), dtype=torch.uint8), torch.zeros((2, 9, 16), dtype=torch.int32)
    w = K.Q4Weight(codes, groups, 17, 288)
    assert w.group == 32 and w.codes is codes and w.groups is groups
    for n, k, c, g in ((33, 288, codes, groups), (16, 288, codes, groups), (17, 416, codes, groups), (0, 288, codes, groups),
                       (17, 0, codes, groups), (17, 288, codes.int(), groups), (17, 288, codes, groups.long()),
                       (17, 288, codes.transpose(2, 3).contiguous().transpose(2, 3), groups),
                       (17, 288, codes, groups[:, :7]), (17, 288, codes, torch.zeros((2, 0, 16), dtype=torch.int32)),
                       (17, 288, codes, groups[0]), (17, 288, codes, torch.zeros((2, 18, 16), dtype=torch.int32))):
        with pytest.raises(ValueError, match="Q4Weight"):
            K.Q4Weight(c, g, n, k)
    with pytest.raises(AttributeError):
        w.codes = codes
    for call in (lambda: K.linear_q4(torch.zeros((2, 288), dtype=torch.bfloat16), w), lambda: K.q4_values(w),
                 lambda: K.quantize_q4(torch.zeros((2, 288), dtype=torch.bfloat16)),
                 lambda: K.pack_q4(torch.zeros((2, 288), dtype=torch.uint8), torch.zeros((2, 9), dtype=torch.bfloat16)),
                 lambda: K.qk_norm_rope(torch.zeros((2, 128), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32),
                                        torch.zeros(32, dtype=torch.float64), num_q_heads=1, num_kv_heads=1, head_dim=64)):
        with pytest.raises(ValueError, match="device"):  # host memory
            call()


def test_rope_frequencies() -> None:
    plain, one = K.rope_frequencies(64, theta=1e6, device="cpu")
    assert plain.dtype == torch.float64 and plain.shape == (32,) and one == 1.0
    assert torch.allclose(plain, torch.tensor([1e6 ** (-2 * j / 64) for j in range(32)], dtype=torch.float64))
    linear, _ = K.rope_frequencies(64, theta=1e6, scaling={"rope_type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(linear, plain / 4)
    yarn, attention = K.rope_frequencies(64, theta=1e6, scaling={"type": "yarn", "factor": 8.0,
                                                                 "original_max_position_embeddings": 4096}, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert abs(attention - (0.1 * math.log(8.0) + 1)) < 1e-12
    assert torch.equal(yarn[turns > 40], plain[turns > 40]) and torch.allclose(yarn[turns < 0.6], plain[turns < 0.6] / 8)
    assert ((yarn <= plain) & (yarn >= plain / 8)).all() and (yarn[1:] < yarn[:-1]).all()
    given = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, "attention_factor": 1.5}
    assert K.rope_frequencies(64, scaling=given, device="cpu")[1] == 1.5
    llama, attention = K.rope_frequencies(64, theta=1e6, scaling={
        "rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192, "low_freq_factor": 1.0,
        "high_freq_factor": 4.0}, device="cpu")
    for got, f in zip(llama.tolist(), plain.tolist()):
        n = 8192 * f / (2 * math.pi)
        share = (n - 1) / 3
        want = f if n > 4 else f / 8 if n < 1 else (1 - share) * f / 8 + share * f
        assert abs(got - want) < 1e-12 * f
    assert attention == 1.0
    for bad in (dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, theta=0.0),
                dict(rotary_dim=64, scaling={"rope_type": "longrope"}),
                dict(rotary_dim=64, scaling={"rope_type": "yarn", "factor": 2.0}),
                dict(rotary_dim=64, scaling={"rope_type": "linear", "factor": 0.5})):
        with pytest.raises(ValueError, match="rope_frequencies"):
            K.rope_frequencies(**bad, device="cpu")


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "factor": 2.0}, {"rope_type": "linear", "factor": 2.0, "beta_fast": 32},
    {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "mscale": 0.7},
    {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "truncate": False},
    {"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 4096, "beta_fast": 32},
    {"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "linear", "factor": 0.5}, {"rope_type": "yarn", "factor": 2.0}])
def test_rope_scaling_that_is_not_known_is_refused(scaling) -> None:
    with pytest.raises(ValueError, match="rope_frequencies"):
        K.rope_frequencies(64, scaling=scaling, device="cpu")


def test_yarn_needs_a_base_above_one() -> None:
    with pytest.raises(ValueError, match="theta"):
        K.rope_frequencies(64, theta=1.0, device="cpu", scaling={"type": "yarn", "factor": 2.0,
                                                                 "original_max_position_embeddings": 4096})


CONTEXT = {"original_max_position_embeddings": 4096}


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear"}, {"rope_type": "yarn", **CONTEXT}, {"rope_type": "llama3", **CONTEXT},
    {"rope_type": "linear", "factor": None}, {"type": "yarn", "factor": None, **CONTEXT},
    {"rope_type": "linear", "factor": math.nan}, {"rope_type": "linear", "factor": math.inf},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": None},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 0},
    {"rope_type": "llama3", "factor": 4.0, "original_max_position_embeddings": -4096},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": math.nan},
    {"rope_type": "yarn", "factor": 4.0, "beta_slow": 0, **CONTEXT},
    {"rope_type": "yarn", "factor": 4.0, "beta_fast": 1, "beta_slow": 32, **CONTEXT},
    {"rope_type": "yarn", "factor": 4.0, "attention_factor": math.nan, **CONTEXT},
    {"rope_type": "llama3", "factor": 4.0, "low_freq_factor": math.nan, **CONTEXT},
    {"rope_type": "linear", "factor": "four"}], ids=str)
def test_rope_scaling_without_its_numbers_is_refused(scaling) -> None:
    """A factor that is not there is not 1: positions would mean something else than they did in training."""
    with pytest.raises(ValueError, match="rope_frequencies"):
        K.rope_frequencies(64, scaling=scaling, device="cpu")


@pytest.mark.parametrize("name,entries", [("yarn", ("beta_fast", "beta_slow", "attention_factor")),
                                          ("llama3", ("low_freq_factor", "high_freq_factor"))])
def test_rope_scaling_entries_of_none_are_their_defaults(name: str, entries) -> None:
    some = {"rope_type": name, "factor": 4.0, **CONTEXT}
    want, one = K.rope_frequencies(64, scaling=some, device="cpu")
    got, two = K.rope_frequencies(64, scaling=some | dict.fromkeys(entries), device="cpu")
    assert torch.equal(got, want) and one == two


def at(offset: int) -> ctypes.c_void_p:
    return ctypes.c_void_p(0x10000000 + offset)


# q, k, v: 100 rows of 512 bytes, 4 KB apart; decay 100 rows of 16; 4 states of 128 KB
ROWS = 100 * 4096
ARRAYS = dict(q=at(0), k=at(512), v=at(1024), decay=at(ROWS), s_in=at(2 * ROWS), s_out=at(2 * ROWS), start=at(4 * ROWS),
              length=at(4 * ROWS + 64), index=at(4 * ROWS + 128), out=at(5 * ROWS), qs=2048, ks=2048, vs=2048, seqs=2, most=40)
STATES = 4 * 4 * 128 * 64 * 4


@pytest.mark.parametrize("meeting", [
    dict(s_out=at(0)), dict(s_out=at(ROWS - 4096 + 512 - 16)), dict(s_out=at(16 - STATES)), dict(s_out=at(512 + 256)),
    dict(s_out=at(ROWS - 4096 + 1024 + 512 - 16)), dict(s_out=at(ROWS)), dict(s_out=at(ROWS + 1600 - 16)),
    dict(s_in=at(0), s_out=at(0)), dict(s_out=at(2 * ROWS + STATES - 16)), dict(s_out=at(2 * ROWS - STATES + 16)),
    dict(s_out=at(4 * ROWS)), dict(s_out=at(4 * ROWS + 64)), dict(s_out=at(4 * ROWS + 128)),
    dict(out=at(2 * ROWS)), dict(out=at(2 * ROWS + STATES - 16)), dict(s_out=at(5 * ROWS + 99 * 512 + 496)),
    dict(out=at(ROWS)), dict(out=at(4 * ROWS)), dict(out=at(4 * ROWS + 128))], ids=str)
def test_linear_attention_does_not_write_over_what_it_reads(meeting) -> None:
    check(attend(**ARRAYS | meeting), INVALID)
    assert b"meet" in _lib.lib().dx_last_error()


# 100 rows of x and y, 4 KB apart; codes of 8 x 256 are 2 KB (two tiles), their groups 128 bytes
PRODUCT = dict(x=at(0), y=at(2 * ROWS), codes=at(ROWS), groups=at(ROWS + 2048), m=100, ldx=2048, ldy=2048)


@pytest.mark.parametrize("meeting", [
    dict(y=at(ROWS)), dict(y=at(ROWS + 2048)), dict(y=at(ROWS - 99 * 4096)), dict(y=at(ROWS + 2048 - 99 * 4096 + 120)),
    dict(y=at(ROWS + 2046)), dict(codes=at(2 * ROWS)), dict(groups=at(2 * ROWS + 5 * 4096)),
    dict(codes=at(2 * ROWS + 4096 - 2032)), dict(y=at(ROWS + 2040), dtype=_lib.DX_F32, ldy=1024)], ids=str)
def test_products_are_not_written_over_the_weight(meeting) -> None:
    check(linear(**PRODUCT | meeting), INVALID)
    assert b"meet" in _lib.lib().dx_last_error()


@pytest.mark.parametrize("dim,theta,context,factor,fast,slow", [
    (64, 1e6, 4096, 8.0, 32.0, 1.0), (128, 1e4, 4096, 4.0, 32.0, 1.0), (256, 1e4, 8192, 2.5, 24.0, 2.0), (16, 500.0, 64, 3.0, 32.0, 1.0),
    (128, 1e6, 1 << 20, 16.0, 32.0, 1.0)])
def test_yarn_ramps_over_the_pairs(dim, theta, context, factor, fast, slow) -> None:
    """From the last pair that turns `beta_fast` times within the length, or the first of all, to the first one that turns no
    more than `beta_slow` times (counted on beyond the rotated pairs, up to the dimension before the last) the share of the
    frequencies that is divided by the factor grows by the same step from pair to pair."""
    turns = [context * theta ** (-2 * j / dim) / (2 * math.pi) for j in range(dim)]
    low = max([j for j in range(dim) if turns[j] >= fast], default=0)
    high = min([j for j in range(dim) if turns[j] <= slow], default=dim - 1)
    assert high > low
    got, _ = K.rope_frequencies(dim, theta=theta, device="cpu", scaling={
        "rope_type": "yarn", "factor": factor, "original_max_position_embeddings": context, "beta_fast": fast, "beta_slow": slow})
    assert got.shape == (dim // 2,)
    for j, f in enumerate(got.tolist()):
        share = min(max((j - low) / (high - low), 0.0), 1.0)
        want = theta ** (-2 * j / dim) * ((1 - share) + share / factor)
        assert abs(f - want) < 1e-12 * want, j


# 100 rows of 384 of x and out, 4 KB apart; 100 positions, 32 frequencies, norms of 64
TURNED = dict(x=at(0), out=at(ROWS), pos=at(2 * ROWS), freq=at(2 * ROWS + 512), qn=at(2 * ROWS + 1024), kn=at(2 * ROWS + 1152),
              rows=100, xs=2048, os=2048)


@pytest.mark.parametrize("meeting", [
    dict(out=at(2 * ROWS)), dict(out=at(2 * ROWS - 99 * 4096 + 384)), dict(pos=at(ROWS - 396)), dict(freq=at(ROWS + 760)),
    dict(qn=at(ROWS + 4096 - 112)), dict(kn=at(ROWS + 99 * 4096 + 752)), dict(x=at(ROWS), pos=at(ROWS + 764))], ids=str)
def test_turned_heads_are_not_written_over_what_is_read(meeting) -> None:
    check(turn(**TURNED | meeting), INVALID)
    assert b"meet" in _lib.lib().dx_last_error()
