"""Refusals of the 4-bit cache's and the log probabilities' entry points, on the CPU: every call here is rejected (or is
empty) before the library touches the device."""

from __future__ import annotations

import ctypes

import pytest

from deciax_amd import _lib

P = ctypes.c_void_p(0x10000)  # an aligned, non-null stand-in; never dereferenced by these calls
ODD = ctypes.c_void_p(0x10008)
F = ctypes.c_float
INVALID, UNSUPPORTED, OK = _lib.DX_ERR_INVALID, _lib.DX_ERR_UNSUPPORTED, _lib.DX_OK
BIG = 1 << 40


def cache(k=0x10000, v=0x10000, ks=0x10000, vs=0x10000, pos=0x10000, pages=8, hkv=2, page=64, d=128):
    return ctypes.byref(_lib.Kv4Cache(k, v, ks, vs, pos, pages, hkv, page, d))


CACHES = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(ks=None), INVALID), (dict(vs=None), INVALID),
          (dict(pos=None), INVALID), (dict(pages=-1), INVALID), (dict(pages=0), INVALID), (dict(hkv=0), INVALID), (dict(d=96), UNSUPPORTED),
          (dict(d=512), UNSUPPORTED), (dict(page=32), UNSUPPORTED), (dict(page=96), UNSUPPORTED),
          (dict(page=1 << 17), UNSUPPORTED), (dict(hkv=70000), UNSUPPORTED), (dict(k=0x10008), INVALID),
          (dict(ks=0x10004), INVALID), (dict(pos=0x10004), INVALID)]


def append(c=None, k=P, v=P, pos=P, table=P, width=4, start=P, new=P, ctx=P, seqs=2, max_new=8, rows=16, ks=256, vs=256,
           dtype=_lib.DX_BF16):
    return "dx_kv4_append", (c or cache(), k, v, pos, table, width, start, new, ctx, seqs, max_new, rows, ks, vs, dtype, None)


def read(c=None, k=P, v=P, table=P, width=4, start=P, new=P, ctx=P, seqs=2, max_new=8, rows=16, ks=256, vs=256):
    return "dx_kv4_read", (c or cache(), k, v, table, width, start, new, ctx, seqs, max_new, rows, ks, vs, None)


def attend(c=None, q=P, out=P, table=P, width=4, start=P, new=P, ctx=P, seqs=2, max_new=8, max_ctx=256, rows=16, hq=4,
           qs=512, os=512, scale=0.1, cap=50.0, window=0, w_in=None, wi=(512, 256), w_out=None, wo=(512, 256),
           dtype=_lib.DX_BF16, ws=P, ws_bytes=BIG):
    return "dx_attn_kv4", (c or cache(), q, out, table, width, start, new, ctx, seqs, max_new, max_ctx, rows, hq, qs, os,
                           F(scale), F(cap), window, w_in, *wi, w_out, *wo, dtype, ws, ws_bytes, None)


def evict(c=None, w=P, wi=(512, 256), table=P, width=4, ctx=P, seqs=2, max_ctx=256, out_table=P, out_width=2, keep=100,
          recent=10, w_out=P, wo=(200, 100), out_len=P, ws=P, ws_bytes=BIG):
    return "dx_kv4_evict", (c or cache(), w, *wi, table, width, ctx, seqs, max_ctx, out_table, out_width, keep, recent,
                            w_out, *wo, out_len, ws, ws_bytes, None)


def score(x=P, t=P, rows=3, vocab=100, ld=100, cap=30.0, top=5, lp=P, ent=P, ids=P, tops=P, dtype=_lib.DX_BF16, ws=P,
          ws_bytes=BIG):
    return "dx_token_logprobs", (x, t, rows, vocab, ld, F(cap), top, lp, ent, ids, tops, dtype, ws, ws_bytes, None)


def status(call) -> int:
    name, args = call
    return getattr(_lib.lib(), name)(*args)


def check(call, want: int) -> None:
    got = status(call)
    assert got == want, (call[0], got, want, _lib.lib().dx_last_error())
    if want != OK:
        assert call[0].removeprefix("dx_").encode() in _lib.lib().dx_last_error()


@pytest.mark.parametrize("make", [append, read, attend, evict], ids=lambda f: f.__name__)
@pytest.mark.parametrize("bad,want", CACHES)
def test_malformed_caches_are_refused(make, bad, want) -> None:
    check(make(c=cache(**bad)), want)


@pytest.mark.parametrize("bad,want", [
    (dict(k=None), INVALID), (dict(v=ODD), INVALID), (dict(pos=None), INVALID), (dict(table=None), INVALID),
    (dict(start=None), INVALID), (dict(new=None), INVALID), (dict(ctx=None), INVALID), (dict(seqs=-1), INVALID),
    (dict(seqs=70000), UNSUPPORTED), (dict(max_new=-1), INVALID), (dict(max_new=(1 << 30) + 1), UNSUPPORTED),
    (dict(max_new=1 << 27), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(width=-1), INVALID), (dict(ks=255), INVALID),
    (dict(vs=260), INVALID), (dict(dtype=7), INVALID), (dict(seqs=0), OK), (dict(max_new=0), OK), (dict(rows=0), OK)])
def test_append(bad, want) -> None:
    check(append(**bad), want)


@pytest.mark.parametrize("bad,want", [
    (dict(k=ODD), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID), (dict(ks=128), INVALID),
    (dict(vs=260), INVALID), (dict(max_new=1 << 27), UNSUPPORTED), (dict(seqs=0), OK), (dict(rows=0), OK)])
def test_read(bad, want) -> None:
    check(read(**bad), want)


@pytest.mark.parametrize("bad,want", [
    (dict(q=None), INVALID), (dict(out=ODD), INVALID), (dict(table=None), INVALID), (dict(hq=3), INVALID),
    (dict(hq=0), INVALID), (dict(qs=256), INVALID), (dict(os=516), INVALID), (dict(scale=0.0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(cap=-1.0), INVALID), (dict(cap=1e-40), INVALID), (dict(cap=1e31), INVALID), (dict(window=-1), INVALID), (dict(dtype=3), INVALID),
    (dict(max_ctx=-1), INVALID), (dict(max_ctx=(1 << 30) + 1), UNSUPPORTED), (dict(max_new=1 << 26), UNSUPPORTED),
    (dict(w_out=P), INVALID), (dict(w_in=P, w_out=P, wi=(512, 255)), INVALID),
    (dict(w_in=P, w_out=P, wo=(512, 100)), INVALID), (dict(ws=None, max_ctx=256, w_in=P, w_out=P), INVALID),
    (dict(ws=ctypes.c_void_p(0x10004), max_ctx=9000), INVALID), (dict(ws_bytes=16, max_ctx=9000), INVALID),
    (dict(seqs=70000), UNSUPPORTED), (dict(seqs=0), OK), (dict(max_new=0), OK), (dict(rows=0), OK)])
def test_attention(bad, want) -> None:
    check(attend(**bad), want)


@pytest.mark.parametrize("bad,want", [
    (dict(w=None), INVALID), (dict(table=None), INVALID), (dict(ctx=None), INVALID), (dict(out_table=None), INVALID),
    (dict(w_out=None), INVALID), (dict(out_len=None), INVALID), (dict(keep=0, recent=0), INVALID),
    (dict(recent=101), INVALID), (dict(recent=-1), INVALID), (dict(out_width=1), INVALID), (dict(wi=(512, 255)), INVALID),
    (dict(wo=(200, 99)), INVALID), (dict(ws=None), INVALID), (dict(ws_bytes=100), INVALID), (dict(max_ctx=-1), INVALID),
    (dict(max_ctx=(1 << 30) + 1), UNSUPPORTED), (dict(seqs=70000), UNSUPPORTED), (dict(seqs=0), OK)])
def test_evict(bad, want) -> None:
    check(evict(**bad), want)


@pytest.mark.parametrize("bad,want", [
    (dict(x=None), INVALID), (dict(t=None), INVALID), (dict(lp=None), INVALID), (dict(ent=None), INVALID),
    (dict(ids=None), INVALID), (dict(tops=None), INVALID), (dict(rows=-1), INVALID), (dict(rows=1 << 31), INVALID),
    (dict(vocab=0), INVALID), (dict(ld=99), INVALID), (dict(cap=-1.0), INVALID), (dict(cap=1e-39), INVALID), (dict(top=-1), INVALID),
    (dict(top=101), INVALID), (dict(top=65), UNSUPPORTED), (dict(dtype=9), INVALID),
    (dict(x=ctypes.c_void_p(0x10001)), INVALID), (dict(x=ctypes.c_void_p(0x10002), dtype=_lib.DX_F32), INVALID),
    (dict(ws=None), INVALID), (dict(ws_bytes=10), INVALID), (dict(vocab=(1 << 30) + 1, ld=1 << 31), UNSUPPORTED),
    (dict(rows=0), OK)])
def test_token_logprobs(bad, want) -> None:
    check(score(**bad), want)


def test_workspaces_are_host_arithmetic() -> None:
    lib = _lib.lib()
    assert lib.dx_kv4_evict_workspace(3, 2, 100) == 2400
    assert lib.dx_token_logprobs_workspace(2, 2049, 0) == 2 * 4 * 2 * 3
    assert lib.dx_token_logprobs_workspace(2, 2049, 1) == 2 * 4 * (2 * 3 + 65)
    assert lib.dx_attn_kv4_workspace(0, 1, 1, 4, 2, 128, 0, 1) == 0
    assert lib.dx_attn_kv4_workspace(2, 1, 256, 4, 2, 128, 0, 0) == 0      # one span: no parts to join
    short = lib.dx_attn_kv4_workspace(2, 1, 9000, 4, 2, 128, 0, 0)
    assert 0 < short <= lib.dx_attn_kv4_workspace(2, 300, 9000, 4, 2, 128, 0, 0)
    assert lib.dx_attn_kv4_workspace(2, 1, 9000, 4, 2, 128, 64, 0) < short  # a window splits less


def test_tensors_in_host_memory_are_refused() -> None:
    import torch

    from deciax_amd import kernels as K

    c = K.kv4_cache(4, 2, 64, device="cpu")
    assert c.k.shape == (4, 2, 64, 32) and c.k_scale.shape == (4, 2, 64, 2) and c.positions.dtype == torch.int32
    x = torch.zeros((3, 128), dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        K.kv4_append(c, x, x, torch.zeros(3, dtype=torch.int32), t, i, i, i, 3)
    with pytest.raises(ValueError, match="device"):
        K.attention_kv4(x, c, t, i, i, i, 3, 3, num_q_heads=2, scale=0.1)
    with pytest.raises(ValueError, match="device"):
        K.token_logprobs(x, torch.zeros(3, dtype=torch.int32))


def test_a_cache_keeps_its_arrays() -> None:
    """The library is given the arrays' addresses once: no other array can take the place of one."""
    import torch

    from deciax_amd import kernels as K

    cache = K.kv4_cache(2, 1, 64, device="cpu")
    for name in ("k", "v", "k_scale", "v_scale", "positions"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(1))
    codes, scales = torch.zeros((2, 1, 64, 32), dtype=torch.uint8), torch.zeros((2, 1, 64, 2), dtype=torch.uint8)
    at = torch.zeros((2, 1, 64), dtype=torch.int32)
    for bad in ((codes[0], codes, scales, scales, at), (codes, codes[:1], scales, scales, at),
                (codes, codes, scales, scales[..., :1], at), (codes, codes, scales, scales, at.long()),
                (codes.int(), codes, scales, scales, at), (codes, codes, scales, scales, at[:, :, :32]),
                (codes.transpose(0, 1).expand(2, 2, 64, 32)[:, :1], codes, scales, scales, at)):
        with pytest.raises(ValueError):
            K.KV4Cache(*bad)
    with pytest.raises(ValueError, match="device"):
        K.kv4_read(cache, torch.zeros((1, 1), dtype=torch.int32), *[torch.zeros(1, dtype=torch.int32)] * 3, 1, rows=1)


@pytest.mark.parametrize("call,what", [
    (lambda: attend(w_in=P, w_out=P), b"out must not be q"),      # the weights read q after out is written
    (lambda: evict(w_out=P, ctx=ODD, table=ODD), b"weights_out"),  # kept weights over those that are still to be read
    (lambda: evict(w_out=ODD, table=ODD), b"out_len"),             # lengths that other heads still read
    (lambda: evict(w_out=ODD, ctx=ODD), b"out_table"),             # the old pages
])
def test_arrays_that_a_call_reads_and_writes_must_differ(call, what: bytes) -> None:
    check(call(), INVALID)
    assert what in _lib.lib().dx_last_error()


def test_a_scale_that_vanishes_beside_the_soft_cap_is_refused() -> None:
    """Scores are taken over the soft-cap: scale / softcap has to be a normal number."""
    check(attend(scale=1e-9, cap=1e30), INVALID)
    check(attend(scale=1e-9, cap=1e28, rows=0), OK)


def test_workspaces_beyond_64_bits_are_refused() -> None:
    """The largest bounds that are taken need more bytes than 64 bits count: no wrapped number stands for them."""
    lib = _lib.lib()
    most = (1 << 63) - 1
    assert lib.dx_attn_kv4_workspace(65535, 1, 1 << 30, 65535, 65535, 64, 0, 1) == most
    assert lib.dx_kv4_evict_workspace(65535, 65535, 1 << 30) == most
    many = cache(hkv=65535, d=64)
    check(attend(c=many, out=ctypes.c_void_p(0x20000), hq=65535, qs=65535 * 64, os=65535 * 64, seqs=65535, max_new=1,
                 max_ctx=1 << 30, w_in=P, w_out=ODD, wi=(1 << 47, 1 << 30), wo=(1 << 47, 1 << 30)), INVALID)
    assert b"workspace" in lib.dx_last_error()
    check(evict(c=many, seqs=65535, keep=1 << 30, out_width=1 << 24, wo=(1 << 47, 1 << 30)), INVALID)
    assert b"workspace" in lib.dx_last_error()
