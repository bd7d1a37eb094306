"""The 4-bit cache on the GPU: writing, reading, attention over it and eviction, against the 64-bit oracle.

Tolerances count roundings (u = half a step of a type). Attention of bf16 queries: each weight is rounded to bf16 once
and the output once, 2^-8 each; a score t is off by at most D sums of fp32 products, the conversion to base 2 and the
soft-cap's arithmetic, `score_error`; that moves a weight, relative to the others, by at most twice as much. fp32
queries: weights and queries in three bf16 parts keep 2^-24; sums run over 32 keys a step.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4 as oracle
from tests.conftest import ROOT, i32, rng, say

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
FIELDS = ("k", "v", "k_scale", "v_scale", "positions")


class Case:
    """A cache with random contents, its sequences' page table and the host's copy of all of it."""

    def __init__(self, seed: int, new: list[int], ctx: list[int], hq: int, hkv: int, d: int, page: int = 64,
                 dtype: str = "bf16", garbage: bool = True) -> None:
        import torch

        from deciax_amd import kernels as K

        r = rng(seed)
        self.new, self.ctx, self.hq, self.hkv, self.d, self.page, self.dtype = new, ctx, hq, hkv, d, page, dtype
        counts = [max(1, -(-c // page)) for c in ctx]
        self.pages = sum(counts) + 3
        order = r.permutation(self.pages)
        self.table = np.full((len(ctx), max(counts) + 1), -1, np.int64)  # unused entries name no page
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.pages, hkv, page)
        # whatever a fresh page holds: every byte, the NaN scale among them
        raw = {n: r.integers(0, 256, (*shape, w)).astype(np.uint8) if garbage else np.zeros((*shape, w), np.uint8)
               for n, w in (("k", d // 2), ("v", d // 2), ("k_scale", d // 32), ("v_scale", d // 32))}
        if garbage:
            for n in ("k_scale", "v_scale"):
                raw[n][r.random(raw[n].shape) < 0.3] = 255
        self.raw = raw
        self.pos = r.integers(0, 1 << 30, shape).astype(np.int32)
        self.cache = K.KV4Cache(*(torch.from_numpy(raw[n].copy()).cuda() for n in ("k", "v", "k_scale", "v_scale")),
                                torch.from_numpy(self.pos.copy()).cuda())
        self.d_table, self.d_new, self.d_ctx = i32(self.table), i32(new), i32(ctx)
        self.starts = np.concatenate([[0], np.cumsum(new)[:-1]]).astype(np.int64)
        self.d_starts = i32(self.starts)
        self.rows, self.max_new, self.max_ctx = sum(new), max(new), max(ctx)
        t = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.t = t
        # columns of one packed buffer, as a projection leaves them, with a margin between
        self.qkv = torch.from_numpy(r.normal(size=(self.rows, (hq + 2 * hkv) * d + 16)).astype(np.float32)).cuda().to(t)
        self.q, self.k = self.qkv[:, :hq * d], self.qkv[:, hq * d:(hq + hkv) * d]
        self.v = self.qkv[:, (hq + hkv) * d + 16:]
        self.positions = i32(np.concatenate([np.arange(c - n, c) for n, c in zip(new, ctx)] or [[]]))

    def fill(self, seed: int, std: float = 1.0) -> None:
        """Proper old slots: quantised normals, positions in order."""
        import torch

        r = rng(seed)
        for b, c in enumerate(self.ctx):
            for j in range(c):
                p = self.table[b, j // self.page]
                self.pos[p, :, j % self.page] = j
            pages = self.table[b, :max(1, -(-c // self.page))]
            for n in ("k", "v"):
                x = r.normal(size=(len(pages), self.hkv, self.page, self.d)) * std
                code, scale = oracle.quantise(x)
                keep = np.arange(len(pages) * self.page).reshape(len(pages), 1, self.page, 1) < c
                self.raw[n][pages] = np.where(keep, oracle.pack(code), self.raw[n][pages])
                self.raw[n + "_scale"][pages] = np.where(keep, scale, self.raw[n + "_scale"][pages])
        for n in ("k", "v", "k_scale", "v_scale"):
            getattr(self.cache, n).copy_(torch.from_numpy(self.raw[n]))
        self.cache.positions.copy_(torch.from_numpy(self.pos))

    def host(self, name: str) -> np.ndarray:
        return getattr(self.cache, name).cpu().numpy()

    def held(self, name: str, b: int, table: np.ndarray | None = None, ctx: int | None = None) -> np.ndarray:
        """[hkv, ctx, d] values of a sequence, from the device's bytes."""
        c = self.ctx[b] if ctx is None else ctx
        pages = (self.table if table is None else table)[b, :-(-c // self.page)]
        code = oracle.unpack(self.host(name)[pages])
        v = oracle.values(code, self.host(name + "_scale")[pages])
        return v.transpose(1, 0, 2, 3).reshape(self.hkv, len(pages) * self.page, self.d)[:, :c]

    def held_positions(self, b: int, table: np.ndarray | None = None, ctx: int | None = None) -> np.ndarray:
        c = self.ctx[b] if ctx is None else ctx
        pages = (self.table if table is None else table)[b, :-(-c // self.page)]
        return self.host("positions")[pages].transpose(1, 0, 2).reshape(self.hkv, len(pages) * self.page)[:, :c].astype(np.int64)

    def append(self) -> None:
        from deciax_amd import kernels as K

        K.kv4_append(self.cache, self.k, self.v, self.positions, self.d_table, self.d_starts, self.d_new, self.d_ctx,
                     self.max_new)

    def attend(self, **kw):
        from deciax_amd import kernels as K

        return K.attention_kv4(self.q, self.cache, self.d_table, self.d_starts, self.d_new, self.d_ctx, self.max_new,
                               self.max_ctx, num_q_heads=self.hq, **kw)

    def check(self, out, weights_out=None, weights_in=None, *, scale: float, softcap: float, window: int) -> None:
        """Device results against the oracle on the device's own cache."""
        got = out.float().cpu().numpy().astype(np.float64)
        q = self.q.float().cpu().numpy().astype(np.float64)
        for b, (n, c) in enumerate(zip(self.new, self.ctx)):
            k, v, pos = self.held("k", b), self.held("v", b), self.held_positions(b)
            rows = slice(self.starts[b], self.starts[b] + n)
            qb = q[rows].reshape(n, self.hq, self.d)
            want, wsum, mass = oracle.attention(qb, k, v, pos, scale=scale, softcap=softcap, window=window)
            finite = np.nan_to_num(k)
            # the largest score of the rows that have one: a query that is NaN has none, and is compared as NaN below
            asked = np.where(np.isnan(qb), 0.0, np.abs(qb))
            biggest = max((asked @ np.abs(finite).reshape(-1, self.d).T).max(initial=0.0) * scale, 1.0)
            seen = min(biggest, softcap) if softcap else biggest
            score_error = self.d * U32 * biggest + 8 * U32 * max(seen, softcap)
            moved = 2 * score_error + 8 * U32
            g = got[rows].reshape(n, self.hq, self.d)
            nan = np.isnan(want)
            assert (np.isnan(g) == nan).all(), f"sequence {b}: NaN at other places"
            steps = 32 + c / 32 + 64
            if self.dtype == "bf16":
                tol = (2.0 ** -8 + moved + steps * U32) * mass + 2.0 ** -8 * np.abs(want)
            else:
                tol = (moved + (steps + 4) * U32) * mass + U32 * np.abs(want)
            err = np.abs(np.where(nan, 0, g) - np.where(nan, 0, want))
            assert (err <= np.where(nan, 0, tol) + 1e-30).all(), \
                f"sequence {b}: {np.nanmax(err - np.where(nan, 0, tol)):.3e} beyond the bound, error {err.max():.3e}"
            if weights_out is not None:
                w = weights_out[b, :, :c].cpu().numpy().astype(np.float64)
                old = weights_in[b, :, :c].astype(np.float64).copy()
                old[:, c - n if c > n else 0:] = 0
                group_rows = n * (self.hq // self.hkv)
                wtol = (moved + (16 + group_rows) * U32) * wsum + U32 * np.abs(old + wsum) + 1e-30
                wn = np.isnan(wsum)
                assert (np.isnan(w) == wn).all()
                assert (np.abs(np.where(wn, 0, w - old - wsum)) <= np.where(wn, 0, wtol)).all(), \
                    f"sequence {b}: weights off by {np.nanmax(np.abs(w - old - wsum)):.3e}"


# ------------------------------------------------------------------------------------------ append and read


@pytest.mark.parametrize("d,hkv,page,dtype", [(64, 1, 64, "bf16"), (128, 3, 64, "bf16"), (256, 8, 128, "f32"),
                                              (64, 5, 256, "f32"), (256, 1, 64, "bf16")])
def test_append_and_read_are_exact(d: int, hkv: int, page: int, dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    new, ctx = [1, 70, 0, 129, 5], [1, 70, 9, 300, 3]  # the last: more new tokens than slots
    say(f"kv4 append d={d} hkv={hkv} page={page} {dtype}")
    c = Case(d + hkv, new, ctx, hkv, hkv, d, page, dtype)
    r = rng(5)
    x = c.qkv.float().cpu().numpy()
    # the whole range, ties, zeros, and what no 4-bit number can hold
    x *= np.exp2(r.integers(-40, 40, (x.shape[0], 1))).astype(np.float32)
    x[0, :] = 0
    x[1] *= np.float32(1e-38)
    x[2, hkv * d + 3] = np.inf
    x[3, hkv * d + 40] = np.nan
    x[4, hkv * d:hkv * d + 32] = np.float32(3e38)
    x[5, hkv * d:hkv * d + 32] = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4, np.float32) * np.float32(0.125)
    c.qkv.copy_(torch.from_numpy(x).to(c.t))
    before = {n: c.host(n).copy() for n in ("k", "v", "k_scale", "v_scale", "positions")}
    c.append()
    torch.cuda.synchronize()
    touched = np.zeros((c.pages, page), bool)
    for b, (n, m) in enumerate(zip(new, ctx)):
        for i in range(n):
            slot = m - n + i
            if slot < 0:
                continue
            p, at = c.table[b, slot // page], slot % page
            touched[p, at] = True
            row = c.starts[b] + i
            for name, t in (("k", c.k), ("v", c.v)):
                code, scale = oracle.quantise(t[row].float().cpu().numpy().reshape(hkv, d))
                np.testing.assert_array_equal(c.host(name)[p, :, at], oracle.pack(code))
                np.testing.assert_array_equal(c.host(name + "_scale")[p, :, at], scale)
            assert (c.host("positions")[p, :, at] == slot).all()
    for n, old in before.items():  # nothing else was written
        np.testing.assert_array_equal(c.host(n).transpose(0, 2, 1, *range(3, old.ndim))[~touched],
                                      old.transpose(0, 2, 1, *range(3, old.ndim))[~touched])
    k, v = K.kv4_read(c.cache, c.d_table, c.d_starts, c.d_new, c.d_ctx, c.max_new, rows=c.rows)
    for name, t in (("k", k), ("v", v)):
        t = t.float().cpu().numpy()
        for b, (n, m) in enumerate(zip(new, ctx)):
            held = c.held(name, b)
            for i in range(n):
                want = held[:, m - n + i].reshape(-1) if m - n + i >= 0 else np.zeros(hkv * d)
                np.testing.assert_array_equal(t[c.starts[b] + i], want.astype(np.float32))


def test_pages_and_rows_out_of_range_are_not_touched() -> None:
    """A table entry outside the pool, and a sequence whose rows leave the packed buffer: nothing is written for them."""
    import torch

    from deciax_amd import kernels as K

    say("kv4 with bad pages and rows")
    c = Case(3, [40, 10], [100, 10], 2, 2, 64, garbage=False)
    c.table[0, 1] = c.pages + 7
    c.d_table = i32(c.table)
    c.d_starts = i32([0, 45])  # rows 50.. of the second do not exist
    c.append()
    k, v = K.kv4_read(c.cache, c.d_table, c.d_starts, c.d_new, c.d_ctx, c.max_new, rows=c.rows)
    torch.cuda.synchronize()
    used = c.table[1, 0]
    held = c.host("k_scale")
    assert (held[used, :, :5] != 0).all() and (held[used, :, 5:] == 0).all()
    assert (k[36:40].float().cpu().numpy() == 0).all()  # slots 96.. lie in the page that is not there
    out = c.attend(scale=0.125)
    torch.cuda.synchronize()
    assert torch.isfinite(out[:40].float()).all()


# ------------------------------------------------------------------------------------------ attention


SHAPES = [  # new, ctx, hq, hkv, d, page
    ([1], [1], 1, 1, 64, 64),
    ([1, 1, 1], [2, 63, 65], 2, 1, 64, 64),
    ([1, 1, 1, 1], [33, 700, 257, 0], 16, 8, 256, 64),
    ([1, 1], [2100, 129], 8, 2, 128, 128),
    ([5, 1, 3], [64, 300, 3], 3, 1, 128, 64),
    ([40, 1, 0, 17], [40, 600, 50, 1000], 4, 2, 256, 256),
    ([150, 33], [500, 33], 8, 8, 64, 64),
    ([3, 2], [1, 2], 8, 1, 128, 64),       # a sequence with more new tokens than slots: its first rows see nothing
    ([20], [9000], 16, 1, 64, 64),
]


@pytest.mark.parametrize("softcap,window", [(0.0, 0), (50.0, 0), (50.0, 70), (0.0, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(shape: int, dtype: str, softcap: float, window: int) -> None:
    import torch

    new, ctx, hq, hkv, d, page = SHAPES[shape]
    say(f"attention_kv4 new={new} ctx={ctx} hq={hq} hkv={hkv} d={d} page={page} {dtype} cap={softcap} window={window}")
    c = Case(17 * shape + d, new, ctx, hq, hkv, d, page, dtype)
    c.fill(shape)
    c.append()
    r = rng(shape)
    w = np.abs(r.normal(size=(len(new), hkv, max(ctx) + 3))).astype(np.float32)
    for b, (n, m) in enumerate(zip(new, ctx)):
        w[b, :, max(m - n, 0):m] = np.nan  # the newest slots' old weights are not read
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.full_like(w_in, -7.0)
    kw = dict(scale=d ** -0.5 * 2, softcap=softcap, window=window)
    plain = c.attend(**kw)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    assert torch.equal(plain, out), "weights change no output"
    c.check(out, w_out, w, **kw)
    for b, m in enumerate(ctx):
        assert (w_out[b, :, m:] == -7.0).all(), "slots behind the sequence were written"
    again = c.attend(weights=w_in, **kw)  # in place
    torch.cuda.synchronize()
    assert torch.equal(again, out)
    for b, m in enumerate(ctx):
        assert torch.equal(w_in[b, :, :m], w_out[b, :, :m])


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "f32"), (256, "bf16")])
def test_values_and_keys_that_are_nan_reach_only_rows_that_see_them(d: int, dtype: str) -> None:
    import torch

    new, ctx, hq, hkv = [20, 1], [90, 200], 4, 2
    say(f"attention_kv4 with NaN, d={d} {dtype}")
    c = Case(d, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(1)
    c.v[7, 33] = float("nan")   # token 7 of sequence 0: one block of one head
    c.v[15, 0] = float("inf")
    c.k[11, 5] = float("nan")
    c.append()
    out = c.attend(scale=0.2, softcap=50.0)
    torch.cuda.synchronize()
    got = out.float().cpu().numpy().reshape(-1, hq, d)
    assert np.isfinite(got[:7]).all() and np.isfinite(got[20]).all()
    assert np.isnan(got[7, 0, 32:64]).all() and np.isfinite(got[7, 0, :32]).all() and np.isfinite(got[7, 2:]).all()
    c.check(out, scale=0.2, softcap=50.0, window=0)


@pytest.mark.parametrize("softcap,window", [(0.0, 0), (50.0, 0), (0.0, 70), (50.0, 700)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,hkv,group", [(64, 2, 3), (128, 1, 8), (256, 2, 1)])
def test_many_rows(d: int, hkv: int, group: int, dtype: str, softcap: float, window: int) -> None:
    """Questions of many rows over states of a few spans, the last tiles of rows and keys half full, with NaN values in
    the middle and in the newest slots and with a query that is NaN, which its KV head's weights show."""
    import torch

    new, ctx, hq = [129, 70, 66], [1300, 70, 97], hkv * group
    say(f"attention_kv4 many rows d={d} hq={hq} hkv={hkv} {dtype} cap={softcap} window={window}")
    c = Case(40 + d, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(3)
    for token, col in ((0, 5), (63, d - 1), (128, 40), (129 + 69, 0)):
        c.v[token, col] = float("nan")
    c.q[129 + 69, 3] = float("nan")
    c.append()
    r = rng(d)
    w = np.abs(r.normal(size=(3, hkv, 1303))).astype(np.float32)
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.full_like(w_in, -7.0)
    kw = dict(scale=d ** -0.5 * 2, softcap=softcap, window=window)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    c.check(out, w_out, w, **kw)
    for b, m in enumerate(ctx):
        assert (w_out[b, :, m:] == -7).all()


def test_infinite_and_nan_queries_stay_in_their_rows() -> None:
    import torch

    say("attention_kv4 with NaN and infinite queries")
    c = Case(2, [4, 1], [100, 50], 4, 2, 128)
    c.fill(2)
    c.q[1, 5] = float("nan")
    c.q[2, 140] = float("inf")
    c.append()
    for cap in (0.0, 50.0):
        out = c.attend(scale=0.1, softcap=cap).float().cpu().numpy().reshape(5, 4, 128)
        assert np.isnan(out[1, 0]).all() and np.isfinite(out[1, 1:]).all()
        assert np.isfinite(out[0]).all() and np.isfinite(out[3:]).all() and np.isfinite(out[2, [0, 2, 3]]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_sequence_does_not_depend_on_its_batch(dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    new, ctx, hq, hkv, d = [1, 60, 7, 1], [3000, 400, 9000, 64], 8, 2, 128
    say(f"attention_kv4 alone and in a batch {dtype}")
    c = Case(9, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(4)
    c.append()
    w = torch.rand((4, hkv, max(ctx)), device="cuda")
    for window in (0, 500):
        kw = dict(num_q_heads=hq, scale=0.1, softcap=50.0, window=window)
        w_all = torch.empty_like(w)
        whole = K.attention_kv4(c.q, c.cache, c.d_table, c.d_starts, c.d_new, c.d_ctx, c.max_new, c.max_ctx, weights=w,
                                weights_out=w_all, **kw)
        for b, (n, m) in enumerate(zip(new, ctx)):
            rows = slice(c.starts[b], c.starts[b] + n)
            w_one = torch.empty((1, hkv, m), device="cuda")
            one = K.attention_kv4(c.q[rows], c.cache, c.d_table[b:b + 1].contiguous(), i32([0]), i32([n]), i32([m]), n, m,
                                  weights=w[b:b + 1], weights_out=w_one, **kw)
            torch.cuda.synchronize()
            assert torch.equal(one, whole[rows]), f"sequence {b} window {window}"
            assert torch.equal(w_one[0], w_all[b, :, :m])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new,ctx,hq,hkv,d", [([2, 1], [700, 90], 4, 2, 64), ([70, 3], [300, 100], 2, 1, 256)])
def test_scores_beyond_the_soft_cap(new: list[int], ctx: list[int], hq: int, hkv: int, d: int, dtype: str) -> None:
    """A cap that scores of 1.6 on average pass by far: both forms of the hyperbolic tangent, and the border of them."""
    import torch

    say(f"attention_kv4 beyond the soft-cap new={new} ctx={ctx} d={d} {dtype}")
    c = Case(12, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(7)
    c.append()
    kw = dict(scale=1.6 / d ** 0.5, softcap=1.5, window=0)
    w_in = np.zeros((2, hkv, max(ctx)), np.float32)
    w = torch.zeros(w_in.shape, device="cuda")
    out = c.attend(weights=w, **kw)
    torch.cuda.synchronize()
    c.check(out, w, w_in, **kw)


@pytest.mark.parametrize("n", [1, 70])
def test_a_large_soft_cap_is_none(n: int) -> None:
    """A cap of 1e6 moves scores of at most some 20 by 1e-9 of themselves, and the arithmetic by 8 u of them: weights by
    2 * 8 * 20 u = 2e-5 of themselves each, averages of values of at most 6 by twice that."""
    import torch

    say(f"attention_kv4 with a soft-cap of 1e6, {n} tokens")
    c = Case(17, [n], [700], 4, 2, 128, 64, "f32")
    c.fill(8)
    c.append()
    capped, plain = (c.attend(scale=0.1, softcap=cap) for cap in (1e6, 0.0))
    torch.cuda.synchronize()
    assert (capped - plain).abs().max().item() <= 2 * 2e-5 * 6


def alone(c: Case, b: int, w, **kw):
    """Output and weights of sequence b of a case in a call of its own."""
    import torch

    from deciax_amd import kernels as K

    n, m = c.new[b], c.ctx[b]
    rows = slice(c.starts[b], c.starts[b] + n)
    w_one = torch.empty((1, c.hkv, m), device="cuda")
    one = K.attention_kv4(c.q[rows], c.cache, c.d_table[b:b + 1].contiguous(), i32([0]), i32([n]), i32([m]), n, m,
                          num_q_heads=c.hq, weights=w[b:b + 1], weights_out=w_one, **kw)
    return one, w_one[0]


# 2048 and more spans of few rows (two a workgroup); more sequences of many rows than a wave has lanes, among others of few
# rows and none; more work items than workgroups
LARGE = [([1] * 96, [1100 + 7 * i for i in range(96)], 8, 8, 64),
         ([60 if i % 3 else i % 2 * 5 for i in range(70)], [64 + 9 * i for i in range(70)], 2, 2, 64),
         ([65] * 34, [4000 + 100 * i for i in range(34)], 8, 8, 64)]


@pytest.mark.parametrize("large", range(len(LARGE)))
def test_large_batches_are_their_sequences(large: int) -> None:
    import torch

    new, ctx, hq, hkv, d = LARGE[large]
    say(f"attention_kv4 of {len(new)} sequences, up to {max(new)} tokens over {max(ctx)} slots")
    c = Case(20 + large, new, ctx, hq, hkv, d, 64, garbage=False)
    codes = rng(large).integers(0, 256, c.raw["k"].shape).astype(np.uint8)
    c.cache.k.copy_(torch.from_numpy(codes))
    c.cache.v.copy_(torch.from_numpy(codes[::-1].copy()))
    for t in (c.cache.k_scale, c.cache.v_scale):
        t.fill_(126)
    c.append()
    kw = dict(scale=0.1, softcap=50.0, window=0)
    w = torch.rand((len(new), hkv, max(ctx)), device="cuda")
    w_all = torch.empty_like(w)
    whole = c.attend(weights=w, weights_out=w_all, **kw)
    torch.cuda.synchronize()
    for b in range(len(new)):
        if new[b] == 0:
            assert torch.equal(w_all[b, :, :ctx[b]], w[b, :, :ctx[b]])
            continue
        one, w_one = alone(c, b, w, **kw)
        torch.cuda.synchronize()
        assert torch.equal(one, whole[c.starts[b]:c.starts[b] + new[b]]), f"sequence {b}"
        assert torch.equal(w_one, w_all[b, :, :ctx[b]]), f"sequence {b}"


@pytest.mark.parametrize("n", [3, 40])
def test_rows_outside_the_packed_ones_add_no_weight(n: int) -> None:
    """The last token of a sequence lies behind the packed rows: the weights are those of the tokens before it. Both sums
    of at most R weights of the same scores are off by R 2^-24 of the sum."""
    import torch

    from deciax_amd import kernels as K

    say(f"attention_kv4 with a token outside the packed rows, {n} new")
    c = Case(15, [2, n], [64, 300], 4, 2, 64)
    c.fill(9)
    c.append()
    kw = dict(num_q_heads=4, scale=0.2)
    w = torch.rand((2, 2, 300), device="cuda")
    got, want = torch.empty_like(w), torch.empty((1, 2, 299), device="cuda")
    K.attention_kv4(c.q[:-1], c.cache, c.d_table, c.d_starts, c.d_new, c.d_ctx, n, 300, weights=w, weights_out=got, **kw)
    K.attention_kv4(c.q[2:-1], c.cache, c.d_table[1:].contiguous(), i32([0]), i32([n - 1]), i32([299]), n - 1, 299,
                    weights=w[1:], weights_out=want, **kw)
    torch.cuda.synchronize()
    assert (got[1, :, 299] == 0).all()
    assert ((got[1, :, :299] - want[0]).abs() <= 2 * 2 * n * U32 * want[0]).all()


def test_window_goes_by_positions_after_eviction_left_gaps() -> None:
    """Positions with gaps: fewer slots than the window spans are seen."""
    import torch

    say("attention_kv4 window over positions with gaps")
    c = Case(6, [2, 1], [300, 150], 4, 2, 64)
    c.fill(3)
    c.append()
    r = rng(0)
    for b, m in enumerate(c.ctx):
        for g in range(c.hkv):
            p = np.sort(r.choice(4 * m, m, replace=False))
            for j in range(m):
                c.pos[c.table[b, j // 64], g, j % 64] = p[j]
    c.cache.positions.copy_(torch.from_numpy(c.pos))
    for window in (1, 100, 100000):
        kw = dict(scale=0.2, softcap=0.0, window=window)
        w = torch.zeros((2, 2, 300), device="cuda")
        out = c.attend(weights=w, **kw)
        torch.cuda.synchronize()
        c.check(out, w, np.zeros((2, 2, 300), np.float32), **kw)


def test_other_streams_and_graph_replays() -> None:
    """A decoding step (append, attend with weights) on a side stream, and captured and replayed with other eager
    calls between the replays."""
    import torch

    say("kv4 step on a side stream and in a graph")
    c = Case(8, [1, 1, 1], [700, 65, 3000], 16, 8, 256)
    c.fill(5)
    kw = dict(scale=1 / 16, softcap=50.0)
    w0 = torch.rand((3, 8, 3000), device="cuda")
    w = w0.clone()
    c.append()
    want = c.attend(weights=w, **kw)
    torch.cuda.synchronize()
    w_want = w.clone()

    side = torch.cuda.Stream()
    w_side = w0.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.append()
        out_side = c.attend(weights=w_side, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out_side, want) and torch.equal(w_side, w_want)

    out = torch.empty_like(want)
    wg = w0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.append()
        c.attend(weights=wg, out=out, **kw)
    other = Case(11, [1, 1], [500, 20], 16, 8, 256)
    other.fill(6)
    for i in range(4):
        out.fill_(float("nan"))
        wg.copy_(w0)
        other.attend(**kw)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(wg, w_want), f"replay {i} differs"


def test_two_graphs_replayed_in_turn() -> None:
    """Graphs of two batches, each with workspace of its own, replayed in turn on one stream and on two."""
    import torch

    say("kv4 two graphs")
    kw = dict(scale=1 / 16, softcap=50.0)
    cases = [Case(8, [1, 20], [1700, 65], 8, 2, 128), Case(9, [1], [2500], 8, 2, 128)]
    graphs, outs, wants = [], [], []
    for i, c in enumerate(cases):
        c.fill(5 + i)
        c.append()
        wants.append(c.attend(**kw))
        outs.append(torch.empty_like(wants[i]))
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            c.attend(out=outs[i], **kw)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams if i % 2 else streams[:1] * 2, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1]), f"replay {i} differs"


def test_refused_tensors() -> None:
    import torch

    from deciax_amd import kernels as K

    say("kv4 refusals of tensors")
    c = Case(30, [1, 1], [70, 20], 4, 2, 64)
    kw = dict(num_q_heads=4, scale=0.1)
    w = torch.zeros((2, 2, 200), device="cuda")

    def attend(q=c.q, table=c.d_table, new=c.d_new, max_ctx=70, **more):
        K.attention_kv4(q, c.cache, table, c.d_starts, new, c.d_ctx, 1, max_ctx, **{**kw, **more})

    for bad in (lambda: attend(q=c.q.half()), lambda: attend(q=c.q.cpu()), lambda: attend(q=c.q[:, :128]),
                lambda: attend(table=c.d_table.long()), lambda: attend(table=c.d_table.cpu()),
                lambda: attend(table=c.d_table.t()), lambda: attend(new=c.d_new[:1]),
                lambda: attend(weights=w[..., :60]), lambda: attend(weights=w.double()), lambda: attend(weights=w[:1]),
                lambda: attend(weights=w[..., ::2]), lambda: attend(weights=w.expand(2, 2, 200)[:, :1].expand(2, 2, 200)),
                lambda: attend(weights=w[..., :100], weights_out=w[..., 50:150]), lambda: attend(weights_out=w),
                lambda: attend(weights=w.as_strided((2, 2, 70), (105, 70, 1))),
                lambda: attend(out=torch.empty_like(c.q, dtype=torch.float32)), lambda: attend(num_q_heads=3),
                lambda: K.kv4_evict(c.cache, w, c.d_table, c.d_ctx, 70, c.d_table, keep=10, weights_out=w[..., 100:110]),
                lambda: K.kv4_read(c.cache, c.d_table, c.d_starts, c.d_new, c.d_ctx, 1, rows=2, out_k=c.k.float()),
                lambda: K.kv4_append(c.cache, c.k, c.v, c.positions.long(), c.d_table, c.d_starts, c.d_new, c.d_ctx, 1),
                lambda: K.kv4_append(c.cache, c.k, c.v.float(), c.positions, c.d_table, c.d_starts, c.d_new, c.d_ctx, 1)):
        with pytest.raises(ValueError):
            bad()
    both = torch.zeros((2, 2, 2, 70), device="cuda")
    attend(weights=both[0], weights_out=both[1])  # one buffer's halves do not meet
    torch.cuda.synchronize()


def test_pages_beyond_32_bit_offsets() -> None:
    """A pool whose arrays pass 4 GiB: pages at its end are addressed in 64 bits."""
    import torch

    from deciax_amd import kernels as K

    say("kv4 pages beyond 4 GiB")
    hkv, d, page = 8, 256, 1024
    pages = (5 << 30) // (hkv * page * d // 2)
    cache = K.kv4_cache(pages, hkv, d, page_size=page)
    r = rng(4)
    n, m = 3, 1500
    x = torch.from_numpy(r.normal(size=(m, 3 * hkv * d)).astype(np.float32)).cuda().bfloat16()
    q, k, v = (x[:, i * hkv * d:(i + 1) * hkv * d] for i in range(3))
    pos = i32(np.arange(m))
    outs = []
    for table in ([0, 1], [pages - 1, pages - 2]):
        t = i32([table])
        K.kv4_append(cache, k, v, pos, t, i32([0]), i32([m]), i32([m]), m)
        outs.append(K.attention_kv4(q[:n], cache, t, i32([0]), i32([n]), i32([m]), n, m, num_q_heads=hkv, scale=1 / 16))
        got = K.kv4_read(cache, t, i32([0]), i32([m]), i32([m]), m, rows=m)
        outs.extend(got)
    torch.cuda.synchronize()
    for a, b in zip(outs[:3], outs[3:]):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------ eviction


@pytest.mark.parametrize("ctx,keep,recent,d,hkv,page", [
    ([1], 1, 0, 64, 1, 64), ([100, 64, 3, 0], 40, 8, 128, 2, 64), ([1000, 5000, 400], 400, 0, 64, 3, 64),
    ([2900], 1000, 1000, 256, 2, 128), ([20000, 17000], 4097, 100, 64, 1, 256), ([300], 299, 1, 64, 2, 64),
    ([70001], 30000, 500, 64, 1, 1024)])
def test_evict(ctx: list[int], keep: int, recent: int, d: int, hkv: int, page: int) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"kv4_evict ctx={ctx} keep={keep} recent={recent} d={d} hkv={hkv} page={page}")
    extra = sum(-(-keep // page) for _ in ctx)
    c = Case(keep, [0] * len(ctx), [*ctx], hkv, hkv, d, page)
    r = rng(keep)
    per = -(-keep // page)
    big = K.kv4_cache(c.pages + extra, hkv, d, page_size=page)
    for n in FIELDS:
        getattr(big, n)[:c.pages] = getattr(c.cache, n)
    c.cache = big
    out_table = c.pages + r.permutation(extra).reshape(len(ctx), per)
    w = np.exp(r.normal(size=(len(ctx), hkv, max(ctx) + 1)) * 3).astype(np.float32)
    w[r.random(w.shape) < 0.3] = 0.0          # many ties
    w[r.random(w.shape) < 0.1] = np.float32(0.5)
    if max(ctx) > 500:
        w[0, 0, 11], w[0, 0, 12], w[0, 0, 13] = np.nan, np.inf, -0.0
    w_dev = torch.from_numpy(w).cuda()
    before = c.host("k").copy()
    w_out, length = K.kv4_evict(c.cache, w_dev, c.d_table, c.d_ctx, max(ctx), i32(out_table), keep=keep, recent=recent)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(c.host("k")[:c.pages], before[:c.pages])
    assert length.cpu().tolist() == [min(n, keep) for n in ctx]
    for b, m in enumerate(ctx):
        n = min(m, keep)
        for g in range(hkv):
            slots = oracle.evict(w[b, g, :m], keep, recent)
            np.testing.assert_array_equal(w_out[b, g, :n].cpu().numpy(), w[b, g, slots])
            assert (w_out[b, g, n:] == 0).all()
            for name in ("k", "v", "k_scale", "v_scale", "positions"):
                a = c.host(name)
                src = a[c.table[b, slots // page], g, slots % page]
                j = np.arange(n)
                np.testing.assert_array_equal(a[out_table[b, j // page], g, j % page], src)


# ------------------------------------------------------------------------------------------ together


def test_a_state_is_kept_cut_and_answered_over() -> None:
    """Append a state, attend while weights accumulate, cut it, append and attend over what is left with a window, and
    score the answer's tokens: every stage against the oracle on the device's own data."""
    import torch

    from deciax_amd import kernels as K

    say("kv4: append, attend, evict, attend, score")
    hq, hkv, d, page, hidden, vocab = 4, 2, 128, 64, 512, 1024
    lengths = [400, 130]
    c = Case(21, lengths, [*lengths], hq, hkv, d, page)
    c.append()
    w = torch.zeros((2, hkv, 448), device="cuda")
    kw = dict(scale=0.1, softcap=50.0, window=0)
    out = c.attend(weights=w, **kw)
    torch.cuda.synchronize()
    c.check(out, w, np.zeros((2, hkv, 448), np.float32), **kw)

    keep = 100
    per = 3  # room for the answer behind what is kept
    big = K.kv4_cache(c.pages + 2 * per, hkv, d, page_size=page)
    for n in FIELDS:
        getattr(big, n)[:c.pages] = getattr(c.cache, n)
    old_w = w[:, :, :].cpu().numpy()
    c.cache = big
    table = c.pages + np.arange(2 * per).reshape(2, per)
    w2, length = K.kv4_evict(big, w, c.d_table, c.d_ctx, max(lengths), i32(table), keep=keep, recent=16)
    torch.cuda.synchronize()
    for b in range(2):
        for g in range(hkv):
            slots = oracle.evict(old_w[b, g, :lengths[b]], keep, 16)
            np.testing.assert_array_equal(c.held_positions(b, table, keep)[g], slots)

    n = 9  # the answer, positions going on from the state's
    a = Case(22, [n, n], [keep + n, keep + n], hq, hkv, d, page)
    a.cache, a.table, a.d_table, a.pages = big, table, i32(table), c.pages + 2 * per
    a.positions = i32(np.concatenate([np.arange(m, m + n) for m in lengths]))
    room = torch.zeros((2, hkv, keep + n), device="cuda")
    room[:, :, :keep] = w2
    a.append()
    kw = dict(scale=0.1, softcap=50.0, window=200)
    out = a.attend(weights=room, **kw)
    torch.cuda.synchronize()
    a.check(out, room, np.concatenate([w2.cpu().numpy(), np.zeros((2, hkv, n), np.float32)], 2), **kw)

    r = rng(3)
    table_w = torch.from_numpy((r.normal(size=(vocab, hidden)) * 0.5).astype(np.float32)).cuda().bfloat16()
    logits = K.linear(out, table_w, out_dtype=torch.float32)
    targets = i32(r.integers(0, vocab, 2 * n))
    lp, ent, ids, tops = K.token_logprobs(logits, targets, top=5, softcap=30.0)
    torch.cuda.synchronize()
    x, t = logits.cpu().numpy(), targets.cpu().numpy()
    for i in range(2 * n):
        want = oracle.token_logprobs(x[i], int(t[i]), 5, 30.0)
        assert abs(lp[i].item() - want[0]) < 1e-4 and abs(ent[i].item() - want[1]) < 1e-4
        assert ids[i].cpu().tolist() == want[2].tolist()


# ------------------------------------------------------------------------------------------ prompts

PROMPTS = [  # new, ctx, hq, hkv, d: more than 2048 rows of a KV head, whose keys are one span, beside sequences of several
    ([1100, 3, 400], [2111, 1300, 1000], 4, 2, 64),
    ([300], [700], 8, 1, 128),
    ([2, 1030], [600, 1100], 2, 1, 256),
]


@pytest.mark.parametrize("softcap,window", [(0.0, 0), (50.0, 700)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("prompt", range(len(PROMPTS)))
def test_prompts(prompt: int, dtype: str, softcap: float, window: int) -> None:
    import torch

    new, ctx, hq, hkv, d = PROMPTS[prompt]
    say(f"attention_kv4 prompts new={new} ctx={ctx} hq={hq} hkv={hkv} d={d} {dtype} cap={softcap} window={window}")
    c = Case(60 + prompt, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(prompt)
    c.append()
    w = np.abs(rng(prompt).normal(size=(len(new), hkv, max(ctx)))).astype(np.float32)
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.full_like(w_in, -7.0)
    kw = dict(scale=d ** -0.5 * 2, softcap=softcap, window=window)
    plain = c.attend(**kw)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    assert torch.equal(plain, out), "weights change no output"
    c.check(out, w_out, w, **kw)
    for b, m in enumerate(ctx):
        assert (w_out[b, :, m:] == -7.0).all(), "slots behind the sequence were written"


# ------------------------------------------------------------------------------------------ slots without a page


@pytest.mark.parametrize("ctx,keep,recent,page,gone", [
    ([1000, 300, 640, 100], 200, 64, 64, [(0, 3), (0, 14), (1, 0), (2, 8), (2, 9), (3, 1)]),  # old and recent slots
    ([300, 100, 64], 250, 250, 64, [(0, 2), (0, 3), (1, 0), (2, 0)]),  # no more than `keep` are left; none are
    ([20000], 4097, 100, 256, [(0, 7), (0, 78)]),
    ([70001, 500], 60000, 500, 1024, [(0, 0), (0, 68), (1, 0)]),
    ([40, 2000], 2000, 0, 64, [(1, 5)]),  # nothing is cut
])
def test_eviction_drops_slots_without_a_page(ctx: list[int], keep: int, recent: int, page: int, gone: list[tuple[int, int]]) -> None:
    """Slots whose page is outside the pool are not seen before an eviction and do not come back by it: they are not kept,
    however heavy or recent, where a used page would stand in for them."""
    import torch

    from deciax_amd import kernels as K

    hkv, d = 2, 64
    say(f"kv4_evict with missing pages ctx={ctx} keep={keep} recent={recent} page={page} gone={gone}")
    per = -(-keep // page)
    c = Case(keep + 1, [0] * len(ctx), [*ctx], hkv, hkv, d, page)
    r = rng(keep)
    extra = per * len(ctx)
    big = K.kv4_cache(c.pages + extra, hkv, d, page_size=page)
    for n in FIELDS:
        getattr(big, n)[:c.pages] = getattr(c.cache, n)
        getattr(big, n)[c.pages:] = 77  # what a used page holds
    c.cache = big
    out_table = c.pages + r.permutation(extra).reshape(len(ctx), per)
    for i, (b, p) in enumerate(gone):
        c.table[b, p] = (-1, c.pages + extra, -(1 << 31), (1 << 31) - 1)[i % 4]
    w = np.exp(r.normal(size=(len(ctx), hkv, max(ctx)))).astype(np.float32)
    for b, p in gone:
        w[b, :, p * page:(p + 1) * page] += 100.0  # heavier than all others
    w_out, length = K.kv4_evict(big, torch.from_numpy(w).cuda(), i32(c.table), c.d_ctx, max(ctx), i32(out_table), keep=keep,
                                recent=recent)
    torch.cuda.synchronize()
    for b, m in enumerate(ctx):
        slot = np.arange(m)
        there = slot[~np.isin(slot // page, [p for s, p in gone if s == b])]
        n = min(len(there), keep)
        assert length[b].item() == n
        for g in range(hkv):
            slots = there[oracle.evict(w[b, g, there], keep, int((there >= m - recent).sum()))]
            assert len(slots) == n
            np.testing.assert_array_equal(w_out[b, g, :n].cpu().numpy(), w[b, g, slots])
            assert (w_out[b, g, n:] == 0).all()
            j = np.arange(per * page)
            for name in FIELDS:
                a = c.host(name)
                new = a[out_table[b, j // page], g, j % page]
                np.testing.assert_array_equal(new[:n], a[c.table[b, slots // page], g, slots % page])
                assert (new[n:] == 77).all()


MISSING = [  # new, ctx, hq, hkv, d, pages that are not there: kept scores, few rows and many rows, spans that start or end in one
    ([2, 1], [1500, 300], 4, 2, 128, [(0, 3), (0, 8), (0, 9), (0, 20), (1, 0), (1, 1)]),
    ([20, 3], [1500, 64], 2, 1, 64, [(0, 0), (0, 11), (0, 22)]),
    ([20], [1100], 1, 1, 256, [(0, 0), (0, 8), (0, 9), (0, 15)]),
    ([150, 60], [1300, 200], 4, 2, 64, [(0, 1), (0, 10), (0, 17), (1, 0)]),
    ([100], [700], 2, 1, 256, [(0, 0), (0, 4), (0, 8)]),
    ([1200], [2000], 2, 1, 128, [(0, 0), (0, 7), (0, 11)]),
]


@pytest.mark.parametrize("softcap,window", [(0.0, 0), (50.0, 400)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("missing", range(len(MISSING)))
def test_slots_without_a_page_are_not_seen(missing: int, dtype: str, softcap: float, window: int,
                                           monkeypatch: pytest.MonkeyPatch) -> None:
    """Outputs and weights are those of the slots that have a page; weights of the others stay. The pool's first rows, which
    hold anything, NaN among it, never stand in for them. Without a window the newest tokens' last page is missing too."""
    import torch

    new, ctx, hq, hkv, d, gone = MISSING[missing]
    if window == 0:
        gone = [*gone, (0, (ctx[0] - 1) // 64)]
    say(f"attention_kv4 with missing pages new={new} ctx={ctx} hq={hq} hkv={hkv} d={d} gone={gone} {dtype} window={window}")
    c = Case(80 + missing, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(missing)
    c.append()
    table = c.table.copy()
    for i, (b, p) in enumerate(gone):
        table[b, p] = (-1, c.pages, (1 << 31) - 1, -(1 << 31))[i % 4]
    c.d_table = i32(table)
    w = np.abs(rng(missing).normal(size=(len(new), hkv, max(ctx)))).astype(np.float32)
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.full_like(w_in, -7.0)
    kw = dict(scale=d ** -0.5 * 2, softcap=softcap, window=window)
    plain = c.attend(**kw)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    assert torch.equal(plain, out), "weights change no output"

    sequences = iter(range(len(new)))

    def seen_only(q, k, v, positions, *, scale, softcap, window):
        b = next(sequences)
        n, slot = len(q), np.arange(ctx[b])
        there = ~np.isin(slot // 64, [p for s, p in gone if s == b])
        o, mass, weights = np.zeros(q.shape), np.zeros(q.shape), np.zeros((hkv, ctx[b]))
        for i in range(n):
            own = ctx[b] - n + i
            for h in range(hq):
                g = h // (hq // hkv)
                see = there & (slot <= own)
                if window > 0:
                    see &= (slot > own - window) & (positions[g] > positions[g][own] - window)
                if not see.any():
                    continue
                t = k[g][see] @ q[i, h] * scale
                t = softcap * np.tanh(t / softcap) if softcap else t
                p = np.exp(t - t.max())
                p /= p.sum()
                o[i, h], mass[i, h] = p @ v[g][see], p @ np.abs(v[g][see])
                weights[g][see] += p
        return o, weights, mass

    monkeypatch.setattr(oracle, "attention", seen_only)
    c.check(out, w_out, w, **kw)
    for b, m in enumerate(ctx):
        assert (w_out[b, :, m:] == -7.0).all(), "slots behind the sequence were written"
        for s, p in gone:
            if s == b and (p + 1) * 64 <= m - new[b]:
                assert torch.equal(w_out[b, :, p * 64:p * 64 + 64], w_in[b, :, p * 64:p * 64 + 64])


# the documents' examples of a kept state
STEPS = [pytest.param(block[len("python\n"):], id=doc.stem) for doc in sorted(ROOT.glob("*.md"))
         for block in doc.read_text().split("```") if block.startswith("python\n") and "kv4_evict(" in block]


@pytest.mark.parametrize("steps", STEPS)
def test_the_documented_steps_go_on_after_an_eviction(steps: str) -> None:
    """The documents' own lines on states of two lengths, then a further token over what they leave: the slots that it sees,
    their weights and their positions are those that were kept."""
    import torch

    say("kv4: documented steps")
    hq, hkv, d, keep, lengths = 4, 2, 64, 100, [400, 130]
    c = Case(50, lengths, [*lengths], hq, hkv, d)
    new_table = c.pages + np.arange(6).reshape(2, 3)  # a page of room
    x = torch.from_numpy(rng(1).normal(size=(c.rows, 128)).astype(np.float32)).cuda().bfloat16()
    w_qkv = torch.from_numpy(rng(2).normal(size=((hq + 2 * hkv) * d, 128)).astype(np.float32) / 12).cuda().bfloat16()
    angle = np.arange(500)[:, None] * 1e4 ** (-np.arange(d // 2) / (d // 2))
    logits = torch.from_numpy(rng(3).normal(size=(5, 1000)).astype(np.float32)).cuda()
    ns = dict(num_pages=c.pages + 6, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, num_seqs=2, max_ctx_len=400, k=c.k, v=c.v,
              q=c.q, positions=c.positions, page_table=c.d_table, seq_start=c.d_starts, seq_len=c.d_new, ctx_len=c.d_ctx,
              max_seq_len=400, new_table=i32(new_table), keep=keep, recent=16, logits=logits, answers=i32([1, 2, 3, 4, 5]),
              x=x, w_qkv=w_qkv, cos=torch.from_numpy(np.cos(angle)).cuda().bfloat16(),
              sin=torch.from_numpy(np.sin(angle)).cuda().bfloat16(), kept_start=i32([0, keep]))
    exec(steps, ns)
    torch.cuda.synchronize()
    assert ns["kept_len"].cpu().tolist() == [keep, keep]

    # a further token
    a = Case(51, [1, 1], [keep + 1, keep + 1], hq, hkv, d)
    a.cache, a.table, a.d_table = ns["cache"], new_table, ns["page_table"]
    a.positions = i32(lengths)
    a.append()
    before = ns["weights"].cpu().numpy().copy()
    kw = dict(scale=1 / 16, softcap=50.0, window=200)
    out = a.attend(weights=ns["weights"], **kw)
    torch.cuda.synchronize()
    a.check(out, ns["weights"], before, **kw)
    assert (before[:, :, :keep] > 0).any() and (before[:, :, keep:] == 0).all()
    for b, n in enumerate(lengths):
        held = a.held_positions(b)
        assert (held[:, keep] == n).all() and (np.diff(held, axis=1) > 0).all()
        assert (held[:, keep - 16:keep] == np.arange(n - 16, n)).all()


@pytest.mark.parametrize("dtype,softcap,window", [("bf16", 50.0, 0), ("f32", 0.0, 0), ("bf16", 0.0, 120000)])
@pytest.mark.parametrize("new,ctx,hq,page", [([2, 1], [150000, 700], 2, 64), ([40], [140001], 1, 64), ([1030], [5000], 2, 64),
                                             ([1, 70], [70000, 300], 2, 65536)])
def test_spans_of_more_pages_than_a_wave_has_lanes(new: list[int], ctx: list[int], hq: int, page: int, dtype: str,
                                                   softcap: float, window: int) -> None:
    """A span's pages are looked up 64 at a time: spans of 65 and more, and pages of 65536 slots."""
    import torch

    say(f"attention_kv4 of long spans new={new} ctx={ctx} page={page} {dtype} cap={softcap} window={window}")
    c = Case(90 + hq, new, ctx, hq, 1, 64, page, dtype)
    c.fill(5)
    c.append()
    w = np.abs(rng(4).normal(size=(len(new), 1, max(ctx)))).astype(np.float32)
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.empty_like(w_in)
    kw = dict(scale=1 / 8, softcap=softcap, window=window)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    c.check(out, w_out, w, **kw)


@pytest.mark.parametrize("large", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_batches_against_the_oracle(large: int, dtype: str) -> None:
    import torch

    new, ctx, hq, hkv, d = LARGE[large]
    say(f"attention_kv4 of {len(new)} sequences against the oracle, {dtype}")
    c = Case(70 + large, new, ctx, hq, hkv, d, 64, dtype)
    c.fill(large)
    c.append()
    w = np.abs(rng(large).normal(size=(len(new), hkv, max(ctx)))).astype(np.float32)
    w_in = torch.from_numpy(w.copy()).cuda()
    w_out = torch.empty_like(w_in)
    kw = dict(scale=1 / 8, softcap=50.0, window=0)
    out = c.attend(weights=w_in, weights_out=w_out, **kw)
    torch.cuda.synchronize()
    c.check(out, w_out, w, **kw)
