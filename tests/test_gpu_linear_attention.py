"""`kernels.linear_attention` on the GPU against the 64-bit oracle.

Tolerance (u = 2^-24), relative to the same recurrence of absolute values (`mass`): a product over k_dim and one over a
chunk's tokens in sequence, decays off by the rounding of their exponent (up to 88 u, where they are worth anything) and of
the exponential, the state multiplied and added to once a chunk: 2 (k_dim + 64) + 128 + 4 chunks, times u. bf16 rows, in
chunks: the weights of a chunk's tokens, and the state that a query multiplies, as two bf16 parts: 2^-16 of the mass; the
result rounded once, 2^-8 of itself.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import token_layer as oracle
from tests.conftest import bf16_np, i32, rng, say, to_dev, to_np

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Case:
    """Packed sequences of some lengths with rows of no sequence between them, states in another order than theirs."""

    def __init__(self, seed: int, lengths, hk: int, h: int, dk: int, dv: int, dtype: str, constant: bool = False) -> None:
        r = rng(seed)
        self.lengths, self.hk, self.h, self.dk, self.dv, self.dtype = list(lengths), hk, h, dk, dv, dtype
        cast = bf16_np if dtype == "bf16" else (lambda t: np.asarray(t, np.float32))
        order = r.permutation(len(lengths))
        self.starts, at = np.zeros(len(lengths), np.int64), 2
        for b in order:
            self.starts[b] = at
            at += lengths[b] + int(r.integers(0, 3))
        self.rows = at + 1
        self.q, self.k = (cast(r.normal(size=(self.rows, hk, dk)) / s) for s in (1.0, dk ** 0.5))
        self.v = cast(r.normal(size=(self.rows, h, dv)))
        rate = np.exp(r.uniform(np.log(1e-4), np.log(3.0), h))
        self.decay = (-rate * np.ones((self.rows, 1)) if constant else -rate * r.random((self.rows, h)) * 2).astype(np.float32)
        self.slots = len(lengths) + 2
        self.index = r.permutation(self.slots)[:len(lengths)]
        self.state = (r.normal(size=(self.slots, h, dk, dv)) * 0.3).astype(np.float32)
        self.scale = dk ** -0.5

    def run(self, rows=None, states=None, **kw):
        """(out, state_out) for all sequences, or some."""
        import torch

        from deciax_amd import kernels as K

        some = list(range(len(self.lengths))) if rows is None else rows
        pad = 4 if self.dtype == "f32" else 8
        qkv = np.concatenate([self.q.reshape(self.rows, -1), self.k.reshape(self.rows, -1), self.v.reshape(self.rows, -1),
                              np.full((self.rows, pad), np.nan, np.float32)], 1)
        x = to_dev(qkv, self.dtype)
        w = self.hk * self.dk
        state = torch.from_numpy(self.state).cuda() if states is None else states
        out = torch.full((self.rows, self.h * self.dv + pad), 9.0, dtype=x.dtype, device="cuda")
        kw = dict(state_out=torch.full_like(state, 4.0)) | kw
        lengths = [self.lengths[b] for b in some]
        K.linear_attention(x[:, :w], x[:, w:2 * w], x[:, 2 * w:-pad], torch.from_numpy(self.decay).cuda(), state,
                           i32(self.starts[some]), i32(lengths), max(lengths, default=0), num_k_heads=self.hk,
                           num_heads=self.h, k_dim=self.dk, v_dim=self.dv, scale=self.scale, out=out,
                           state_index=i32(self.index[some]), **kw)
        torch.cuda.synchronize()
        self.out = out
        kept = kw["state_out"] if kw["state_out"] is not None else state
        return to_np(out), to_np(kept)

    def check(self, out: np.ndarray, state: np.ndarray, untouched: float = 4.0) -> None:
        seen = np.zeros(self.rows, bool)
        width = self.h * self.dv
        for b, n in enumerate(self.lengths):
            rows = slice(self.starts[b], self.starts[b] + n)
            seen[rows] = True
            args = [t[rows] for t in (self.q, self.k, self.v, self.decay)]
            want, end = oracle.linear_attention(*args, self.state[self.index[b]], self.scale)
            mass, most = oracle.linear_attention(np.abs(args[0]), np.abs(args[1]), np.abs(args[2]), args[3],
                                                 np.abs(self.state[self.index[b]]), self.scale)
            steps = (2 * (self.dk + 64) + 128 + 4 * (n // 16 + 1)) * U
            tol = (steps + (2.0 ** -16 if self.dtype == "bf16" else 0.0)) * mass
            tol = tol + (2.0 ** -8 if self.dtype == "bf16" else U) * np.abs(want)
            off = np.abs(out[rows, :width].reshape(want.shape) - want)
            assert (off <= tol).all(), (b, n, float((off / np.maximum(tol, 1e-300)).max()))
            off = np.abs(state[self.index[b]] - end)
            assert (off <= steps * most).all(), (b, n, float((off / (steps * most + 1e-300)).max()))
            # errors of random signs are far smaller than the bound
            assert np.linalg.norm(off) <= 1e-6 * np.linalg.norm(end), (b, n, np.linalg.norm(off) / np.linalg.norm(end))
        assert (out[~seen] == 9).all() and (out[:, width:] == 9).all()
        others = np.setdiff1d(np.arange(self.slots), self.index)
        assert (state[others] == untouched).all() if untouched is not None else True


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,hk,h,dk,dv", [
    ([1], 1, 1, 64, 64), ([0, 1, 2], 2, 4, 128, 64), ([16, 3, 0, 9], 1, 3, 256, 128), ([17], 2, 2, 64, 256),
    ([1, 31, 32, 33, 5], 2, 4, 128, 128), ([63, 64, 65, 0, 15, 16], 1, 2, 64, 128), ([127, 200], 3, 3, 128, 64),
    ([100, 257], 1, 1, 256, 256), ([511, 512], 1, 2, 64, 64)])
def test_against_the_oracle(lengths, hk: int, h: int, dk: int, dv: int, dtype: str) -> None:
    say(f"linear_attention {lengths} {hk}/{h} {dk}x{dv} {dtype}")
    c = Case(sum(lengths) + dk, lengths, hk, h, dk, dv, dtype)
    c.check(*c.run())


@pytest.mark.parametrize("constant", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,dk,dv", [([513, 2, 700], 128, 64), ([1025, 4097, 33], 64, 64), ([2111], 256, 64)])
def test_long_sequences(lengths, dk: int, dv: int, dtype: str, constant: bool) -> None:
    """Sequences of several segments; decays that are the same for every token, whose errors would add up."""
    say(f"linear_attention long {lengths} {dk}x{dv} {dtype} constant={constant}")
    c = Case(len(lengths) + dk, lengths, 1, 2, dk, dv, dtype, constant)
    c.check(*c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_in_place_and_state_out_give_the_same(dtype: str) -> None:
    import torch

    say(f"linear_attention in place {dtype}")
    c = Case(5, [600, 1, 40, 0, 1300], 1, 2, 64, 128, dtype)
    out, state = c.run()
    c.check(out, state)
    mine = torch.from_numpy(c.state).cuda()
    out2, state2 = c.run(states=mine, state_out=None)
    assert np.array_equal(out, out2)
    assert np.array_equal(state2[c.index], state[c.index])
    others = np.setdiff1d(np.arange(c.slots), c.index)
    assert np.array_equal(state2[others], c.state[others])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_results_do_not_depend_on_the_batch(dtype: str) -> None:
    say(f"linear_attention alone and in a batch {dtype}")
    c = Case(6, [1, 900, 16, 17, 64, 0, 3000, 513], 2, 4, 64, 64, dtype)
    out, state = c.run()
    for b, n in enumerate(c.lengths):
        one, s = c.run(rows=[b])
        rows = slice(c.starts[b], c.starts[b] + n)
        assert np.array_equal(one[rows], out[rows]) and np.array_equal(s[c.index[b]], state[c.index[b]]), n


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_then_steps_is_the_whole(dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"linear_attention prompt and steps {dtype}")
    n, first = 150, 131
    c = Case(7, [n], 1, 2, 128, 64, dtype)
    want, end = c.run()
    rows = slice(c.starts[0], c.starts[0] + n)
    x = [to_dev(t[rows].reshape(n, -1), dtype) for t in (c.q, c.k, c.v)]
    g, state = torch.from_numpy(c.decay[rows]).cuda(), torch.from_numpy(c.state[c.index]).cuda()
    outs = []
    for a, b in [(0, first)] + [(t, t + 1) for t in range(first, n)]:
        outs.append(K.linear_attention(*(t[a:b] for t in x), g[a:b], state, i32([0]), i32([b - a]), b - a, num_k_heads=1,
                                       num_heads=2, k_dim=128, v_dim=64, scale=c.scale))
    got = to_np(torch.cat(outs)).reshape(n, -1)
    mass, most = oracle.linear_attention(*(np.abs(t[rows]) for t in (c.q, c.k, c.v)), c.decay[rows],
                                         np.abs(c.state[c.index[0]]), c.scale)
    steps = 2 * (2 * (128 + 64) + 128 + 4 * n) * U
    loose = (steps + (2.0 ** -15 if dtype == "bf16" else 0)) * mass.reshape(n, -1)
    loose = loose + (2.0 ** -7 if dtype == "bf16" else 0) * np.abs(want[rows, :128])
    assert (np.abs(got - want[rows, :128]) <= loose).all()
    assert (np.abs(to_np(state)[0] - end[c.index[0]]) <= steps * most).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths", [[8], [200], [1100]])
def test_forgetting(lengths, dtype: str) -> None:
    """Decays of nothing, of everything (-inf, the type's lowest value) and far below what exp holds."""
    say(f"linear_attention resets {lengths} {dtype}")
    c = Case(8, lengths, 1, 3, 64, 64, dtype)
    n = c.rows
    c.decay[:, 0] = 0.0
    c.decay[::5, 1] = -np.inf
    c.decay[1::7, 1] = np.finfo(np.float32).min
    c.decay[:, 2] = -np.where(np.arange(n) % 3 == 0, 300.0, 1e-3)
    c.check(*c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("at", [0, 5, 40, 63, 64, 100, 700])
def test_lost_values_reach_later_tokens_only(at: int, dtype: str) -> None:
    say(f"linear_attention NaN and infinity at {at} {dtype}")
    for what in ("q", "k", "v", "decay"):
        for bad in (np.nan, np.inf):
            c = Case(9, [at + 30, 12], 1, 2, 64, 64, dtype)
            clean, clean_state = c.run()
            row = c.starts[0] + at
            t = getattr(c, what)
            if what == "decay":
                if bad == np.inf:
                    continue
                t[row, 1] = bad
            else:
                t[row, 0, 3] = bad
            out, state = c.run()
            head = slice(0, 64) if what == "v" else slice(64, 128) if what == "decay" else slice(0, 128)
            before, after = slice(c.starts[0], row), slice(row, c.starts[0] + at + 30)
            # another order of the chunk's sums at most: far fewer than the bound's roundings
            near = (2.0 ** -7 if dtype == "bf16" else 2.0 ** -18) * np.abs(clean[before]).max(initial=0.0)
            assert (np.abs(out[before] - clean[before]) <= near).all(), (what, bad)
            hit = ~np.isfinite(out[after, head])
            if what == "q":
                assert hit[0].all() and not hit[1:].any()
                assert np.array_equal(state, clean_state)
            elif what == "v":
                assert hit[:, 3].all() and not np.delete(hit, 3, 1).any(), (what, bad)
            else:
                assert hit.all()
            other = np.ones(128, bool)
            other[head] = False
            assert np.array_equal(out[after, :128][:, other], clean[after, :128][:, other])
            second = slice(c.starts[1], c.starts[1] + 12)
            assert np.array_equal(out[second], clean[second])


def test_bad_rows_and_states_are_not_touched() -> None:
    """Sequences that reach outside the packed rows have no tokens; indices outside start from zeros and keep nothing."""
    import torch

    from deciax_amd import kernels as K

    say("linear_attention malformed sequences")
    r = rng(10)
    rows, h, d = 50, 2, 64
    for n in (10, 40):
        x = [to_dev(r.normal(size=(rows, h * d)).astype(np.float32), "f32") for _ in range(3)]
        g = torch.from_numpy(-r.random((rows, h)).astype(np.float32)).cuda()
        state = torch.from_numpy(r.normal(size=(5, h, d, d)).astype(np.float32)).cuda()
        kept, out = torch.full_like(state, 4.0), torch.full((rows, h * d), 9.0, device="cuda")
        starts, lengths, index = [-1, rows - n + 1, 0, 2 ** 31 - 5, 0], [n, n, n, n, -7], [0, 1, 77, 2, 4]
        kw = dict(num_k_heads=h, num_heads=h, k_dim=d, v_dim=d, scale=0.125)
        K.linear_attention(*x, g, state, i32(starts), i32(lengths), n, state_index=i32(index), state_out=kept, out=out, **kw)
        torch.cuda.synchronize()
        assert (out[n:] == 9).all() and (kept[3] == 4).all()
        for b in (0, 1, 2, 4):
            assert torch.equal(kept[b], state[b])  # no tokens: as they were
        want, _ = oracle.linear_attention(*(to_np(t)[:n].reshape(n, h, d) for t in x), to_np(g)[:n], np.zeros((h, d, d)), 0.125)
        mass, _ = oracle.linear_attention(*(np.abs(to_np(t)[:n].reshape(n, h, d)) for t in x), to_np(g)[:n],
                                          np.zeros((h, d, d)), 0.125)
        assert (np.abs(to_np(out)[:n].reshape(n, h, d) - want) <= 600 * U * mass).all()
        longer = K.linear_attention(*x, g, state, i32([0]), i32([rows]), n, state_out=kept, **kw)  # cut to max_seq_len
        cut = K.linear_attention(*x, g, state, i32([0]), i32([n]), n, state_out=kept, **kw)
        assert torch.equal(longer[:n], cut[:n])


def test_streams_and_graphs() -> None:
    import torch

    from deciax_amd import kernels as K

    say("linear_attention on a side stream, in a graph")
    r = rng(11)
    lengths, h, d = [1300, 1, 20], 2, 64
    rows = sum(lengths)
    x = [to_dev(bf16_np(r.normal(size=(rows, h * d)))) for _ in range(3)]
    g = torch.from_numpy(-r.random((1, h)).astype(np.float32)).cuda().expand(rows, h)  # one row for all tokens
    state = torch.from_numpy(r.normal(size=(3, h, d, d)).astype(np.float32)).cuda()
    args = (i32([0, 1300, 1301]), i32(lengths), 1300)
    kw = dict(num_k_heads=h, num_heads=h, k_dim=d, v_dim=d, scale=0.125)
    kept = torch.empty_like(state)

    def call(keep=kept):
        return K.linear_attention(*x, g, state, *args, state_out=keep, **kw)

    want = call().clone()
    end = kept.clone()
    same = K.linear_attention(*x, g.contiguous(), state, *args, state_out=kept, **kw)
    assert torch.equal(same, want) and torch.equal(kept, end)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(kept, end)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, their replays in turn
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call())
    for i in range(6):
        outs[i % 2].fill_(3)
        kept.fill_(5)
        call(torch.empty_like(state))
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want) and torch.equal(kept, end)


def test_refusals() -> None:
    import torch

    from deciax_amd import kernels as K

    q = torch.zeros((8, 128), device="cuda")
    v = torch.zeros((8, 256), device="cuda")
    g, s = torch.zeros((8, 4), device="cuda"), torch.zeros((3, 4, 64, 64), device="cuda")

    def call(q=q, k=q.clone(), v=v, g=g, s=s, starts=i32([0, 4]), lengths=i32([4, 4]), most=4, hk=2, h=4, dk=64, dv=64,
             scale=0.1, **kw):
        return K.linear_attention(q, k, v, g, s, starts, lengths, most, num_k_heads=hk, num_heads=h, k_dim=dk, v_dim=dv,
                                  scale=scale, **kw)

    call()
    for bad in (dict(hk=3), dict(h=0), dict(dk=32), dict(dv=128), dict(q=q.half()), dict(k=q.bfloat16()), dict(k=q[:7]),
                dict(q=q[0]), dict(v=v[:, :128]), dict(g=g.double()), dict(g=g[:, :3]), dict(g=g.T.contiguous().T),
                dict(s=s.bfloat16()), dict(s=s[:1]), dict(s=s[:, :2]), dict(s=s.transpose(2, 3)), dict(starts=i32([0])),
                dict(lengths=i32([4, 4]).long()), dict(state_index=i32([0])), dict(scale=0.0), dict(scale=float("nan")),
                dict(state_out=s[:2]), dict(out=q), dict(out=torch.empty((8, 100), device="cuda")), dict(out=v),
                dict(out=torch.empty((8, 256), dtype=torch.bfloat16, device="cuda")), dict(most=-1),
                dict(q=q[:1].expand(8, 128)), dict(k=torch.zeros((8, 130), device="cuda")[:, 1:129])):
        with pytest.raises(ValueError):
            call(**bad)
    big = torch.zeros((5, 4, 64, 64), device="cuda")
    with pytest.raises(ValueError, match="state_out"):
        call(s=big[:3], state_out=big[1:4])
    assert call(starts=i32([]), lengths=i32([]), s=s[:0], most=0).shape == (8, 256)
    assert call(q=q[:0], k=q[:0], v=v[:0], g=g[:0], lengths=i32([0, 0])).shape == (0, 256)


@pytest.mark.parametrize("dk,dv,h", [(64, 128, 4), (128, 128, 4), (256, 128, 3), (128, 256, 2), (256, 256, 2)])
def test_large_batches_are_their_sequences(dk: int, dv: int, h: int) -> None:
    """Workgroups of twice the columns, where a batch has more of them than there are CUs: the same results to the bit."""
    say(f"linear_attention in a batch of many heads {dk} x {dv}")
    lengths = [1, 5, 6, 7, 40, 64, 65, 0, 769, 130] + [17 + b % 40 for b in range(256 * 64 // (h * dv))]
    c = Case(12, lengths, 1, h, dk, dv, "bf16")
    assert h * dv // 64 * len(lengths) > 256
    out, state = c.run()
    for b, n in enumerate(lengths[:12]):
        one, s = c.run(rows=[b])
        rows = slice(c.starts[b], c.starts[b] + n)
        assert np.array_equal(one[rows], out[rows]) and np.array_equal(s[c.index[b]], state[c.index[b]]), n
    small = Case(13, [7, 8, 9, 16, 769, 1041], 1, h, dk, dv, "bf16")
    small.check(*small.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lengths_around_a_rule(dtype: str) -> None:
    say(f"linear_attention lengths around the rules {dtype}")
    c = Case(14, [4, 5, 6, 7, 8, 9, 10, 767, 768, 769, 832, 961, 1024], 1, 1, 64, 64, dtype)
    c.check(*c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("rate", [0.0, 1e-3, 0.08, 1.0])
def test_largest_values_stay_finite(rate: float, dk: int, dv: int, dtype: str) -> None:
    """Values up to bf16's largest number, keys so small that the states and all sums stay below 2^-4 of fp32's range: what
    is finite token by token is finite in chunks and segments, whatever the state has been scaled by in between."""
    say(f"linear_attention largest values, rate {rate}, {dk} x {dv} {dtype}")
    c = Case(15, [3, 40, 64, 65, 200, 900], 1, 2, dk, dv, dtype)
    most = float.fromhex("0x1.fep127")
    c.v = np.where(np.abs(c.v) > 0.5, np.sign(c.v) * most, bf16_np(c.v.clip(-1, 1) * 2.0 ** 126)).astype(np.float32)
    c.k = bf16_np(c.k * 2.0 ** -20)
    c.state = (c.state * 2.0 ** 108).astype(np.float32)
    c.decay = (-rate * np.ones_like(c.decay)).astype(np.float32)
    out, state = c.run()
    assert np.isfinite(out[:, :2 * dv]).all() and np.isfinite(state).all()
    c.check(out, state)


def test_states_between_the_rows() -> None:
    """States may lie in the same stretch of memory as the rows, but not on one of them, nor on the decays."""
    import torch

    from deciax_amd import kernels as K

    say("linear_attention states between rows")
    r = rng(16)
    n, d = 40, 64
    room = torch.zeros((n, 3 * d + d * d), device="cuda")
    room[:, :3 * d] = torch.from_numpy(r.normal(size=(n, 3 * d)).astype(np.float32))
    q, k, v = room[:, :3 * d].split(d, 1)
    g = torch.from_numpy(-r.random((n, 1)).astype(np.float32)).cuda()
    kw = dict(num_k_heads=1, num_heads=1, k_dim=d, v_dim=d, scale=0.125)
    args = (i32([0]), i32([n]), n)
    want_state = torch.zeros((1, 1, d, d), device="cuda")
    want = K.linear_attention(q, k, v, g, want_state, *args, **kw)
    state = room[7, 3 * d:].view(1, 1, d, d)  # behind the seventh row's values, in front of the eighth's
    before = room[:, :3 * d].clone()
    got = K.linear_attention(q, k, v, g, state, *args, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(state, want_state) and torch.equal(room[:, :3 * d], before)
    flat = room.view(-1)
    for at in (7 * room.shape[1] + 3 * d - 4, 7 * room.shape[1] + 3 * d + 4, 0):
        with pytest.raises(ValueError, match="meet"):
            K.linear_attention(q, k, v, g, flat[at:at + d * d].view(1, 1, d, d), *args, **kw)
    rows = torch.zeros((1, 1, d, d), device="cuda")
    with pytest.raises(ValueError, match="meet"):
        K.linear_attention(q, k, v, rows.view(-1, 1)[:n], rows, *args, **kw)
    assert torch.equal(room[:, :3 * d], before)


@pytest.mark.parametrize("most", [-1, 2 ** 31, 2 ** 32 + 5, 2 ** 40])
def test_bounds_that_the_c_entry_cannot_hold_are_refused(most: int) -> None:
    import torch

    from deciax_amd import kernels as K

    x, g, s = torch.zeros((8, 64), device="cuda"), torch.zeros((8, 1), device="cuda"), torch.zeros((1, 1, 64, 64), device="cuda")
    with pytest.raises(ValueError, match="max_seq_len"):
        K.linear_attention(x, x, x, g, s, i32([0]), i32([8]), most, num_k_heads=1, num_heads=1, k_dim=64, v_dim=64, scale=0.1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_small_values_keep_their_precision(dtype: str) -> None:
    """Values around 2^-100 beside large keys: the parts that they are split into are numbers of full precision still."""
    say(f"linear_attention small values {dtype}")
    c = Case(17, [5, 64, 200, 900], 1, 2, 64, 128, dtype)
    c.v = np.sign(c.v) * bf16_np((np.abs(c.v) + 1) * 2.0 ** -100)
    c.k = bf16_np(c.k * 2.0 ** 50)
    c.state = (c.state * 2.0 ** -50).astype(np.float32)
    c.check(*c.run())
