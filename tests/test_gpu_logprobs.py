"""`kernels.token_logprobs` on the GPU against the 64-bit oracle.

Tolerance (u = 2^-24): with a soft-cap a capped logit is off by at most 6 u cap on the way (product, exponential,
reciprocal, scale), without one the difference to the largest by u |x| and its conversion to base 2 by as much; a sum of
positive terms by its depth, 32 + 6 + 8 + 2 + chunk joins < 96; the logarithm and the last difference by u of their size.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv4 as oracle
from tests.conftest import i32, rng, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(x: np.ndarray, targets: np.ndarray, top: int, cap: float, got, size: float | None = None) -> None:
    lp, ent, ids, tops = (t.cpu().numpy().astype(np.float64) for t in got)
    for i in range(len(x)):
        want = oracle.token_logprobs(x[i], int(targets[i]), top, cap)
        finite = np.abs(x[i][np.isfinite(x[i])])
        tol = 2 * (12 * (size or cap or finite.max(initial=1.0)) + 96 + 8) * U
        for g, w, what in ((lp[i], want[0], "log probability"), (ent[i], want[1], "entropy")):
            assert np.isnan(g) == np.isnan(w) and np.isinf(g) == np.isinf(w), (i, what, g, w)
            if np.isfinite(w):
                scale = 1 + abs(want[1]) if what == "entropy" else 1.0
                assert abs(g - w) <= tol * scale + 4 * U * abs(w), (i, what, g, w, tol)
        assert ids[i].tolist() == want[2].tolist(), (i, ids[i], want[2])
        t = want[3]
        assert (np.isnan(tops[i]) == np.isnan(t)).all() and (np.isneginf(tops[i]) == np.isneginf(t)).all()
        f = np.isfinite(t)
        assert (np.abs(tops[i][f] - t[f]) <= tol + 4 * U * np.abs(t[f])).all(), (i, tops[i], t)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 31, 31), (2, 64, 64), (5, 2047, 3), (4, 2048, 0),
                                            (3, 2049, 1), (2, 32001, 20), (2, 50257, 64), (1, 256000, 8)])
def test_logprobs(rows: int, vocab: int, top: int, cap: float, dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs rows={rows} vocab={vocab} top={top} cap={cap} {dtype}")
    r = rng(vocab + rows)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    buf = torch.full((rows, vocab + 5), 77.0, device="cuda", dtype=t)  # rows of an odd stride, larger values beside them
    x = torch.from_numpy((r.normal(size=(rows, vocab)) * 4).astype(np.float32)).cuda().to(t)
    logits = buf[:, 1:vocab + 1]
    logits.copy_(x)
    targets = r.integers(0, vocab, rows)
    targets[0] = vocab - 1
    got = K.token_logprobs(logits, i32(targets), top=top, softcap=cap)
    torch.cuda.synchronize()
    check(x.float().cpu().numpy(), targets, top, cap, got)


@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_masks_ties_and_lost_rows(cap: float) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs special rows cap={cap}")
    vocab, top = 5000, 6
    r = rng(1)
    x = r.normal(size=(12, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, 4321] = -29.0                    # one token left
    x[2, :4990] = -np.inf
    x[3] = 1.5                            # all equal: the lowest tokens
    x[4, 2500] = np.nan
    x[5, 7] = np.inf
    x[6] = np.float32(torch.finfo(torch.float32).min)
    x[7] = np.arange(vocab) * 1e-3        # rising: every group is better than the last
    x[8] = -0.0
    x[8, 1::2] = 0.0                      # the two zeros are equal
    x[9] = 1e30
    x[9, 100:] = -1e30
    x[10] = np.where(np.arange(vocab) % 7 == 3, 2.0, 1.0)
    targets = np.array([5, 4321, 3, 4999, 1, 7, 0, 4999, 2, 50, -1, 10])
    got = K.token_logprobs(torch.from_numpy(x).cuda(), i32(targets), top=top, softcap=cap)
    torch.cuda.synchronize()
    # rows of huge logits without a cap: differences of 2e30 underflow to weight 0, the rest are exact
    check(x, targets, top, cap, got)
    bad = K.token_logprobs(torch.from_numpy(x[10:]).cuda(), i32([vocab, -2]), top=0, softcap=cap)
    assert torch.isnan(bad[0]).all() and torch.isfinite(bad[1]).all()


def test_rows_do_not_depend_on_the_batch_and_streams_and_graphs() -> None:
    import torch

    from deciax_amd import kernels as K

    say("token_logprobs alone, on a side stream, in a graph")
    r = rng(2)
    x = torch.from_numpy((r.normal(size=(70, 32001)) * 3).astype(np.float32)).cuda()
    targets = i32(r.integers(0, 32001, 70))
    want = K.token_logprobs(x, targets, top=7, softcap=30.0)
    torch.cuda.synchronize()
    for i in (0, 33, 69):
        one = K.token_logprobs(x[i:i + 1], targets[i:i + 1], top=7, softcap=30.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a[0], b[i]) for a, b in zip(one, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.token_logprobs(x, targets, top=7, softcap=30.0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = K.token_logprobs(x, targets, top=7, softcap=30.0)
    for _ in range(4):
        for t in kept:
            t.fill_(3)
        K.token_logprobs(x[:5], targets[:5], top=3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_many_rows() -> None:
    """More rows than a grid's y dimension holds."""
    import torch

    from deciax_amd import kernels as K

    say("token_logprobs 70000 rows")
    r = rng(5)
    x = torch.from_numpy(r.normal(size=(70000, 40)).astype(np.float32)).cuda()
    targets = i32(r.integers(0, 40, 70000))
    lp, ent, ids, _ = K.token_logprobs(x, targets, top=2)
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double().cpu(), 1)
    assert (lp.cpu().double() - want.gather(1, targets.cpu().long()[:, None])[:, 0]).abs().max() < 1e-5
    assert (ids[:, 0].cpu() == x.cpu().argmax(1)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap", [41.0, 50.0, 120.0, 1000.0, 1e7, 1e38])
def test_large_soft_caps(cap: float, dtype: str) -> None:
    """Caps far above the logits and logits far below minus the cap: e^{t - cap} is no number there. A capped logit is off
    by 8 u of itself (a fraction cut at 0.4 u and seven roundings; the form beyond 0.9 of the cap likewise), so by 8 u of
    the smaller of the cap and the largest logit; its difference to the largest and its conversion by 4 u more."""
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs cap={cap} {dtype}")
    r = rng(int(min(cap, 9999)))
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = (r.normal(size=(6, 5000)) * 4).astype(np.float32)
    x[1] -= min(3 * cap, 1000.0)
    x[2] *= 20
    x[3, ::2] = -np.inf
    x[4, :] = -np.inf
    x[4, 77] = -5.0
    x[5, 9] = np.inf
    logits = torch.from_numpy(x).cuda().to(t)
    host = logits.float().cpu().numpy()
    targets = r.integers(0, 5000, 6)
    targets[4] = 77
    got = K.token_logprobs(logits, i32(targets), top=6, softcap=cap)
    torch.cuda.synchronize()
    for i in range(6):
        finite = np.abs(host[i][np.isfinite(host[i])])
        size = min(cap, max(finite.max(), cap if i == 5 else 0.0))
        check(host[i:i + 1], targets[i:i + 1], 6, cap, [g[i:i + 1] for g in got], size)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_chunks_masked_with_the_lowest_value(dtype: str) -> None:
    """The type's lowest value as a mask, over whole chunks of 2048 logits or the short last one: their weight is 0, and
    the entropy that of the others."""
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs with chunks of the lowest value {dtype}")
    vocab = 5000
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    lowest = torch.finfo(t).min
    logits = torch.from_numpy((rng(3).normal(size=(6, vocab)) * 4).astype(np.float32)).cuda().to(t)
    logits[0, 2048:4096] = lowest
    logits[1, 4096:] = lowest
    logits[2, :4096] = lowest
    logits[3, 1:] = lowest
    logits[4, 100:] = lowest
    logits[4, 2048:4000] = -float("inf")
    logits[5, :4090] = -float("inf")
    logits[5, 4096:] = lowest
    host = logits.float().cpu().numpy()
    targets = np.array([5, 4999, 4200, 0, 99, 4095])
    got = K.token_logprobs(logits, i32(targets), top=6)
    torch.cuda.synchronize()
    check(host, targets, 6, 0.0, got, float(np.abs(host[host > lowest]).max(where=np.isfinite(host[host > lowest]), initial=1.0)))


@pytest.mark.parametrize("cap", [1e37, 1e38, 3e38])
def test_logits_near_a_cap_near_the_largest_number(cap: float) -> None:
    """Logits of up to such a cap beside ordinary ones: t is at most the cap, a number, whatever its factors are. Ordinary
    logits weigh nothing beside those."""
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs of huge logits, cap={cap}")
    x = (rng(8).normal(size=(4, 3000)) * 4).astype(np.float32)
    for i, y in enumerate((0.3, 0.6, 0.85, 1.0)):
        x[i, 2500] = np.float32(cap * y)
    x[1, :2000] = -np.inf
    x[2, 7] = x[2, 2500]
    low = x.copy()
    low[:, :2000] = -np.float32(cap)  # weighs nothing either
    # one logit far above all others, or (row 2 of x) two equal ones: a few roundings of 1
    for logits, targets, want in ((x, [2500, 2500, 7, 2500], [0.0, 0.0, -np.log(2), 0.0]), (low, [2500] * 4, [0.0] * 4)):
        lp, ent, ids, tops = (t.cpu().numpy().astype(np.float64) for t in
                              K.token_logprobs(torch.from_numpy(logits).cuda(), i32(targets), top=1, softcap=cap))
        for got in (lp, -ent, tops[:, 0]):
            assert (np.abs(got - want) <= 16 * U).all(), (cap, got, want)
        assert ids[:, 0].tolist() == targets


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap,vocab", [(0.0, 3000), (30.0, 3000), (30.0, 50257), (40.0, 3000), (50.0, 3000), (30.0, 90)])
def test_tokens_of_a_probability_near_one(cap: float, vocab: int, dtype: str) -> None:
    """One logit far above the others: its log probability is -log(1 + R), R the others' weights beside its own, and keeps
    the precision of R, however small. With s the larger of the capped logits, each weight's exponent is off by 2 * 8 u s
    (see above) and 3 u times its size of at most 2 s, itself by 2 u, their sum by 96 u, the logarithm by 2: 22 s + 100
    roundings relative to R, below the bound of `check` relative to the value. The entropy, log(1 + R) - E / (1 + R) with
    both terms positive, takes the exponents' error once more. No log probability is above 0 and no entropy below."""
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs of near certain tokens vocab={vocab} cap={cap} {dtype}")
    r = rng(vocab)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    sizes = np.array([22.0, 23.0, 26.0, 30.0, 40.0, 55.0, 70.0, 130.0])
    x = r.normal(size=(len(sizes), vocab)).astype(np.float32)
    targets = r.integers(0, vocab, len(sizes))
    x[np.arange(len(sizes)), targets] = sizes
    logits = torch.from_numpy(x).cuda().to(t)
    host = logits.float().cpu().numpy()
    lp, ent, ids, tops = (g.cpu().numpy().astype(np.float64) for g in K.token_logprobs(logits, i32(targets), top=2, softcap=cap))
    for i in range(len(sizes)):
        row = host[i].astype(np.float64)
        c = cap * np.tanh(row / cap) if cap else row
        d = np.delete(c, targets[i]) - c[targets[i]]
        others = np.exp(d).sum()  # by themselves: of 1 + R, 64 bits too lose what is below 1e-16
        want, want_ent = -np.log1p(others), np.log1p(others) - (np.exp(d) * d).sum() / (1 + others)
        assert want > -1e-3
        tol = 2 * (12 * min(cap or 1e9, sizes[i]) + 96 + 8) * U
        assert lp[i] <= 0 and ent[i] >= 0, (i, lp[i], ent[i])
        assert abs(lp[i] - want) <= tol * abs(want) + 1e-37, (i, lp[i], want)
        assert abs(ent[i] - want_ent) <= 2 * tol * want_ent + 1e-36, (i, ent[i], want_ent)
        assert tops[i, 0] == lp[i] and ids[i].tolist() == oracle.token_logprobs(host[i], int(targets[i]), 2, cap)[2].tolist()


def test_more_rows_than_one_launch_holds() -> None:
    """2^23 workgroups of 512 threads are as many threads as 32 bits count. Two logits a row: log p = -log(1 + e^d) with
    d = x_other - x_target exact in fp32 (both are bf16 near each other): a few roundings of it."""
    import torch

    from deciax_amd import kernels as K

    rows = (1 << 23) + 77
    say(f"token_logprobs {rows} rows")
    x = torch.randn((rows, 2), device="cuda", dtype=torch.bfloat16)
    targets = torch.arange(rows, device="cuda", dtype=torch.int32) % 3 - 1
    lp, ent, ids, tops = K.token_logprobs(x, targets, top=1)
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double(), 1)
    at = want.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]
    at = torch.where(targets < 0, 0.0, at)
    assert ((lp - at).abs() <= 16 * U * (1 + at.abs())).all()
    assert ((ent + (want.exp() * want).sum(1)).abs() <= 16 * U * 2).all()
    assert (ids[:, 0] == (x[:, 1] > x[:, 0]).int()).all()
    assert ((tops[:, 0] - want.amax(1)).abs() <= 16 * U).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("vocab,top", [(262145, 64), (600001, 7), (1100003, 64), (5000000, 1)])
def test_vocabularies_beyond_a_workgroups_registers(vocab: int, top: int, cap: float, dtype: str) -> None:
    """More groups than the threads hold at once, and more chunks than threads, with ties among the best."""
    import torch

    from deciax_amd import kernels as K

    say(f"token_logprobs vocab={vocab} top={top} cap={cap} {dtype}")
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    x = torch.from_numpy((rng(vocab).normal(size=(2, vocab)) * 3).astype(np.float32)).cuda().to(t)
    x[1, vocab - 1] = x[1, 5] = x[1, vocab // 2] = x[1].max() + 1
    targets = np.array([vocab // 3, vocab - 1])
    got = K.token_logprobs(x, i32(targets), top=top, softcap=cap)
    torch.cuda.synchronize()
    check(x.float().cpu().numpy(), targets, top, cap, got)
