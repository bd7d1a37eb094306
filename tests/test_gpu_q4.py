"""`kernels.linear_q4` and what makes its weights, on the GPU against the 64-bit oracle.

Tolerance (u = 2^-24). A group's products x (8 + code / 2) and x are exact, their sums and that of X off by at most g u of
the sum of |x| 15.5 each (g: the group's size); the difference is rounded once. Then the scale and the sum over the groups
of a wave, k / group / 8 + 1 of them, and over eight waves, each off by u of what is added. A bf16 result by 2^-8 of itself.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import token_layer as oracle
from tests.conftest import bf16_np, rng, say, to_dev, to_np

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def weight(r: np.random.Generator, n: int, k: int, group: int):
    code = r.integers(0, 16, (n, k)).astype(np.uint8)
    scale = bf16_np(np.exp(r.normal(size=(n, k // group)) * 0.4) * 0.02)
    zero = r.integers(0, 16, (n, k // group)).astype(np.uint8)
    return code, scale, zero


def packed(code: np.ndarray, scale: np.ndarray, zero: np.ndarray):
    import torch

    from deciax_amd import kernels as K

    return K.pack_q4(torch.from_numpy(code).cuda(), to_dev(scale), torch.from_numpy(zero).cuda())


def check(got: np.ndarray, x: np.ndarray, parts, bf16: bool) -> None:
    code, scale, zero = parts
    n, groups = scale.shape
    k = code.shape[1]
    g = k // groups
    x = x.astype(np.float64)
    want = x @ oracle.q4_values(*parts).T
    size = np.abs(x).reshape(len(x), groups, g).sum(-1)                            # [m, groups]
    each = np.einsum("mgk,ngk->mng", x.reshape(len(x), groups, g), oracle.q4_values(*parts).reshape(n, groups, g))
    tol = U * (2 * 15.5 * 2 * g * (size @ np.abs(scale).T) + (groups / 8 + 12) * np.abs(each).sum(-1))
    tol = tol + (2.0 ** -8 * np.abs(want) if bf16 else U * np.abs(want))
    off = np.abs(got - want)
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), np.unravel_index((off - tol).argmax(), off.shape))
    # the bound is for errors that all point one way: those of random signs are far smaller
    assert np.linalg.norm(off) <= (2.0 ** -8 if bf16 else 1e-6) * np.linalg.norm(want)


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (33, 192, 64), (40, 4096, 64)])
def test_formats(n: int, k: int, group: int) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"q4 formats {n} x {k} group {group}")
    r = rng(n + k)
    parts = weight(r, n, k, group)
    w = packed(*parts)
    torch.cuda.synchronize()
    codes, groups = oracle.lay_out(*parts)
    assert (w.codes.cpu().numpy() == codes).all() and (w.groups.cpu().numpy() == groups).all()
    assert np.array_equal(to_np(K.q4_values(w)), oracle.q4_values(*parts).astype(np.float32))
    half = np.exp(r.normal(size=parts[1].shape)).astype(np.float16)
    half[0, 0] = 6e-8  # a subnormal number
    w = K.pack_q4(torch.from_numpy(parts[0]).cuda(), torch.from_numpy(half).cuda())
    want = oracle.q4_values(parts[0], half, np.full_like(parts[2], 8))
    assert np.array_equal(to_np(K.q4_values(w)), want.astype(np.float32))

    x = bf16_np(r.normal(size=(n, k)) * np.exp(r.normal(size=(n, 1))))
    x[0, :32] = 0.0
    if n > 20:
        x[3, 5], x[4, 40], x[5] = np.inf, np.nan, 0.75
        x[6, 3], x[7] = 3e38, 1e-40
    wide = to_dev(np.concatenate([x, np.full((n, 8), 99.0, np.float32)], 1))
    parts = oracle.quantise_q4(x, group)
    w = K.quantize_q4(wide[:, :k], group=group)
    torch.cuda.synchronize()
    codes, groups = oracle.lay_out(*parts)
    nan = np.isnan(parts[1])
    assert (w.codes.cpu().numpy() == codes).all()
    got, same = w.groups.cpu().numpy(), np.zeros(groups.shape, bool)
    same[np.arange(n) // 16, :, np.arange(n) % 16] = nan
    assert (got[~same] == groups[~same]).all()
    with np.errstate(invalid="ignore"):
        assert np.array_equal(to_np(K.q4_values(w)), oracle.q4_values(*parts).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 32, 32), (1, 17, 160, 32), (2, 100, 128, 128), (3, 64, 1088, 64), (15, 33, 1152, 128), (16, 250, 96, 32),
    (17, 16, 2080, 32), (31, 70, 256, 128), (32, 257, 640, 64), (33, 65, 1056, 32), (48, 80, 1152, 128), (64, 64, 320, 64),
    (65, 130, 1280, 128), (129, 191, 544, 32), (300, 515, 1024, 64), (1, 3584, 4096, 128), (7, 515, 14336, 128)])
def test_products(m: int, n: int, k: int, group: int, dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 {m} x {n} x {k} group {group} {dtype}")
    r = rng(m * n + k)
    parts = weight(r, n, k, group)
    w = packed(*parts)
    x = bf16_np(r.normal(size=(m, k)) * np.exp(r.normal(size=k) * 0.5))
    wide = to_dev(np.concatenate([np.full((m, 8), np.nan, np.float32), x, np.full((m, 8), np.nan, np.float32)], 1))
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    room = torch.full((m + 1, n + 3), 5.0, dtype=t, device="cuda")  # rows of an odd stride
    out = K.linear_q4(wide[:, 8:8 + k], w, out=room[:m, 1:n + 1], out_dtype=t)
    torch.cuda.synchronize()
    check(to_np(out), x, parts, dtype == "bf16")
    assert (room[m] == 5).all() and (room[:, 0] == 5).all() and (room[:, n + 1:] == 5).all()


@pytest.mark.parametrize("group,k", [(32, 2080), (64, 1344), (128, 3584)])
def test_rows_do_not_depend_on_the_batch(group: int, k: int) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 rows alone and in batches, group {group}")
    r = rng(group)
    w = packed(*weight(r, 300, k, group))
    x = to_dev(bf16_np(r.normal(size=(400, k))))
    want = K.linear_q4(x, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    for m in (1, 2, 5, 16, 17, 32, 33, 40, 64, 65, 100, 128, 129, 200, 256, 257, 399):
        for at in (0, 400 - m):
            got = K.linear_q4(x[at:at + m], w, out_dtype=torch.float32)
            assert torch.equal(got, want[at:at + m]), (m, at)


def test_lost_rows_stay_apart() -> None:
    """Infinities and NaN in rows of x, and groups of a weight that read as NaN, reach their own rows and columns."""
    import torch

    from deciax_amd import kernels as K

    say("linear_q4 with infinities and NaN")
    r = rng(11)
    parts = weight(r, 50, 256, 64)
    for m in (5, 40, 100):
        x = bf16_np(r.normal(size=(m, 256)))
        x[1, 3], x[3, 200] = np.nan, np.inf
        wx = r.normal(size=(50, 256))
        wx[7, 70] = np.inf
        got = K.linear_q4(to_dev(x), K.quantize_q4(to_dev(bf16_np(wx)), group=64))
        torch.cuda.synchronize()
        fine = np.isfinite(to_np(got))
        want = np.ones((m, 50), bool)
        want[[1, 3]], want[:, 7] = False, False
        assert (fine == want).all()
    x = bf16_np(r.normal(size=(3, 256)))
    got = K.linear_q4(to_dev(x), packed(*parts), out_dtype=torch.float32)
    torch.cuda.synchronize()
    check(to_np(got), x, parts, False)


def test_zero_weights_are_zero() -> None:
    import torch

    from deciax_amd import kernels as K

    w = K.quantize_q4(torch.zeros((20, 128), dtype=torch.bfloat16, device="cuda"))
    assert (K.linear_q4(torch.full((3, 128), 1e30, dtype=torch.bfloat16, device="cuda"), w) == 0).all()
    assert K.linear_q4(torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"), w).shape == (0, 20)


def test_streams_and_graphs() -> None:
    import torch

    from deciax_amd import kernels as K

    say("linear_q4 on a side stream, in graphs")
    r = rng(12)
    w = packed(*weight(r, 333, 1152, 128))
    xs = [to_dev(bf16_np(r.normal(size=(m, 1152)))) for m in (3, 70)]
    want = [K.linear_q4(x, w) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [K.linear_q4(x, w) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [K.linear_q4(x, w) for x in xs]
    for _ in range(4):
        for t in kept:
            t.fill_(3)
        K.linear_q4(xs[1][:9], w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_refusals() -> None:
    import torch

    from deciax_amd import kernels as K

    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    w = K.quantize_q4(x)
    for bad in (lambda: K.linear_q4(x.float(), w), lambda: K.linear_q4(x[:, :128], w), lambda: K.linear_q4(x[0], w),
                lambda: K.linear_q4(x.cpu(), w), lambda: K.linear_q4(x, w, out_dtype=torch.float16),
                lambda: K.linear_q4(x, w, out=torch.empty((4, 5), dtype=torch.bfloat16, device="cuda")),
                lambda: K.linear_q4(x, w, out=x[:, :4]), lambda: K.linear_q4(x.T.contiguous().T, w),
                lambda: K.linear_q4(x[:1].expand(4, 256), w),
                lambda: K.linear_q4(x, w, out=torch.empty((4, 4), device="cuda")),
                lambda: K.quantize_q4(x, group=48), lambda: K.quantize_q4(x[:, :96], group=64), lambda: K.quantize_q4(x.float()),
                lambda: K.pack_q4(x, x), lambda: K.pack_q4(x.byte(), x[:, :3]), lambda: K.pack_q4(x.byte(), x[:, :2].float()),
                lambda: K.pack_q4(x.byte(), x[:, :2], x[:, :1].byte()), lambda: K.pack_q4(x.byte(), x[:, :1])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n,k,group", [(16400, 160, 32), (33000, 96, 32), (4200, 5248, 128), (4200, 8192, 64),
                                       (4200, 8320, 64), (5000, 3200, 32)])
def test_rows_of_weights_do_not_depend_on_their_number(n: int, k: int, group: int) -> None:
    """Kernels are chosen by the rows of x and of the weight; a result is the same to the bit whichever ran."""
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 of {n} rows of weights, k {k}")
    r = rng(n + k)
    parts = weight(r, n, k, group)
    w, part = packed(*parts), packed(*(t[:48] for t in parts))
    x = bf16_np(r.normal(size=(300, k)))
    dev = to_dev(x)
    want = K.linear_q4(dev, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    check(to_np(want[:4, :48]), x[:4], tuple(t[:48] for t in parts), False)
    check(to_np(want[:2]), x[:2], parts, False)
    for m in (1, 16, 17, 40, 64, 65, 128, 129, 257, 300):
        assert torch.equal(K.linear_q4(dev[:m], w, out_dtype=torch.float32), want[:m]), m
        assert torch.equal(K.linear_q4(dev[:m], part, out_dtype=torch.float32), want[:m, :48]), m


def test_products_over_the_weight_are_refused() -> None:
    import torch

    from deciax_amd import kernels as K

    w = K.quantize_q4(torch.zeros((64, 256), dtype=torch.bfloat16, device="cuda"))
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    for out in (w.codes.view(-1)[:256].view(torch.bfloat16).view(2, 64), w.groups.view(-1)[:128].view(torch.float32).view(2, 64)):
        with pytest.raises(ValueError, match="meet"):
            K.linear_q4(x[:2], w, out=out, out_dtype=out.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k,group", [
    (128, 16400, 3584, 64), (129, 8200, 3584, 32), (130, 8192, 3584, 128), (257, 5500, 1344, 64), (300, 5450, 1344, 32),
    (70, 16390, 1024, 128), (65, 16384, 1152, 128), (200, 8193, 14336, 128), (129, 8192, 14336, 32)])
def test_many_rows_of_large_weights(m: int, n: int, k: int, group: int, dtype: str) -> None:
    """A tile of 128 by 64 for every CU: all eight sums in one wave, some with a tile more than others. Against the oracle
    at the edges of the tiles, and to the bit what the same rows give where the eight sums are eight waves'."""
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 many rows {m} x {n} x {k} group {group} {dtype}")
    assert m > 64 and -(-n // 64) * -(-m // 128) >= 256
    r = rng(m + n + k)
    parts = weight(r, n, k, group)
    w = packed(*parts)
    x = bf16_np(r.normal(size=(m, k)) * np.exp(r.normal(size=k) * 0.5))
    dev = to_dev(x)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    room = torch.full((m + 1, n + 3), 5.0, dtype=t, device="cuda")
    out = K.linear_q4(dev, w, out=room[:m, 1:n + 1], out_dtype=t)
    torch.cuda.synchronize()
    rows = sorted({0, 15, 16, 31, 32, 63, 64, m // 2, m - 1} & set(range(m)))
    cols = sorted({0, 15, 16, 63, 64, n // 2, n // 2 + 1, n - 17, n - 1})
    check(to_np(out)[np.ix_(rows, cols)], x[rows], tuple(p[cols] for p in parts), dtype == "bf16")
    for at in (0, m - 64, m - 16):
        few = K.linear_q4(dev[at:at + 64], w, out_dtype=t)
        assert torch.equal(few, out[at:at + len(few)]), at
    assert (room[m] == 5).all() and (room[:, 0] == 5).all() and (room[:, n + 1:] == 5).all()


@pytest.mark.parametrize("group,k", [(32, 2080), (64, 1344), (128, 3584)])
def test_rows_of_large_weights_do_not_depend_on_the_batch(group: int, k: int) -> None:
    """As above for 300 rows of weights: with 16400 the rows of a batch pass through every kernel."""
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 rows alone and in batches, 16400 rows of weights, group {group}")
    r = rng(group + 1)
    w = packed(*weight(r, 16400, k, group))
    x = to_dev(bf16_np(r.normal(size=(300, k))))
    want = K.linear_q4(x, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    for m in (1, 2, 16, 17, 32, 33, 48, 64, 65, 66, 100, 128, 129, 192, 193, 256, 257, 299):
        for at in (0, 300 - m):
            got = K.linear_q4(x[at:at + m], w, out_dtype=torch.float32)
            assert torch.equal(got, want[at:at + m]), (m, at)


@pytest.mark.parametrize("m", [3, 40, 130])
def test_largest_scales(m: int) -> None:
    """Scales below 2^127 are numbers like others; larger ones are lost in their own column of the result alone."""
    import torch

    from deciax_amd import kernels as K

    say(f"linear_q4 scales of 2^126, {m} rows")
    r = rng(13)
    parts = weight(r, 8200, 256, 64)
    parts[1][5], parts[1][17, 2] = 2.0 ** 126, -(2.0 ** 126)
    x = bf16_np(r.normal(size=(m, 256)) * 2.0 ** -20)
    got = K.linear_q4(to_dev(x), packed(*parts), out_dtype=torch.float32)
    torch.cuda.synchronize()
    cols = [0, 4, 5, 6, 17, 18, 8199]
    check(to_np(got)[:, cols], x, tuple(p[cols] for p in parts), False)
    parts[1][5, 1] = 2.0 ** 127
    lost = K.linear_q4(to_dev(x), packed(*parts), out_dtype=torch.float32)
    torch.cuda.synchronize()
    other = torch.arange(8200, device="cuda") != 5
    assert torch.equal(lost[:, other], got[:, other])
