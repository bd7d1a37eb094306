"""`kernels.qk_norm_rope` on the GPU against the 64-bit oracle.

Tolerance (u = 2^-24). The norm: a sum of D squares, eight in turn and log2(D / 8) joins, half of its error in the root,
2 u for the root and 3 products: under 16 u of a normed value; the rotation: a share of a turn rounded to fp32 (an angle off
by u pi at most), cos and sin off by 2 u, the factor, two products and their sum: under 10 u of |a| + |b|. Rounded once.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import token_layer as oracle
from tests.conftest import bf16_np, i32, rng, say, to_dev, to_np

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(got, x, positions, freq, qn, kn, *, heads, d, eps, interleaved, factor, bf16) -> None:
    kw = dict(heads=heads, d=d, eps=eps, interleaved=interleaved)
    want = oracle.qk_norm_rope(x, positions, freq, qn, kn, factor=factor, **kw)
    normed = oracle.qk_norm_rope(x, positions, np.zeros(0), qn, kn, factor=1.0, **kw).reshape(len(x), -1, d)
    size = np.abs(normed)
    pairs = len(freq)
    first = np.arange(pairs) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    both = (size[..., first] + size[..., second]) * abs(factor)
    size[..., first], size[..., second] = both, both
    tol = 26 * U * size.reshape(len(x), -1) + (2.0 ** -8 if bf16 else U) * np.abs(want)
    off = np.abs(got - want)
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), np.unravel_index((off - tol).argmax(), off.shape))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,hq,hkv,d,rot,norm", [
    (1, 1, 1, 64, 64, True), (3, 4, 2, 64, 16, True), (5, 3, 1, 64, 48, False), (7, 16, 8, 256, 256, False),
    (9, 2, 0, 128, 128, True), (4, 0, 3, 128, 32, True), (13, 5, 5, 256, 64, True), (6, 7, 1, 256, 240, True),
    (33, 32, 16, 128, 0, True), (301, 12, 4, 64, 32, True), (2, 1, 0, 256, 0, False)])
def test_against_the_oracle(rows: int, hq: int, hkv: int, d: int, rot: int, norm: bool, layout: str, dtype: str) -> None:
    import torch

    from deciax_amd import kernels as K

    say(f"qk_norm_rope rows={rows} {hq}/{hkv} x {d} rot={rot} {layout} norm={norm} {dtype}")
    r = rng(rows * d + rot)
    width = (hq + hkv) * d
    cast = bf16_np if dtype == "bf16" else (lambda t: t.astype(np.float32))
    x = cast(r.normal(size=(rows, width)) * np.exp(r.normal(size=(rows, 1)) * 2))
    qn, kn = (cast(r.normal(size=d) * 0.4) if norm else None for _ in "qk")
    positions = r.integers(-5, 2_000_000, rows)
    positions[0] = 2 ** 31 - 1
    freq, _ = K.rope_frequencies(max(rot, 2), theta=10000.0, scaling={"rope_type": "yarn", "factor": 4.0,
                                                                      "original_max_position_embeddings": 4096})
    freq = freq[:rot // 2].contiguous()
    factor = 1.25 if rot else 1.0
    kw = dict(num_q_heads=hq, num_kv_heads=hkv, head_dim=d, eps=1e-5, layout=layout, attention_factor=factor,
              q_norm=to_dev(qn, dtype) if norm else None, k_norm=to_dev(kn, dtype) if norm else None)
    row = to_dev(np.concatenate([x, np.full((rows, 16), 7.0, np.float32)], 1), dtype)
    out = torch.full((rows + 1, width + 8), 3.0, dtype=row.dtype, device="cuda")
    K.qk_norm_rope(row, i32(positions), freq, out=out, **kw)
    torch.cuda.synchronize()
    checked = dict(heads=(hq, hkv), d=d, eps=1e-5, interleaved=layout == "interleaved", factor=factor, bf16=dtype == "bf16")
    check(to_np(out)[:rows, :width], x, positions, freq.cpu().numpy(), qn, kn, **checked)
    assert (out[rows] == 3).all() and (out[:, width:] == 3).all()
    assert K.qk_norm_rope(row, i32(positions), freq, **kw) is row  # in place
    torch.cuda.synchronize()
    assert torch.equal(row[:, :width], out[:rows, :width]) and (row[:, width:] == 7).all()


def test_is_rope_where_rope_applies() -> None:
    """Without norms, half pairs: `rope` up to its own roundings (tables and products in bf16)."""
    import torch

    from deciax_amd import kernels as K

    say("qk_norm_rope beside rope")
    r = rng(3)
    x = to_dev(bf16_np(r.normal(size=(50, 24 * 64))))
    positions = i32(r.integers(0, 5000, 50))
    freq, _ = K.rope_frequencies(64)
    angle = torch.arange(5000, dtype=torch.float64, device="cuda")[:, None] * freq
    old = K.rope(x.clone(), positions, angle.cos().bfloat16(), angle.sin().bfloat16(), num_heads=24, head_dim=64)
    new = K.qk_norm_rope(x.clone(), positions, freq, num_q_heads=16, num_kv_heads=8, head_dim=64)
    torch.cuda.synchronize()
    size = x.float().view(50, 24, 2, 32).abs().sum(2, keepdim=True).expand(50, 24, 2, 32).reshape(50, -1)
    # table, product and result: three half steps of 2^-8 of both terms
    assert ((old.float() - new.float()).abs() <= 4 * 2.0 ** -8 * size).all()


def test_lost_heads_stay_apart() -> None:
    import torch

    from deciax_amd import kernels as K

    say("qk_norm_rope with infinities, NaN and zeros")
    r = rng(4)
    x = r.normal(size=(6, 4 * 128)).astype(np.float32)
    x[1, 130], x[2, 300] = np.nan, np.inf
    x[4] = 0.0
    freq, _ = K.rope_frequencies(64)
    w = to_dev(np.zeros(128, np.float32), "f32")
    y = K.qk_norm_rope(to_dev(x, "f32"), i32(range(6)), freq, num_q_heads=3, num_kv_heads=1, head_dim=128, q_norm=w, k_norm=w)
    torch.cuda.synchronize()
    bad = ~np.isfinite(to_np(y)).reshape(6, 4, 128).all(-1)
    want = np.zeros((6, 4), bool)
    want[1, 1] = want[2, 2] = True
    assert (bad == want).all() and (y[4] == 0).all()


def test_many_rows_streams_and_graphs() -> None:
    import torch

    from deciax_amd import kernels as K

    say("qk_norm_rope 40000 rows, a side stream, a graph")
    r = rng(5)
    freq, _ = K.rope_frequencies(32)
    x = to_dev(bf16_np(r.normal(size=(40000, 3 * 64))))
    positions = i32(r.integers(0, 100000, 40000))
    w = to_dev(bf16_np(r.normal(size=64) * 0.2))
    kw = dict(num_q_heads=2, num_kv_heads=1, head_dim=64, q_norm=w, k_norm=w)
    want = K.qk_norm_rope(x, positions, freq, out=torch.empty_like(x), **kw)
    torch.cuda.synchronize()
    for at in (0, 1, 39999):
        one = K.qk_norm_rope(x[at:at + 1].clone(), positions[at:at + 1], freq, **kw)
        assert torch.equal(one[0], want[at])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.qk_norm_rope(x, positions, freq, out=torch.empty_like(x), **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.qk_norm_rope(x, positions, freq, out=out, **kw)
    for _ in range(3):
        out.fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals() -> None:
    import torch

    from deciax_amd import kernels as K

    x = torch.zeros((4, 384), dtype=torch.bfloat16, device="cuda")
    p, (f, _) = i32(range(4)), K.rope_frequencies(64)
    w = torch.zeros(64, dtype=torch.bfloat16, device="cuda")

    def call(x=x, p=p, f=f, hq=4, hkv=2, d=64, **kw):
        return K.qk_norm_rope(x, p, f, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, **kw)

    call()
    for bad in (dict(hq=5), dict(d=96), dict(hq=-1), dict(p=p.long()), dict(p=p[:3]), dict(f=f.float()), dict(f=f[:3]),
                dict(f=torch.cat([f, f])), dict(f=f.cpu()), dict(q_norm=w), dict(q_norm=w.float(), k_norm=w.float()),
                dict(q_norm=w[:32], k_norm=w[:32]), dict(q_norm=w, k_norm=w, eps=-1.0), dict(layout="pairs"),
                dict(x=x.half()), dict(x=x[0]), dict(out=x[1:]), dict(out=torch.empty((4, 100), dtype=x.dtype, device="cuda")),
                dict(out=x.float()), dict(x=x[:, 4:], hq=3), dict(x=x[:, 1::2][:, :128], hq=1, hkv=1)):
        with pytest.raises(ValueError):
            call(**bad)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_cosines_and_sines_keep_their_own_precision(layout: str) -> None:
    """Pairs (1, 0) turn to (cos, sin), whose small values beside a multiple of a quarter turn are as exact as the large ones.
    sincospi's cosine and sine are off by 2 u of themselves, the angle behind its fp32 number by a product and a sum: under
    8 u. The angle itself: three roundings of 2^-53 of at most 20000 radians, 7e-12."""
    import torch

    from deciax_amd import kernels as K

    say(f"qk_norm_rope cosines and sines, {layout}")
    rows, pairs = 5000, 32
    freq, _ = K.rope_frequencies(2 * pairs, theta=500.0)
    x = np.zeros((rows, 2, pairs) if layout == "half" else (rows, pairs, 2), np.float32)
    (x[:, 0] if layout == "half" else x[..., 0])[:] = 1.0
    positions = rng(6).integers(0, 20000, rows)
    got = K.qk_norm_rope(to_dev(x.reshape(rows, -1), "f32"), i32(positions), freq, num_q_heads=1, num_kv_heads=0, head_dim=64,
                         layout=layout)
    torch.cuda.synchronize()
    angle = positions[:, None] * freq.cpu().numpy()
    want = np.stack([np.cos(angle), np.sin(angle)], 1 if layout == "half" else 2).reshape(rows, -1)
    off = np.abs(to_np(got) - want)
    tol = 8 * U * np.abs(want) + 7e-12
    assert (off <= tol).all(), (float((off / tol).max()), float(off.max() / U))
