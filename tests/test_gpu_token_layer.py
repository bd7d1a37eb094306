"""The operators of a token layer together, as a model's layers would run them: 4-bit projections, head norms with rotation,
the 4-bit cache with attention over it, linear attention with its kept state; a prompt, then single tokens, eager and as a
graph. Each step's result is checked against the 64-bit oracle of what the step read, with the bounds of its own tests.
"""

from __future__ import annotations

import numpy as np
import pytest

from tests import test_gpu_kv4 as kv4
from tests import test_gpu_linear_attention as mixer
from tests import test_gpu_q4 as q4
from tests import test_gpu_qk_norm_rope as rope
from tests.conftest import bf16_np, i32, rng, say, to_dev, to_np

pytestmark = pytest.mark.gpu

WIDTH, HQ, HKV, D, HK, H, DIM, PAGE = 256, 4, 2, 64, 2, 4, 64, 64
EPS, FACTOR = 1e-6, 1.1


class Layers:
    """An attention layer over the 4-bit cache and a layer of linear attention, for some sequences with their states."""

    def __init__(self, seed: int, prompts: list[int], most: int) -> None:
        import torch

        from deciax_amd import kernels as K

        r = rng(seed)
        self.n = len(prompts)
        self.parts = {name: q4.weight(r, n, k, group) for name, n, k, group in (
            ("qkv", (HQ + 2 * HKV) * D, WIDTH, 64), ("o", WIDTH, HQ * D, 128), ("mix", 2 * HK * DIM + H * DIM, WIDTH, 32),
            ("decay", H, WIDTH, 64), ("out", WIDTH, H * DIM, 32))}
        self.weights = {name: q4.packed(*p) for name, p in self.parts.items()}
        self.q_norm, self.k_norm = (bf16_np(r.normal(size=D) * 0.3) for _ in "qk")
        self.norms = dict(q_norm=to_dev(self.q_norm), k_norm=to_dev(self.k_norm))
        self.freq, _ = K.rope_frequencies(32, theta=1e6)
        pages = -(-most // PAGE)
        self.table = r.permutation(self.n * pages + 2)[:self.n * pages].reshape(self.n, pages)
        self.d_table, self.cache = i32(self.table), K.kv4_cache(self.n * pages + 2, HKV, D, page_size=PAGE)
        self.index = r.permutation(self.n + 1)[:self.n]
        self.d_index = i32(self.index)
        self.state = torch.zeros((self.n + 1, H, DIM, DIM), device="cuda")

    def run(self, x, positions, starts, lengths, ctx, most: int, most_ctx: int) -> dict:
        """Every step's result by name, for packed rows x."""
        import torch

        from deciax_amd import kernels as K

        s = {"x": x, "qkv": K.linear_q4(x, self.weights["qkv"])}
        heads = dict(num_q_heads=HQ, num_kv_heads=HKV, head_dim=D)
        s["turned"] = K.qk_norm_rope(s["qkv"].clone(), positions, self.freq, eps=EPS, attention_factor=FACTOR, **heads,
                                     **self.norms)
        q, k, v = s["turned"].split([HQ * D, HKV * D, HKV * D], 1)
        K.kv4_append(self.cache, k, v, positions, self.d_table, starts, lengths, ctx, most)
        s["attended"] = K.attention_kv4(q, self.cache, self.d_table, starts, lengths, ctx, most, most_ctx, num_q_heads=HQ,
                                        scale=D ** -0.5)
        s["o"] = K.linear_q4(s["attended"], self.weights["o"])
        s["y"] = (x + s["o"]) * 0.1
        s["mix"] = K.linear_q4(s["y"], self.weights["mix"])
        s["decay"] = K.linear_q4(s["y"], self.weights["decay"], out_dtype=torch.float32)
        s["g"] = -torch.nn.functional.softplus(s["decay"])
        q, k, v = s["mix"].split([HK * DIM, HK * DIM, H * DIM], 1)
        s["before"] = self.state.clone()
        s["mixed"] = K.linear_attention(q, k, v, s["g"], self.state, starts, lengths, most, num_k_heads=HK, num_heads=H,
                                        k_dim=DIM, v_dim=DIM, scale=DIM ** -0.5, state_index=self.d_index)
        s["after"] = self.state.clone()
        s["out"] = K.linear_q4(s["mixed"], self.weights["out"])
        return s

    def check(self, s: dict, positions: np.ndarray, starts: list[int], lengths: list[int], ctx: list[int]) -> None:
        import torch

        torch.cuda.synchronize()
        h = {name: to_np(t) for name, t in s.items()}
        for name, of in (("qkv", "x"), ("o", "attended"), ("mix", "y"), ("decay", "y"), ("out", "mixed")):
            q4.check(h[name], h[of], self.parts[name], name != "decay")
        heads = (HQ + HKV) * D
        rope.check(h["turned"][:, :heads], h["qkv"][:, :heads], positions, self.freq.cpu().numpy(), self.q_norm, self.k_norm,
                   heads=(HQ, HKV), d=D, eps=EPS, interleaved=False, factor=FACTOR, bf16=True)
        assert np.array_equal(h["turned"][:, heads:], h["qkv"][:, heads:])
        a = object.__new__(kv4.Case)
        a.cache, a.table, a.q, a.page, a.dtype = self.cache, self.table, s["turned"][:, :HQ * D], PAGE, "bf16"
        a.new, a.ctx, a.starts, a.hq, a.hkv, a.d = lengths, ctx, starts, HQ, HKV, D
        a.check(s["attended"], scale=D ** -0.5, softcap=0.0, window=0)
        m = object.__new__(mixer.Case)
        m.lengths, m.starts, m.rows, m.hk, m.h, m.dk, m.dv, m.dtype = lengths, starts, len(positions), HK, H, DIM, DIM, "bf16"
        m.q, m.k = (h["mix"][:, i * HK * DIM:(i + 1) * HK * DIM].reshape(-1, HK, DIM) for i in range(2))
        m.v, m.decay = h["mix"][:, 2 * HK * DIM:].reshape(-1, H, DIM), h["g"]
        m.state, m.index, m.slots, m.scale = h["before"], self.index, self.n + 1, DIM ** -0.5
        m.check(np.pad(h["mixed"], ((0, 0), (0, 8)), constant_values=9.0), h["after"], untouched=0.0)


def step_inputs(lengths: list[int], before: list[int]):
    starts = [int(t) for t in np.cumsum([0] + lengths)[:-1]]
    ctx = [b + n for b, n in zip(before, lengths)]
    positions = np.concatenate([np.arange(b, c) for b, c in zip(before, ctx)])
    return starts, ctx, positions


@pytest.mark.parametrize("prompts", [[1], [37, 1, 130, 700], [5, 6, 7, 8, 9, 16, 17, 63, 64, 65]])
def test_prompt_and_steps(prompts: list[int]) -> None:
    import torch

    say(f"token layer, prompts {prompts}")
    most = max(prompts) + 8
    layers, r = Layers(len(prompts), prompts, most), rng(3)
    before = [0] * len(prompts)
    for lengths in (prompts, [1] * len(prompts), [(b + 2) % 4 for b in range(len(prompts))], [1] * len(prompts)):
        starts, ctx, positions = step_inputs(lengths, before)
        x = to_dev(bf16_np(r.normal(size=(len(positions), WIDTH))))
        s = layers.run(x, i32(positions), i32(starts), i32(lengths), i32(ctx), max(lengths), max(ctx))
        layers.check(s, positions, starts, lengths, ctx)
        before = ctx
    torch.cuda.synchronize()


def test_steps_from_a_graph() -> None:
    """Single tokens from one captured graph, its inputs rewritten between replays, against the same steps run eagerly."""
    import torch

    say("token layer, steps replayed")
    prompts, steps = [40, 3, 90], 5
    most = max(prompts) + steps
    eager, captured = Layers(9, prompts, most), Layers(9, prompts, most)
    r = rng(4)
    starts, ctx, positions = step_inputs(prompts, [0] * 3)
    x = to_dev(bf16_np(r.normal(size=(len(positions), WIDTH))))
    for layers in (eager, captured):
        layers.run(x, i32(positions), i32(starts), i32(prompts), i32(ctx), max(prompts), max(ctx))
    ones, at = i32([1, 1, 1]), i32([0, 1, 2])
    x1, d_pos, d_ctx = torch.zeros((3, WIDTH), dtype=torch.bfloat16, device="cuda"), i32(ctx), i32([c + 1 for c in ctx])
    kept = captured.state.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = captured.run(x1, d_pos, at, ones, d_ctx, 1, most)
    torch.cuda.synchronize()
    assert torch.equal(captured.state, kept)  # a capture runs nothing
    for i in range(steps):
        x1.copy_(to_dev(bf16_np(r.normal(size=(3, WIDTH)))))
        now = [c + i for c in ctx]
        d_pos.copy_(i32(now))
        d_ctx.copy_(i32([c + 1 for c in now]))
        graph.replay()
        want = eager.run(x1, d_pos, at, ones, d_ctx, 1, most)
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(got[name], want[name]), (i, name)
        captured.check(got, np.array(now), [0, 1, 2], [1, 1, 1], [c + 1 for c in now])


def far_rows(rows: int, stride: int, last: int, width: int):
    """A bf16 buffer of more than 2^31 elements whose last rows hold values; the rest is not written."""
    import torch

    x = torch.empty((rows, stride), dtype=torch.bfloat16, device="cuda")
    assert rows * stride > 2 ** 31
    x[-last:, :width] = to_dev(bf16_np(rng(last).normal(size=(last, width))))
    return x


def test_weights_beyond_32_bit_offsets() -> None:
    import torch

    from deciax_amd import kernels as K

    say("linear_q4 of a weight of 4.8 GB")
    n, k = 2_300_000, 4096
    r = torch.Generator(device="cuda").manual_seed(1)
    tiles = n // 16
    codes = torch.empty((tiles, k // 128, 64, 16), dtype=torch.uint8, device="cuda")
    assert codes.numel() > 2 ** 32
    codes[-20:] = torch.randint(0, 256, (20, k // 128, 64, 16), dtype=torch.uint8, device="cuda", generator=r)
    groups = torch.zeros((tiles, k // 128, 16), dtype=torch.int32, device="cuda")
    groups[-20:] = torch.rand((20, k // 128, 16), device="cuda", generator=r).to(torch.bfloat16).float().view(torch.int32) | 7
    w, part = K.Q4Weight(codes, groups, n, k), K.Q4Weight(codes[-20:].clone(), groups[-20:].clone(), 320, k)
    x = to_dev(bf16_np(rng(5).normal(size=(70, k))))
    for m in (1, 20, 70):
        got, want = K.linear_q4(x[:m], w), K.linear_q4(x[:m], part)
        assert torch.equal(got[:, -320:], want) and (got[:, :1000] == 0).all(), m


def test_rows_beyond_32_bit_offsets() -> None:
    import torch

    from deciax_amd import kernels as K

    say("token layer rows beyond 2^31 elements")
    x = far_rows(150_000, 16384, 40, 512)
    w = q4.packed(*q4.weight(rng(6), 300, 512, 128))
    out = K.linear_q4(x[:, :512], w)
    assert torch.equal(out[-40:], K.linear_q4(x[-40:, :512].contiguous(), w))
    freq, _ = K.rope_frequencies(64)
    positions = torch.arange(150_000, dtype=torch.int32, device="cuda")
    kw = dict(num_q_heads=6, num_kv_heads=2, head_dim=64)
    want = K.qk_norm_rope(x[-40:, :512].clone(), positions[-40:].clone(), freq, **kw)
    K.qk_norm_rope(x, positions, freq, **kw)
    assert torch.equal(x[-40:, :512], want)
    g = -torch.rand((150_000, 2), device="cuda")
    mixer_kw = dict(num_k_heads=1, num_heads=2, k_dim=64, v_dim=64, scale=0.125)

    def run(x, g, start: int, state, **more):
        return K.linear_attention(x[:, :64], x[:, 64:128], x[:, 128:256], g, state, i32([start]), i32([40]), 40, **mixer_kw,
                                  **more)

    state, near = (torch.zeros((1, 2, 64, 64), device="cuda") for _ in range(2))
    room = torch.empty((150_000, 16384), dtype=torch.bfloat16, device="cuda")
    run(x, g, 150_000 - 40, state, out=room[:, :128])
    want = run(x[-40:, :256].contiguous(), g[-40:].contiguous(), 0, near)
    assert torch.equal(room[-40:, :128], want) and torch.equal(state, near)
    del room, x
    pool = torch.empty((70_000, 2, 128, 128), device="cuda")
    assert pool.numel() > 2 ** 31
    y = to_dev(bf16_np(rng(7).normal(size=(900, 512))))
    for n in (1, 50, 900):  # token by token, one segment, more of them
        pool[-1] = 0.5
        near = torch.full((1, 2, 128, 128), 0.5, device="cuda")
        outs = [K.linear_attention(y[:n, :128], y[:n, 128:256], y[:n, 256:], g[:n], s, i32([0]), i32([n]), n, num_k_heads=1,
                                   num_heads=2, k_dim=128, v_dim=128, scale=0.1, state_index=i32([len(s) - 1]))
                for s in (pool, near)]
        assert torch.equal(*outs) and torch.equal(pool[-1], near[0]), n
    del pool
    torch.cuda.empty_cache()
