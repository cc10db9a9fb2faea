"""Whole prompts attended from their rows, and rows rotated by scaled frequencies on 16-bit and float
pools, against 64 bits; and a run of a small model's layers over a pool held in 4 bits."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests import fp4_ref as ref
from tests.gpu_util import new_context
from tests.operator_ref import DTYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


class Prompts:
    """A pool of 16-bit or float rows (which no call here reads) and packed prompts."""

    def __init__(self, ctx, dtype, counts, heads, d, seed, page=16):
        self.g, self.name, self.dtype = torch.Generator().manual_seed(seed), dtype, DTYPES[dtype]
        self.counts, self.h, self.d, self.n = counts, heads, d, sum(counts)
        pages = [max(1, -(-c // page)) for c in counts]
        cache = [torch.full((1, sum(pages), page, heads, d), math.nan, dtype=self.dtype, device="cuda") for _ in range(2)]
        self.pool = ckv.Pool(ctx, 1, sum(pages), page, heads, d, self.dtype, *cache)
        starts = np.concatenate([[0], np.cumsum(pages)[:-1]])
        seq = np.repeat(np.arange(len(counts)), counts)
        self.positions = np.concatenate([np.arange(c) for c in counts])
        self.pool.upload(np.arange(sum(pages)), starts[seq], np.array(pages)[seq], self.positions)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def attended(self, q, k, v, scale):
        got, at = [], 0
        for c in self.counts:
            s = slice(at, at + c)
            got.append(ref.attention(q[s], k[s], v[s], np.arange(1, c + 1), scale, **ref.tile_bits(self.name)))
            at += c
        return [torch.cat(x) for x in zip(*got)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,group,d", [(2, 2, 128), (1, 1, 64), (2, 4, 256), (1, 3, 128), (3, 8, 64), (1, 6, 256), (2, 1, 128), (1, 16, 128)])
@pytest.mark.parametrize("counts,split", [([1], None), ([1, 1, 1], None), ([2, 33, 1, 64, 130], None), ([300], "1"), ([300, 40], "4"), ([520, 1, 9], "16")])
def test_prompts(ctx, monkeypatch, dtype, heads, group, d, counts, split):
    print(f"prompts {dtype} {heads} x {group} x {d} {counts} {split}", flush=True)
    if split:
        monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    x = Prompts(ctx, dtype, counts, heads, d, 21)
    q, k, v, gate = (x.randn(x.n, n, d) for n in (heads * group, heads, heads, heads * group))
    qd, kd, vd, gd = (t.cuda().flatten(1) for t in (q, k, v, gate))
    out = torch.full_like(qd, math.nan)
    x.pool.prompt_attention(qd, kd, vd, heads * group, 1 / math.sqrt(d), out)
    want, bound = x.attended(q, k, v, 1 / math.sqrt(d))
    ref.assert_within(out, want, bound, "prompts")
    x.pool.prompt_attention(qd, kd, vd, heads * group, 1 / math.sqrt(d), out, gate=gd)
    ref.assert_within(out, *ref.gated(want, bound, gate), "gated")
    x.pool.close()


@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f32", 2, 1, 128), ("f16", 1, 4, 64), ("bf16", 4, 2, 256)])
def test_many_prompts(ctx, dtype, heads, group, d):
    """More tiles than the chip holds at once, one prompt far longer than the others."""
    print(f"many {dtype} {heads} {group} {d}", flush=True)
    counts = [40 + 13 * (i % 17) for i in range(100)] + [2100] + [1] * 20
    x = Prompts(ctx, dtype, counts, heads, d, 22)
    q, k, v = (x.randn(x.n, n, d) for n in (heads * group, heads, heads))
    qd, kd, vd = (t.cuda().flatten(1) for t in (q, k, v))
    out = torch.full_like(qd, math.nan)
    x.pool.prompt_attention(qd, kd, vd, heads * group, 0.1, out)
    again = torch.empty_like(out)
    x.pool.prompt_attention(qd, kd, vd, heads * group, 0.1, again)
    assert torch.equal(out, again) and torch.isfinite(out).all()
    at = np.concatenate([[0], np.cumsum(counts)])
    for i in (0, 16, 99, 100, 120):  # some of them in 64 bits, of the long one its last rows
        s = slice(at[i], at[i + 1])
        rows = np.arange(counts[i])[-50:]
        want = ref.attention(q[s][rows], k[s], v[s], rows + 1, 0.1, **ref.tile_bits(dtype))
        ref.assert_within(out[s][rows.tolist()], *want, f"prompt {i}")
    x.pool.close()


@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f16", 2, 4, 64), ("f32", 1, 2, 128), ("bf16", 1, 1, 256), ("f16", 1, 4, 128)])
@pytest.mark.parametrize("gap,odd", [(0, 0), (8, 0), (3, 1)])
def test_parts_of_wider_rows(ctx, dtype, heads, group, d, gap, odd):
    """Queries, keys and values as parts of one projection's rows, at any alignment; what is between
    them is not read."""
    print(f"strided {dtype} {heads} {group} {d} gap {gap} odd {odd}", flush=True)
    x = Prompts(ctx, dtype, [70, 5], heads, d, 23)
    qf, kf = heads * group * d, heads * d
    wide = torch.full((x.n, qf + 2 * kf + gap + odd), math.nan, dtype=x.dtype, device="cuda")
    q, k, v = x.randn(x.n, heads * group, d), x.randn(x.n, heads, d), x.randn(x.n, heads, d)
    parts = [wide[:, odd:odd + qf], wide[:, odd + qf:odd + qf + kf], wide[:, odd + qf + kf:odd + qf + 2 * kf]]
    for part, t in zip(parts, (q, k, v)):
        part.copy_(t.flatten(1))
    out = torch.full((x.n * qf + odd,), math.nan, dtype=x.dtype, device="cuda")[odd:].view(x.n, qf)
    x.pool.prompt_attention(*parts, heads * group, 0.1, out)
    ref.assert_within(out, *x.attended(q, k, v, 0.1), "strided")
    x.pool.close()


@pytest.mark.parametrize("scale", [0.0, -0.15, 2.0])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256)])
def test_scales(ctx, scale, dtype, d):
    x = Prompts(ctx, dtype, [90, 33], 1, d, 24)
    q, k, v = x.randn(x.n, 2, d), x.randn(x.n, 1, d), x.randn(x.n, 1, d)
    out = torch.empty_like(q.cuda().flatten(1))
    x.pool.prompt_attention(*(t.cuda().flatten(1) for t in (q, k, v)), 2, scale, out)
    ref.assert_within(out, *x.attended(q, k, v, scale), f"scale {scale}")
    x.pool.close()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,d,split", [("bf16", 128, None), ("f16", 64, None), ("f32", 128, None), ("f16", 256, "4"), ("bf16", 128, "4")])
def test_what_is_not_attended_weighs_nothing(ctx, monkeypatch, bad, dtype, d, split):
    """A value and a key that are not finite reach the rows behind them in their prompt alone."""
    if split:
        monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    x = Prompts(ctx, dtype, [100, 200, 60], 2, d, 25)
    q, k, v = x.randn(x.n, 4, d), x.randn(x.n, 2, d), x.randn(x.n, 2, d)
    clean = x.attended(q, k, v, 0.1)
    row = 100 + 150
    k[row, 0, 3], v[row, 1, 7] = math.nan, bad
    out = torch.empty_like(q.cuda().flatten(1))
    x.pool.prompt_attention(*(t.cuda().flatten(1) for t in (q, k, v)), 4, 0.1, out)
    got = out.cpu().view(x.n, 4, d)
    lost = torch.zeros(x.n, 4, d, dtype=torch.bool)
    lost[row:300, :2] = True  # a NaN score
    lost[row:300, 2:, 7] = True
    assert not torch.isfinite(got[lost].float()).any()
    if math.isinf(bad):
        assert torch.equal(got[row:300, 2:, 7].double(), torch.full((50, 2), bad, dtype=torch.float64))
    ref.assert_within(torch.where(lost, 0, got), torch.where(lost, 0.0, clean[0]), torch.where(lost, 0.0, clean[1]), "the others")
    x.pool.close()


def test_what_is_refused(ctx):
    x = Prompts(ctx, "bf16", [9, 4], 2, 64, 26)
    rows, out = torch.zeros(13, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(13, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="one stride"):
        x.pool.prompt_attention(rows, torch.zeros(13, 300, dtype=torch.bfloat16, device="cuda")[:, :128], rows, 2, 1.0, out)
    with pytest.raises(ValueError, match="side by side"):
        x.pool.prompt_attention(rows, torch.zeros(128, 13, dtype=torch.bfloat16, device="cuda").t(), rows, 2, 1.0, out)
    for first in ([3, 0], [0, 1]):  # a chunk among the prompts
        x.pool.upload([0, 1], [0] * 4 + [1] * 3, [1] * 7, [*range(first[0], first[0] + 4), *range(first[1], first[1] + 3)])
        with pytest.raises(ckv.CkvError) as refused:
            x.pool.prompt_attention(rows[:7], rows[:7], rows[:7], 2, 1.0, out[:7])
        assert refused.value.name == "ckv.invalid_argument"
    x.pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,q_heads,d,rotary,rows", [(2, 4, 128, 0, 50), (1, 3, 96, 40, 7), (2, 2, 256, 64, 333), (1, 1, 10, 6, 5), (8, 16, 128, 128, 1), (3, 0, 33 * 2, 0, 18)])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rotations_of_wider_pools(ctx, dtype, heads, q_heads, d, rotary, rows, layout):
    """Any head width: rows rotated, in place too; keys and values in the slots and in held rows."""
    print(f"rotate {dtype} {heads} {q_heads} {d} {rotary} {rows} {layout}", flush=True)
    x = Prompts(ctx, dtype, [rows], heads, d, 27)
    rotation = ckv.Rotation(3e4, rotary, layout, "bands", 4.0, 1.0, 4.0, 512)
    n = -(-rows // 16)
    cache = [torch.full((n * 16, heads * d), 7.0, dtype=x.dtype, device="cuda") for _ in range(2)]
    pool = ckv.Pool(ctx, 1, n, 16, heads, d, x.dtype, *cache)
    slots = np.random.RandomState(3).permutation(n * 16)[:rows]
    pool.upload(np.arange(n), [0] * rows, [n] * rows, x.positions, slots)
    q, k, v = x.randn(rows, max(q_heads, 1), d), x.randn(rows, heads, d), x.randn(rows, heads, d)
    qd, kd, vd = (t.cuda().flatten(1) for t in (q, k, v))
    turned, held = torch.empty_like(qd), [torch.empty_like(kd), torch.empty_like(kd)]
    pool.rotate_append(0, rotation, qd if q_heads else None, turned if q_heads else None, q_heads, kd, vd, *held)
    k64, room = ref.rotated(k, x.positions, rotation)
    at = torch.from_numpy(slots).cuda()
    ref.assert_within(cache[0][at], k64, room, "cached keys")
    assert torch.equal(cache[1][at], vd) and torch.equal(held[1], vd) and torch.equal(held[0], cache[0][at])
    rest = torch.ones(n * 16, dtype=torch.bool)
    rest[slots] = False
    assert all(bool((c[rest.cuda()] == 7).all()) for c in cache)
    q64, room = ref.rotated(q, x.positions, rotation)
    if q_heads:
        ref.assert_within(turned, q64, room, "queries")
    out = torch.empty_like(qd)
    pool.rotate(rotation, qd, out, q.shape[1])
    ref.assert_within(out, q64, room, "rotate")
    pool.rotate(rotation, qd, qd, q.shape[1])
    assert torch.equal(qd, out)
    if q_heads:
        again = q.cuda().flatten(1)
        pool.rotate_append(0, rotation, again, again, q_heads, kd, vd)
        assert torch.equal(again, turned)
        plain = torch.empty_like(again)
        pool.rotate_append(0, None, again, plain, q_heads, kd, vd)
        assert torch.equal(plain, again) and torch.equal(cache[0][at], kd)
    pool.close()
    x.pool.close()


@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f32", 1, 4, 64), ("f16", 2, 3, 256), ("bf16", 1, 2, 96)])
def test_steps_on_wider_pools(ctx, dtype, heads, group, d):
    """rotate_append_decode is rotate_append and the attention, on pools of 16-bit and float rows."""
    rotation, n = ckv.Rotation(1e4, 0, "pairs", "yarn", 4.0, original=64), 40
    x = Prompts(ctx, dtype, [n], heads, d, 28)
    pages = -(-n // 16)
    cache = [x.randn(pages * 16, heads * d).cuda() for _ in range(2)]
    pool = ckv.Pool(ctx, 1, pages, 16, heads, d, x.dtype, *cache)
    pool.upload(np.arange(pages), [0], [pages], [n - 1], [n - 1])
    q, k, v, gate = (x.randn(1, h, d).cuda().flatten(1) for h in (heads * group, heads, heads, heads * group))
    out, held, turned, two = torch.empty_like(q), [torch.empty_like(k) for _ in range(2)], torch.empty_like(q), torch.empty_like(q)
    pool.rotate_append_decode(0, rotation, k, v, q, heads * group, 0.1, out, gate, *held)
    first = [c.clone() for c in cache]
    assert torch.equal(held[0], cache[0][n - 1:n]) and torch.equal(held[1], v)
    pool.rotate_append(0, rotation, q, turned, heads * group, k, v)
    pool.attention_gated(0, turned, heads * group, 0.1, gate, two)
    assert torch.equal(two, out) and all(torch.equal(a, b) for a, b in zip(first, cache))
    q64, _ = ref.rotated(turned.cpu().view(1, -1, d), [0], ckv.Rotation(1e4))  # (as it is: a turn by nothing)
    seen = [c[:n].cpu().view(n, heads, d) for c in cache]
    want, bound = ref.attention(q64, *seen, [n], 0.1, **ref.tile_bits(dtype))
    ref.assert_within(out, *ref.gated(want, bound, gate.cpu().view(1, -1, d)), "step")
    pool.close()
    x.pool.close()


def test_captured_prompts():
    """A captured prompt launch replays on new rows; a batch's first is refused under capture, which
    goes on."""
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        x = Prompts(own, "bf16", [900, 40], 2, 128, 29)
        q, k, v = (x.randn(x.n, h, 128).cuda().flatten(1) for h in (4, 2, 2))
        out = torch.empty_like(q)
        call = lambda: x.pool.prompt_attention(q, k, v, 4, 0.09, out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(ckv.CkvError) as refused:
                call()
            assert refused.value.name == "ckv.invalid_argument"
            out.zero_()
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(4):
            for t in (q, k, v):
                t.normal_()
            call()
            stream.synchronize()
            want = out.clone()
            out.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want)
        x.pool.close()
    own.close()


@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f16", 1, 4, 256), ("f32", 2, 1, 64)])
def test_a_run_of_them(ctx, dtype, heads, group, d):
    """Prompts, further chunks and single tokens of a model of two layers, as a program runs them: every
    output attends exactly what the pool holds, whichever call put it there."""
    print(f"run {dtype} {heads} {group} {d}", flush=True)
    cache = ref.Cache(ctx, dtype, [150, 61, 33], heads, d, layers=2, seed=30)
    pool, scale, hq = cache.pool, 1 / math.sqrt(d), heads * group
    rotation = ckv.Rotation(1e5, d // 2, "halves", "yarn", 4.0, original=64)
    done = [0, 0, 0]
    for counts in ([70, 18, 30], [33, 40, 0], [1, 1, 1], [1, 0, 1], [40, 1, 1], [1, 1, 0], [1, 0, 0]):
        positions = cache.upload(done, counts)
        prompts = not any(done)
        for layer in range(2):
            q, k, v = (cache.randn(sum(counts), h, d) for h in (hq, heads, heads))
            qd, kd, vd = (t.cuda().flatten(1) for t in (q, k, v))
            out, turned = torch.empty_like(qd), torch.empty_like(qd)
            q64, _ = ref.rotated(q, positions, rotation)
            k64, _ = ref.rotated(k, positions, rotation)
            cache.keep(layer, k64, v)
            if max(counts) == 1:
                pool.rotate_append_decode(layer, rotation, kd, vd, qd, hq, scale, out)
                want, bound = cache.attended(q64, scale, layer, **ref.decode_bits(dtype))
                bound = bound + cache.attended(q64, scale, layer, q_half=24 * ref.STEP32)[1]
            else:
                held = [torch.empty_like(kd) for _ in range(2)]
                pool.rotate_append(layer, rotation, qd, turned, hq, kd, vd, *held)
                if prompts:
                    pool.prompt_attention(turned, *held, hq, scale, out)
                else:
                    pool.attention(layer, turned, hq, scale, out)
                q64 = turned.cpu().double().view(q.shape)  # as the attention reads them
                want, bound = cache.attended(q64, scale, layer, **ref.tile_bits(dtype))
            ref.assert_within(out, want, bound, f"layer {layer} {counts}")
        done = [a + b for a, b in zip(done, counts)]
    cache.lengths = done
    for layer in range(2):
        cache.check(layer, "at the end")
    pool.close()


@pytest.mark.parametrize("heads,group,d", [(2, 2, 128), (1, 4, 64), (1, 1, 256)])
def test_floats_past_the_largest_bf16(ctx, heads, group, d):
    """Numbers between bf16's largest and float's own round to an infinity as bf16 terms: the rows that
    attend them are right all the same, as are numbers that leave nothing in the lower terms."""
    print(f"large floats {heads} {group} {d}", flush=True)
    x = Prompts(ctx, "f32", [70, 150], heads, d, 36)
    q, k, v = x.randn(x.n, heads * group, d), x.randn(x.n, heads, d), x.randn(x.n, heads, d)
    v[90, 0, 3] = torch.finfo(torch.float32).max
    v[20, 0, 5] = -torch.finfo(torch.float32).max * 0.9999
    v[30:40] = torch.round(v[30:40])
    v[100, 0, 9] = 2.0 ** -140
    out = torch.empty_like(q.cuda().flatten(1))
    x.pool.prompt_attention(*(t.cuda().flatten(1) for t in (q, k, v)), heads * group, 0.1, out)
    ref.assert_within(out, *x.attended(q, k, v, 0.1), "large floats")
    x.pool.close()


def test_terms_keep_their_bits(ctx):
    """Values that cancel: float rows' results are those of 24 bits, not of one bf16 term or two."""
    x = Prompts(ctx, "f32", [64], 1, 128, 37)
    q, k = torch.zeros(64, 1, 128), torch.zeros(64, 1, 128)
    v = x.randn(64, 1, 128)
    v[1::2] = -v[::2] * (1 - 2.0 ** -14)  # pairs leave 2^-14 of themselves
    out = torch.empty(64, 128, device="cuda")
    x.pool.prompt_attention(q.cuda().flatten(1), k.cuda().flatten(1), v.cuda().flatten(1), 1, 1.0, out)
    # equal weights of 2^-1 .. 2^-6 at these rows: means of what floats hold, summed in 32 bits
    for r in (1, 3, 7, 15, 31, 63):
        want = v[:r + 1, 0].double().mean(0)
        room = (r + 4) * 2.0 ** -23 * v[:r + 1, 0].double().abs().mean(0)
        assert ((out[r].cpu().double() - want).abs() <= room).all(), r
    x.pool.close()
