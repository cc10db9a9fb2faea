"""Compaction against its definition: kept tokens in place and in other pages, keys turned to their
new positions, values bit for bit, everything else untouched; and the attention that reads it."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context
from tests.operator_ref import Cache, assert_within, attention, frequencies, seen, turned, turned_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def kept_tokens(pattern, n, rng):
    if pattern == "middle":
        return np.concatenate([np.arange(min(4, n)), np.arange(max(4, n // 2), n)])
    if pattern == "one":  # a single token near the front leaves: every other is read by its neighbour's move
        return np.delete(np.arange(n), min(3, n - 1))
    if pattern == "all":
        return np.arange(n)
    pick = rng.rand(n) < 0.5
    pick[n - 1] = True
    return np.flatnonzero(pick)


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("pattern", ["middle", "one", "scattered", "all"])
@pytest.mark.parametrize("dtype,heads,d,rotary,page,layers", [
    ("bf16", 8, 128, 0, 16, 3), ("f16", 2, 256, 64, 16, 2), ("f32", 2, 128, 0, 16, 2), ("bf16", 1, 80, 32, 16, 2),
    ("f32", 1, 33, None, 7, 1), ("f16", 3, 130, 66, 5, 2), ("bf16", 2, 64, 48, 16, 4), ("f16", 1, 512, 512, 16, 1)])
def test_compact(ctx, dtype, heads, d, rotary, page, layers, pattern, fresh):
    print(f"compact {dtype} {heads} x {d} rotary {rotary} page {page} {pattern} fresh {fresh}", flush=True)
    rng = np.random.RandomState(d)
    lengths = [1, 5, 40, 300, 1031 if heads * layers < 12 else 700]
    kept = [kept_tokens(pattern, n, rng) for n in lengths]
    spare = sum(-(-x.size // page) for x in kept) + 2
    cache = Cache(ctx, dtype, lengths, heads, d, page=page, layers=layers, spare=spare, seed=d)
    pool = cache.to_device()
    tables, at = cache.tables, 0
    if fresh:
        tables = []
        for x in kept:
            need = -(-x.size // page)
            tables.append(cache.free[at:at + need])
            at += need
    source = np.concatenate([cache.slots(t, x) for t, x in zip(cache.tables, kept)])
    target = np.concatenate([cache.slots(t, np.arange(x.size)) for t, x in zip(tables, kept)])
    shift = None if rotary is None else np.concatenate([np.arange(x.size) - x for x in kept])
    theta = 1e4
    pool.compact(source, target, [x.size for x in kept], shift, theta, rotary or 0)
    ctx.sync()
    before = cache.k[:, source].clone()
    cache.v[:, target] = cache.v[:, source].clone()
    cache.k[:, target] = cache.kd.cpu()[:, target]
    cache.unchanged()  # values bit for bit, the rest as it was
    got = cache.kd.cpu()[:, target]
    width = 0 if rotary is None else rotary or d
    still = np.ones(source.size, bool) if shift is None else shift == 0
    assert torch.equal(got[:, still], before[:, still]) and torch.equal(got[..., width:], before[..., width:])
    if width:
        angle = torch.from_numpy(shift[:, None].astype(np.float64)) * frequencies(theta, width)
        for layer in range(layers):
            want, bound = turned(before[layer], angle, width), turned_bound(before[layer], width)
            assert_within(got[layer][~still], want[~still], bound[~still], f"layer {layer}")
    pool.close()


def test_shifts_of_any_size_and_sign(ctx):
    """Keys turned in place by shifts as far as 32 bits go."""
    n, d = 64, 128
    cache = Cache(ctx, "f32", [n], 2, d, seed=3)
    pool = cache.to_device()
    slots = cache.slots(cache.tables[0], np.arange(n))
    rng = np.random.RandomState(1)
    shift = rng.randint(-100_000, 100_000, n)
    shift[:4] = [2147483647, -2147483648, 1, -1]
    pool.compact(slots, slots, [n], shift, 1e6)
    ctx.sync()
    angle = torch.from_numpy(shift[:, None].astype(np.float64)) * frequencies(1e6, d)
    bound = turned_bound(cache.k[0, slots], d)
    bound += (angle.abs() * 2.0 ** -50).repeat(1, 2)[:, None] * float(cache.k[0, slots].abs().max()) * 2
    assert_within(cache.kd[0, slots], turned(cache.k[0, slots], angle, d), bound, "turned keys")
    cache.v[0, slots] = cache.vd.cpu()[0, slots]
    pool.close()


def test_refused_moves_change_nothing(ctx):
    cache = Cache(ctx, "bf16", [50], 2, 128, seed=3)
    pool = cache.to_device()
    a = cache.slots(cache.tables[0], np.arange(50))
    for source, target, name in ((a[:3], a[1:4], "tensor_op.unsupported_aliasing"),
                                 (a[:2], a[[7, 7]], "tensor_op.unsupported_aliasing"),
                                 (a[:2], [a[3], 10 ** 6], "tensor_op.cache_slot_out_of_range")):
        with pytest.raises(ckv.CkvError) as e:
            pool.compact(source, target, [len(source)], [0] * len(source), 1e4)
        assert e.value.name == name
    ctx.sync()
    cache.unchanged()
    pool.close()


def test_a_chat_that_outgrows_its_cache(ctx):
    """As they are used together: a prompt rotated and appended, decode steps through a window, the
    cache compacted (the sinks and the newest half stay), and steps on the compacted cache at the new
    positions. Every step's output is the definition's over what the cache holds."""
    heads, group, d, window, sinks, theta = 2, 2, 128, 40, 4, 1e4
    cache = Cache(ctx, "bf16", [200], heads, d, seed=11)
    pool = cache.to_device()
    scale, axis = 1 / math.sqrt(d), ckv.rope_pair_axes([24, 20, 20], True)
    held = 0

    def rows(n):
        return [cache.randn(n, x, d).cuda().flatten(1) for x in (heads * group, heads, heads)]

    def check(out, q, first):
        slots = cache.slots(cache.tables[0], np.arange(held))
        k, v = cache.kd[0, slots].cpu(), cache.vd[0, slots].cpu()
        for i in range(out.shape[0]):
            t = seen(first + i, window, sinks)
            want, bound = attention(q[i:i + 1].view(1, heads * group, d).cpu(), k[t], v[t], [np.arange(len(t))], scale, p_bits=16)
            assert_within(out[i].view(1, heads * group, d), want, bound, f"position {first + i}")

    def step(n):  # n tokens appended behind `held`, rotated on three axes, attended
        nonlocal held
        cache.upload([held], [n])
        pool.upload_axes(np.stack([np.arange(held, held + n)] * 3))
        q, k, v = rows(n)
        rq, out = torch.empty_like(q), torch.empty_like(q)
        pool.rope_axes_append(0, q, rq, heads * group, k, v, theta, axis)
        pool.attention_window(0, rq, heads * group, scale, window, out, sinks=sinks)
        ctx.sync()
        held += n
        check(out, rq, held - n)

    step(130)
    for _ in range(3):
        step(1)
    keep = np.concatenate([np.arange(sinks), np.arange(held // 2, held)])
    before = cache.kd[0, cache.slots(cache.tables[0], keep)].cpu()
    pool.compact(cache.slots(cache.tables[0], keep), cache.slots(cache.tables[0], np.arange(keep.size)), [keep.size],
                 np.arange(keep.size) - keep, theta)
    ctx.sync()
    held = keep.size
    angle = torch.from_numpy((np.arange(keep.size) - keep)[:, None].astype(np.float64)) * frequencies(theta, d)
    got = cache.kd[0, cache.slots(cache.tables[0], np.arange(held))]
    assert_within(got, turned(before, angle, d), turned_bound(before, d), "turned keys")
    for n in (1, 1, 25, 1):
        step(n)
    pool.close()
