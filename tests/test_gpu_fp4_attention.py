"""Attention over pools held in 4 bits against 64 bits: decode rows and tiles over every head layout,
page size and plan, masked infinities and NaN, device tables, other streams."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests import fp4_ref as ref
from tests.gpu_util import force_plan, new_context

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def attend(cache, q, scale, layer=0, gate=None):
    x = q.cuda().flatten(1)
    out = torch.full_like(x, math.nan)
    if gate is None:
        cache.pool.attention(layer, x, q.shape[1], scale, out)
    else:
        cache.pool.attention_gated(layer, x, q.shape[1], scale, gate.cuda().flatten(1), out)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page", [(2, 2, 128, 16), (1, 1, 64, 16), (3, 3, 128, 32), (2, 4, 256, 16), (1, 6, 64, 64),
                                                (2, 8, 128, 16), (1, 9, 256, 32), (2, 16, 128, 16), (8, 1, 128, 16), (1, 33, 64, 16)])
@pytest.mark.parametrize("lengths,split", [([1], None), ([1, 2, 15, 16, 17, 31, 32, 33, 48], None), ([700, 3, 97], None),
                                           ([700, 3, 97, 260], "1"), ([700, 3, 97, 1, 64], "b3"), ([500, 500], "0")])
def test_decode_rows(ctx, monkeypatch, dtype, heads, group, d, page, lengths, split):
    print(f"decode {dtype} {heads} x {group} x {d} pages of {page}: {lengths} {split}", flush=True)
    force_plan(monkeypatch, split)
    cache = ref.Cache(ctx, dtype, lengths, heads, d, page=page, seed=11)
    cache.fill()
    cache.upload([n - 1 for n in lengths], [1] * len(lengths), with_slots=False)
    q = cache.randn(len(lengths), heads * group, d)
    out = attend(cache, q, 1 / math.sqrt(d))
    want, bound = cache.attended(q, 1 / math.sqrt(d), **ref.decode_bits(dtype))
    ref.assert_within(out, want, bound, "decode")
    gate = cache.randn(*q.shape)
    ref.assert_within(attend(cache, q, 1 / math.sqrt(d), gate=gate), *ref.gated(want, bound, gate), "gated")
    cache.pool.close()


@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f16", 1, 8, 256), ("f32", 2, 1, 64), ("bf16", 8, 4, 64)])
def test_long_and_many_rows(ctx, dtype, heads, group, d):
    """Rows of one to thousands of tokens in one batch, and more rows than the chip holds at once."""
    print(f"long {dtype} {heads} {group} {d}", flush=True)
    lengths = [9001, 1, 2500] + [40 + 7 * i for i in range(60)]
    cache = ref.Cache(ctx, dtype, lengths, heads, d, seed=12)
    cache.fill()
    cache.upload([n - 1 for n in lengths], [1] * len(lengths), with_slots=False)
    q = cache.randn(len(lengths), heads * group, d)
    first = attend(cache, q, 0.09)
    ref.assert_within(first, *cache.attended(q, 0.09, **ref.decode_bits(dtype)), "long")
    assert torch.equal(attend(cache, q, 0.09), first)  # the same bits each time
    cache.pool.close()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dtype,group,d,counts", [("bf16", 2, 128, [1, 1, 1]), ("f32", 3, 64, [1, 1, 1]), ("f16", 4, 256, [40, 1, 70]),
                                                  ("bf16", 1, 64, [40, 1, 70]), ("f32", 2, 128, [40, 1, 70])])
def test_scales(ctx, scale, dtype, group, d, counts):
    """Equal weights, the least of the products, and weights of almost one key alone."""
    print(f"scale {scale} {dtype} {group} {d} {counts}", flush=True)
    cache = ref.Cache(ctx, dtype, [80, 33, 300], 2, d, seed=13)
    cache.fill()
    cache.upload([n - c for n, c in zip(cache.lengths, counts)], counts, with_slots=False)
    q = cache.randn(sum(counts), 2 * group, d)
    bits = ref.decode_bits(dtype) if max(counts) == 1 else ref.tile_bits(dtype)
    ref.assert_within(attend(cache, q, scale), *cache.attended(q, scale, **bits), f"scale {scale}")
    cache.pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page", [(2, 2, 128, 16), (1, 1, 64, 32), (2, 4, 256, 16), (1, 3, 128, 64), (3, 8, 64, 16), (1, 6, 256, 16)])
@pytest.mark.parametrize("first,counts,split", [([0, 5, 31], [2, 33, 1], None), ([45, 900], [130, 64], None), ([0], [300], "1"),
                                                ([700, 20], [40, 70], "5"), ([1500], [65], "16")])
def test_chunks(ctx, monkeypatch, dtype, heads, group, d, page, first, counts, split):
    print(f"chunk {dtype} {heads} x {group} x {d} pages of {page}: {first} {counts} {split}", flush=True)
    if split:
        monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    cache = ref.Cache(ctx, dtype, [f + c for f, c in zip(first, counts)], heads, d, page=page, seed=14)
    cache.fill()
    cache.upload(first, counts, with_slots=False)
    q = cache.randn(sum(counts), heads * group, d)
    out = attend(cache, q, 1 / math.sqrt(d))
    want, bound = cache.attended(q, 1 / math.sqrt(d), **ref.tile_bits(dtype))
    ref.assert_within(out, want, bound, "chunk")
    gate = cache.randn(*q.shape)
    ref.assert_within(attend(cache, q, 1 / math.sqrt(d), gate=gate), *ref.gated(want, bound, gate), "gated")
    cache.pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,group,split", [(128, 2, None), (64, 1, None), (256, 4, None), (128, 4, "4")])
def test_what_is_not_attended_weighs_nothing(ctx, monkeypatch, dtype, d, group, split):
    """Blocks of NaN in keys and values, attended by the rows behind them alone, there in their head
    alone; NaN beyond a sequence's end and in pages of nobody."""
    if split:
        monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    n, bad = 200, 150
    cache = ref.Cache(ctx, dtype, [n], 2, d, seed=15)

    def make(*shape):
        x = cache.randn(*shape)
        x[bad, 1, 5] = math.inf if len(cache.rows) % 2 else math.nan
        return x

    cache.fill(make=make)
    q = cache.randn(n, 2 * group, d)
    cache.upload([0], [n], with_slots=False)
    out = attend(cache, q, 0.1)
    want, bound = cache.attended(q, 0.1, **ref.tile_bits(dtype))
    mine = torch.zeros(n, 2 * group, d, dtype=torch.bool)
    mine[bad:, group:] = True  # rows that attend the bad token, in its head: a NaN score spoils all of the row
    got = out.cpu().view(n, 2 * group, d)
    assert torch.isnan(got[mine].float()).all() and torch.isfinite(got[~mine].float()).all()
    ref.assert_within(torch.where(mine, 0, got), torch.where(mine, 0.0, want), torch.where(mine, 0.0, bound), "the others")
    for last in (bad - 1, bad, n - 1):
        cache.upload([last], [1], with_slots=False)
        one = attend(cache, q[last:last + 1], 0.1).cpu().view(2 * group, d).float()
        assert torch.isfinite(one[:group]).all()
        assert torch.isnan(one[group:]).all() if last >= bad else torch.isfinite(one[group:]).all()
    cache.pool.close()


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 1, 64), ("f16", 8, 256)])
@pytest.mark.parametrize("first,counts", [([700, 15, 0, 333], [1, 1, 1, 1]), ([700, 15, 0], [90, 1, 40])])
def test_device_tables_and_patched_pages(ctx, dtype, group, d, first, counts):
    """The same rows by uploaded tables and by the sequence tables on the device: the same bits, and
    the same cache after appends by either."""
    print(f"device tables {dtype} {group} {d} {counts}", flush=True)
    cache = ref.Cache(ctx, dtype, [f + c for f, c in zip(first, counts)], 2, d, seed=16)
    cache.fill()
    q, outs = cache.randn(sum(counts), 2 * group, d), []
    cache.upload(first, counts)
    outs.append(attend(cache, q, 0.1))
    moved, old = cache.free[0], cache.tables[0][0]  # the first page elsewhere, by a patch
    cache.pool.copy_blocks([old], [moved])
    cache.pool.patch([0], [moved])
    outs.append(attend(cache, q, 0.1))
    cache.pool.patch([0], [old])
    pool, ids = cache.pool, [3, 1, 4, 0][:len(counts)]
    pool.reserve_sequences(5, 60)
    seq = np.repeat(ids, [t.size for t in cache.tables])
    index = np.concatenate([np.arange(t.size) for t in cache.tables])
    pool.update_sequences(seq, index, np.concatenate(cache.tables), ids, [t.size for t in cache.tables])
    pool.upload_batch(ids, first, counts)
    outs.append(attend(cache, q, 0.1))
    k, v = cache.randn(sum(counts), 2, d), cache.randn(sum(counts), 2, d)
    pool.append(0, k.cuda().flatten(1), v.cuda().flatten(1))
    cache.keep(0, k, v)
    outs.append(attend(cache, q, 0.1))
    cache.upload(first, counts)
    cache.check(0, "appended by device tables")
    outs.append(attend(cache, q, 0.1))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and torch.equal(outs[3], outs[4])
    bits = ref.decode_bits(dtype) if max(counts) == 1 else ref.tile_bits(dtype)
    ref.assert_within(outs[3], *cache.attended(q, 0.1, **bits), "after the append")
    cache.pool.close()


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 5, 64), ("f16", 1, 256), ("bf16", 16, 128)])
@pytest.mark.parametrize("scaled", [None, "plain", "yarn"])
def test_steps(ctx, dtype, group, d, scaled):
    """A decode step in one call: the cache, the held rows and the output; and by the older calls."""
    print(f"step {dtype} {group} {d} {scaled}", flush=True)
    lengths = [1, 90, 16, 17, 333]
    cache = ref.Cache(ctx, dtype, lengths, 2, d, layers=3, seed=17)
    for layer in range(3):
        cache.fill(layer)
    n, scale = len(lengths), 1 / math.sqrt(d)
    positions = cache.upload([x - 1 for x in lengths], [1] * n)
    q, k, v, gate = (cache.randn(n, x, d) for x in (2 * group, 2, 2, 2 * group))
    dev = [x.cuda().flatten(1) for x in (q, k, v, gate)]
    rotation = {None: None, "plain": ckv.Rotation(1e5, 32), "yarn": ckv.Rotation(1e5, 0, "pairs", "yarn", 4.0, original=128)}[scaled]
    if rotation is None:
        q64, room, k64 = q.double(), 0.0, k.double()
    else:
        q64, room = ref.rotated(q, positions, rotation)
        k64, _ = ref.rotated(k, positions, rotation)
    out, held = torch.empty_like(dev[0]), [torch.empty_like(dev[1]) for _ in range(2)]
    kept = dev[0].clone()
    cache.pool.rotate_append_decode(0, rotation, dev[1], dev[2], dev[0], 2 * group, scale, out, dev[3], *held)
    cache.keep(0, k64, v)
    cache.check(0, "cache")
    assert torch.equal(dev[0], kept)
    for got, want in zip(held, (cache.k, cache.v)):
        assert torch.equal(got.cpu().double().view(n, 2, d), want[0, cache.at])
    # rotated queries enter with 16 bits (24 with float rows), and the rotation's own error
    want, bound = cache.attended(q64, scale, **ref.decode_bits(dtype))
    if rotation is not None:
        _, more = cache.attended(q64, scale, q_half=6 * ref.STEP32 * 4)
        bound = bound + more
    ref.assert_within(out, *ref.gated(want, bound, gate), "step")
    if scaled == "plain":
        older = torch.empty_like(out)
        cache.pool.rope_append_decode(1, dev[1], dev[2], dev[0], 2 * group, scale, 1e5, older, 32)
        cache.keep(1, k64, v)
        cache.check(1, "the older call")
        w, b = cache.attended(q64, scale, 1, **ref.decode_bits(dtype))
        ref.assert_within(older, w, b + cache.attended(q64, scale, 1, q_half=6 * ref.STEP32 * 4)[1], "the older call")
    if scaled is None:
        older = torch.empty_like(out)
        cache.pool.append_decode(1, dev[1], dev[2], dev[0], 2 * group, scale, older)
        cache.keep(1, k64, v)
        cache.check(1, "append_decode")
        ref.assert_within(older, *cache.attended(q64, scale, 1, **ref.decode_bits(dtype)), "append_decode")
    cache.check(2, "another layer")
    cache.pool.close()


def test_on_another_stream_and_beside_another_pool():
    """A context whose stream changes, and two pools of one context whose launches alternate."""
    own = ckv.Context(0, stream=torch.cuda.current_stream())
    caches = [ref.Cache(own, "bf16", [900, 40], 2, 128, seed=18), ref.Cache(own, "f16", [3000], 1, 64, seed=19)]
    qs, wants = [], []
    for c in caches:
        c.fill()
        c.upload([n - 1 for n in c.lengths], [1] * len(c.lengths), with_slots=False)
        qs.append(c.randn(len(c.lengths), 4, c.d))
        wants.append(c.attended(qs[-1], 0.1, **ref.decode_bits(c.name)))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.current_stream(), other, torch.cuda.current_stream(), other):
        own.set_stream(stream)
        with torch.cuda.stream(stream):
            outs = [[attend(c, q, 0.1) for c, q in zip(caches, qs)] for _ in range(3)]
            stream.synchronize()
        for both in outs:
            for out, (want, bound) in zip(both, wants):
                ref.assert_within(out, want, bound, "alternating")
    for c in caches:
        c.pool.close()
    own.close()
