"""Windowed attention, rotation on several axes and compaction where batches come by other ways:
tables kept on the device, pages given back by patches, pools past 4 GiB, sequences that move
nothing, calls on another stream."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context
from tests.operator_ref import Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def bits(x):
    return x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 8, 128), ("f16", 4, 256), ("bf16", 2, 96)])
@pytest.mark.parametrize("first,counts", [([700, 15, 0, 333], [1, 1, 1, 1]), ([700, 15, 0], [90, 1, 40])])
def test_device_tables_and_patched_pages(ctx, dtype, group, d, first, counts):
    """The same rows by uploaded tables, by the sequence tables on the device, and once the pages
    that no row attends were given back by a patch: the same bits."""
    print(f"device tables {dtype} group {group} d {d} rows {counts}", flush=True)
    heads, window, sinks, rows = 2, 50, 4, sum(counts)
    cache = Cache(ctx, dtype, [f + c for f, c in zip(first, counts)], heads, d, seed=21)
    pool = cache.to_device()
    q = cache.randn(rows, heads * group, d).cuda().flatten(1)
    scale, outs = 1 / math.sqrt(d), []

    def attend(w=window):
        out = torch.full_like(q, math.nan)
        pool.attention_window(0, q, heads * group, scale, w, out, sinks=sinks)
        outs.append(out)

    cache.upload(first, counts, slots=False)
    attend()
    attend(10_000)
    flat, at, trap = np.concatenate(cache.tables), 0, cache.free[0]
    gone = []
    for t, f, c in zip(cache.tables, first, counts):
        low = max(0, f - window + 1) // 16
        gone += [at + i for i in range(1, low)]
        at += t.size
    if gone:
        pool.patch(gone, [trap] * len(gone))
    attend()
    pool.reserve_sequences(5, 60)
    seq = np.repeat([3, 1, 4, 0][:len(counts)], [t.size for t in cache.tables])
    index = np.concatenate([np.arange(t.size) for t in cache.tables])
    pool.update_sequences(seq, index, flat, [3, 1, 4, 0][:len(counts)], [t.size for t in cache.tables])
    pool.upload_batch([3, 1, 4, 0][:len(counts)], first, counts, with_slots=False)
    attend()
    attend(10_000)
    ctx.sync()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[0], outs[3]) and torch.equal(outs[1], outs[4])
    assert torch.all(torch.isfinite(outs[0])) and not torch.equal(outs[0], outs[1])
    pool.close()


@pytest.mark.parametrize("dtype,heads,d,blocks", [("bf16", 8, 128, 70_000), ("f32", 8, 128, 36_000), ("f16", 2, 256, 140_000)])
def test_pools_past_four_gigabytes(ctx, dtype, heads, d, blocks):
    """The last pages of the second layer lie past 2^32 bytes: what the operators give there is what
    they give in a small pool, bit for bit."""
    print(f"far pages {dtype} {heads} x {d}", flush=True)
    lengths, page, got = [301, 40], 16, []
    for count in (90, blocks):
        cache = Cache(ctx, dtype, lengths, heads, d, layers=2, spare=90 - 19 - 3, seed=31)
        assert cache.blocks == 90
        shape = (2, count * page, heads * d)
        k = torch.empty(shape, dtype=cache.dtype, device="cuda")
        v = torch.empty_like(k)
        lift = count - 90  # the small pool's pages are the other's last
        for dev, host in ((k, cache.k), (v, cache.v)):
            dev[:, lift * page:] = host.flatten(2).cuda()
        if lift:
            assert k.numel() * k.element_size() > 2 ** 32 and (k.numel() // 2 + (count - 90) * page * heads * d) * k.element_size() > 2 ** 32
        pool = ckv.Pool(ctx, 2, count, page, heads, d, cache.dtype, k.view(-1), v.view(-1))
        tables = [t + np.uint32(lift) for t in cache.tables]
        flat, starts = np.concatenate(tables), [0, tables[0].size]
        scale, theta, axis = 1 / math.sqrt(d), 1e4, ckv.rope_pair_axes([d // 4, d // 4])

        def upload(first, counts):
            s = np.repeat([0, 1], counts)
            pos = np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)])
            slots = [int(tables[i][p // page]) * page + p % page for i, p in zip(s, pos)]
            pool.upload(flat, np.take(starts, s), [tables[i].size for i in s], pos, slots)
            pool.upload_axes(np.stack([pos, 2 * pos]))
            n = len(pos)
            return [cache.randn(n, x, d).cuda().flatten(1) for x in (2 * heads, heads, heads)]

        outs = []
        for first, counts in (([300, 39], [1, 1]), ([200, 0], [60, 30])):
            q, kr, vr = upload(first, counts)
            out, rotated = torch.empty_like(q), torch.empty_like(q)
            pool.rope_axes_append(1, q, rotated, 2 * heads, kr, vr, theta, axis)
            pool.attention_window(1, rotated, 2 * heads, scale, 77, out, sinks=4)
            outs += [rotated, out]
            if counts == [1, 1]:
                out = torch.empty_like(q)
                pool.append_decode_window(1, kr, vr, q, 2 * heads, scale, 77, out, sinks=4)
                outs.append(out)
        keep = np.concatenate([np.arange(4), np.arange(150, 301)])
        at = [int(tables[0][i // page]) * page + i % page for i in range(301)]
        pool.compact(np.take(at, keep), at[:keep.size], [keep.size], np.arange(keep.size) - keep, theta)
        ctx.sync()
        outs += [k[:, lift * page:], v[:, lift * page:]]
        got.append([bits(x.contiguous()).cpu() for x in outs])
        pool.close()
        del k, v, outs
        torch.cuda.empty_cache()
    for i, (small, far) in enumerate(zip(*got)):
        assert torch.equal(small, far), f"output {i}"


def test_sequences_that_move_nothing_and_shared_sources(ctx):
    """Counts of zero, moves to their own place, and one source for several targets."""
    cache = Cache(ctx, "bf16", [64, 30], 2, 128, layers=2, spare=8, seed=41)
    pool = cache.to_device()
    a, b = (cache.slots(t, np.arange(t.size * 16)) for t in cache.tables)
    fresh = cache.slots(cache.free, np.arange(cache.free.size * 16))
    source = np.concatenate([a[[40, 40, 41, 3]], b[:5], a[[7] * 20]])
    target = np.concatenate([a[[0, 1, 2, 3]], b[:5], fresh[:20]])
    # a[40] is read by two moves, and 20 fresh places take a[7]: of the sequence that reads both
    pool.compact(source[:4], target[:4], [0, 4, 0])
    pool.compact(source[4:], target[4:], [5, 0, 20])
    pool.compact([], [], [0, 0])
    ctx.sync()
    for x, dev in ((cache.k, cache.kd), (cache.v, cache.vd)):
        x[:, target] = x[:, source].clone()
    cache.unchanged()
    pool.close()


@pytest.mark.parametrize("rows", [1, 40])
def test_on_another_stream_and_back(ctx, rows):
    """A context whose stream changes between calls: plans and scratch made on one stream serve on
    the other."""
    own = ckv.Context(0, stream=torch.cuda.current_stream())
    cache = Cache(own, "bf16", [500, 90], 2, 128, seed=51)
    pool = cache.to_device()
    first = [500 - rows, 90 - rows]
    cache.upload(first, [rows] * 2, slots=False)
    pool.upload_axes(np.arange(4 * rows).reshape(2, -1))
    q = cache.randn(2 * rows, 4, 128).cuda().flatten(1)
    axis, other, outs = ckv.rope_pair_axes([32, 32]), torch.cuda.Stream(), []
    other.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), other, torch.cuda.current_stream(), other):
        own.set_stream(stream)
        with torch.cuda.stream(stream):
            rotated, out = torch.empty_like(q), torch.empty_like(q)
            pool.rope_axes(q, rotated, 4, 1e4, axis)
            pool.attention_window(0, rotated, 4, 0.1, 60, out, sinks=2)
            stream.synchronize()
            outs.append((rotated, out))
    for rotated, out in outs[1:]:
        assert torch.equal(rotated, outs[0][0]) and torch.equal(out, outs[0][1])
    pool.close()
    own.close()


def test_captured_axes_and_what_capture_refuses(ctx):
    """A captured rotation with append replays on new inputs; uploads of positions and compactions are
    refused under capture and leave it going."""
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    n, heads, d = 37, 2, 128
    cache = Cache(own, "bf16", [60], heads, d, seed=61)
    with torch.cuda.stream(stream):
        pool = cache.to_device()
        _, _, at = cache.upload([60 - n], [n])
        positions = np.stack([np.arange(n), 7 * np.arange(n), 3 + 0 * np.arange(n)])
        pool.upload_axes(positions)
        axis = ckv.rope_pair_axes([24, 20, 20], True)
        q, k, v = (cache.randn(n, x, d).cuda().flatten(1) for x in (2 * heads, heads, heads))
        rotated = torch.empty_like(q)
        slots = cache.slots(cache.tables[0], np.arange(20))
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pool.rope_axes_append(0, q, rotated, 2 * heads, k, v, 1e4, axis)
            for call in (lambda: pool.upload_axes(positions), lambda: pool.compact(slots[10:], slots[:10], [10])):
                with pytest.raises(ckv.CkvError) as refused:
                    call()
                assert refused.value.name == "ckv.invalid_argument"
        for _ in range(3):
            for x in (q, k, v):
                x.normal_()
            pool.rope_axes_append(0, q, rotated, 2 * heads, k, v, 1e4, axis)
            stream.synchronize()
            want = rotated.clone(), cache.kd[0, at].clone(), cache.vd[0, at].clone()
            rotated.zero_()
            cache.kd[0, at] = 0
            cache.vd[0, at] = 0
            graph.replay()
            stream.synchronize()
            for got, w in zip((rotated, cache.kd[0, at], cache.vd[0, at]), want):
                assert torch.equal(got, w)
        pool.compact(slots[10:], slots[:10], [10])
        stream.synchronize()
    pool.close()
    own.close()


@pytest.mark.parametrize("dtype,heads,d,layers", [("bf16", 8, 128, 3), ("f32", 1, 33, 2), ("f16", 2, 256, 1)])
def test_a_chain_that_is_cut_and_one_that_is_not(ctx, dtype, heads, d, layers):
    """One token leaves long sequences: every move's source is the target of the next, cut into runs
    whose first reads were saved, in place and with keys turned."""
    lengths = [2000, 700, 70]
    print(f"chains {dtype} {heads} x {d} layers {layers}", flush=True)
    cache = Cache(ctx, dtype, lengths, heads, d, layers=layers, seed=71)
    pool = cache.to_device()
    gone = [5, 300, 68]
    source = np.concatenate([cache.slots(t, np.delete(np.arange(n), x)) for t, n, x in zip(cache.tables, lengths, gone)])
    target = np.concatenate([cache.slots(t, np.arange(n - 1)) for t, n in zip(cache.tables, lengths)])
    for _ in range(2):  # twice the same moves, over what the first left
        pool.compact(source, target, [n - 1 for n in lengths])
        for x in (cache.k, cache.v):
            x[:, target] = x[:, source].clone()
    ctx.sync()
    cache.unchanged()
    pool.close()
