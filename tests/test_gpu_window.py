"""Attention through a window with sinks against its definition in 64 bits.

Pages that no row attends hold NaN and are replaced in the tables by a page of NaN, as a
sequence that gave them back would have them; keys outside the window in pages that are
read are infinite or NaN. Any of them that were read into a result would show in it."""
import math

import numpy as np
import pytest
import torch

from tests.gpu_util import force_plan, new_context
from tests.operator_ref import Cache, assert_within, attention, seen

pytestmark = pytest.mark.gpu

LENGTHS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 130, 255, 256, 257, 401]


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def poison(cache, attended, bad=math.nan):
    """Unattended tokens become `bad` (keys) and infinite (values); pages without an attended
    token are given back: a page of NaN takes their place in the table."""
    trap = cache.free[0]
    for s, (table, t) in enumerate(zip(cache.tables, attended)):
        drop = np.setdiff1d(np.arange(cache.lengths[s]), t)
        at = torch.from_numpy(cache.slots(table, drop))
        cache.k[:, at], cache.v[:, at] = bad, math.inf
        given = np.setdiff1d(np.arange(table.size), np.unique(np.asarray(t) // cache.page))
        table[given] = trap


def decode_case(ctx, dtype, heads, group, d, window, sinks, page=16, lengths=LENGTHS, gated=False, seed=1,
                scale=None, bad=math.nan, fused=True):
    cache = Cache(ctx, dtype, lengths, heads, d, page=page, seed=seed)
    attended = [seen(n - 1, window, sinks) for n in lengths]
    rows = len(lengths)
    q, k, v = cache.randn(rows, heads * group, d), cache.randn(rows, heads, d), cache.randn(rows, heads, d)
    gate = cache.randn(rows, heads * group, d) if gated else None
    poison(cache, attended, bad)
    pool = cache.to_device()
    _, _, at = cache.upload([n - 1 for n in lengths], [1] * rows)
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.full((rows, heads * group * d), math.nan, dtype=cache.dtype, device="cuda")
    args = (0, k.cuda().flatten(1), v.cuda().flatten(1), q.cuda().flatten(1), heads * group, scale, window, out)
    gd = None if gate is None else gate.cuda().flatten(1)
    if fused:
        pool.append_decode_window(*args, sinks=sinks, gate=gd)
    else:
        pool.append(0, *args[1:3])
        pool.attention_window(0, *args[3:], sinks=sinks, gate=gd)
    ctx.sync()
    cache.unchanged(but=at)
    assert torch.equal(cache.kd.cpu()[0, at], k) and torch.equal(cache.vd.cpu()[0, at], v)
    for r, (table, t) in enumerate(zip(cache.tables, attended)):
        slots = cache.slots(table, t)
        kk, vv = cache.kd.cpu()[0, slots], cache.vd.cpu()[0, slots]
        want, bound = attention(q[r:r + 1], kk, vv, [np.arange(len(t))], scale)
        if gated:
            g = torch.sigmoid(gate[r:r + 1].double())
            want, bound = want * g, bound * g + want.abs() * 16 * 2.0 ** -23
        assert_within(out[r].view(1, heads * group, d), want, bound, f"row {r} of {lengths[r]} tokens")
    pool.close()
    return out.cpu()


WINDOWS = [(1, 0), (1, 4), (16, 0), (17, 1), (40, 4), (64, 16), (100, 33), (256, 300), (5000, 4)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("dtype,group,d,page", [
    ("bf16", 2, 128, 16), ("f16", 4, 256, 16), ("f32", 1, 128, 16), ("bf16", 3, 80, 8), ("f32", 2, 96, 5)])
def test_window_decode(ctx, dtype, group, d, page, window, sinks):
    print(f"window decode {dtype} group {group} d {d} page {page} window {window} sinks {sinks}", flush=True)
    decode_case(ctx, dtype, 2, group, d, window, sinks, page=page)


@pytest.mark.parametrize("dtype,heads,group,d", [
    ("bf16", 2, 1, 128), ("bf16", 2, 4, 128), ("f16", 1, 8, 128), ("f32", 2, 8, 128), ("f32", 1, 2, 256),
    ("bf16", 2, 2, 256), ("bf16", 1, 8, 256), ("f32", 3, 4, 256), ("f16", 2, 2, 64)])
@pytest.mark.parametrize("gated,fused", [(True, True), (False, False)])
def test_window_decode_geometries(ctx, dtype, heads, group, d, gated, fused):
    print(f"window decode {dtype} {heads} x {group} d {d} gated {gated} fused {fused}", flush=True)
    decode_case(ctx, dtype, heads, group, d, 50, 4, gated=gated, fused=fused, bad=math.inf)


@pytest.mark.parametrize("split", ["0", "1", "2", "3", "b2", "b5"])
def test_window_decode_plans(ctx, split, monkeypatch):
    print(f"window decode plan {split}", flush=True)
    force_plan(monkeypatch, split)
    for d, dtype in ((128, "bf16"), (256, "f16"), (128, "f32")):
        decode_case(ctx, dtype, 2, 2, d, 140, 20, seed=5)


@pytest.mark.parametrize("scale", [0.0, -0.07])
def test_window_decode_any_scale(ctx, scale):
    decode_case(ctx, "bf16", 2, 2, 128, 33, 4, scale=scale)


def test_long_rows_through_a_small_window(ctx):
    """Rows far past the window, one of them long enough that its offsets in the table and
    the pool are large; a single row; and the same answer each time."""
    lengths = [20_011, 1, 37, 9_000]
    one = decode_case(ctx, "bf16", 8, 2, 128, 700, 4, lengths=lengths, seed=9)
    assert torch.equal(one, decode_case(ctx, "bf16", 8, 2, 128, 700, 4, lengths=lengths, seed=9))
    decode_case(ctx, "bf16", 8, 2, 128, 4096, 4, lengths=[12_345], seed=10)


def prefill_case(ctx, dtype, heads, group, d, window, sinks, first, counts, gated=False, page=16, seed=3, p_bits=16,
                 odd=None):
    """odd: (sequence, token, value) of a V row that is not finite."""
    lengths = [f + c for f, c in zip(first, counts)]
    cache = Cache(ctx, dtype, lengths, heads, d, page=page, seed=seed)
    rows = sum(counts)
    each = [[seen(f + i, window, sinks) for i in range(c)] for f, c in zip(first, counts)]
    poison(cache, [np.unique(np.concatenate(e)) for e in each])
    if odd is not None:
        cache.v[0, cache.slots(cache.tables[odd[0]], [odd[1]])[0]] = odd[2]
    q = cache.randn(rows, heads * group, d)
    gate = cache.randn(rows, heads * group, d) if gated else None
    pool = cache.to_device()
    cache.upload(first, counts, slots=False)
    scale = 1 / math.sqrt(d)
    behind = 5  # rows past the last: left as they are
    out = torch.full((rows + behind, heads * group * d), 7.0, dtype=cache.dtype, device="cuda")
    pool.attention_window(0, q.cuda().flatten(1), heads * group, scale, window, out, sinks=sinks,
                          gate=None if gate is None else gate.cuda().flatten(1))
    ctx.sync()
    cache.unchanged()
    assert torch.all(out[rows:] == 7.0)
    row = 0
    for s, (e, c) in enumerate(zip(each, counts)):
        n = lengths[s]
        at = cache.slots(cache.tables[s], np.arange(n))
        kk, vv = cache.k[0, at], cache.v[0, at]
        for i, t in enumerate(e):
            r = row + i
            if dtype == "f32" or 0 < i < c - 1 and i % 7 and odd is None:  # f32: a row in three; others: ends and every seventh
                if dtype != "f32" or i % 3:
                    continue
            want, bound = attention(q[r:r + 1], kk[t], vv[t], [np.arange(len(t))], scale, p_bits=p_bits)
            if gated:
                g = torch.sigmoid(gate[r:r + 1].double())
                want, bound = want * g, bound * g + want.abs() * 16 * 2.0 ** -23
            assert_within(out[r].view(1, heads * group, d), want, bound, f"sequence {s} row {i}")
        row += c
    pool.close()
    return out.cpu()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (31, 0), (32, 4), (33, 33), (64, 4), (100, 1), (300, 40), (9999, 0)])
@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f16", 4, 256), ("f32", 2, 128)])
def test_window_prefill(ctx, dtype, group, d, window, sinks):
    print(f"window prefill {dtype} group {group} d {d} window {window} sinks {sinks}", flush=True)
    prefill_case(ctx, dtype, 1, group, d, window, sinks, [0, 150, 37, 511], [70, 40, 2, 129])


@pytest.mark.parametrize("dtype,heads,group,d,page", [
    ("bf16", 2, 1, 128, 16), ("bf16", 1, 8, 128, 16), ("f16", 2, 4, 128, 16), ("bf16", 1, 8, 256, 16),
    ("bf16", 2, 1, 256, 16), ("f16", 1, 2, 256, 16), ("f32", 1, 1, 128, 16), ("f32", 1, 4, 128, 16),
    ("f32", 1, 8, 128, 16), ("f32", 1, 2, 256, 16), ("bf16", 1, 2, 64, 16), ("bf16", 1, 2, 128, 8)])
def test_window_prefill_geometries(ctx, dtype, heads, group, d, page):
    print(f"window prefill {dtype} {heads} x {group} d {d} page {page}", flush=True)
    prefill_case(ctx, dtype, heads, group, d, 75, 4, [3, 200], [90, 35], gated=True, page=page)


@pytest.mark.parametrize("split", ["1", "2", "3", "8"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 256), ("f32", 128)])
def test_window_prefill_key_ranges(ctx, dtype, d, split, monkeypatch):
    """A tile's keys in several ranges, some of which hold none that a row attends."""
    print(f"window prefill {dtype} d {d} split {split}", flush=True)
    monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    monkeypatch.setenv("CKV_PREFILL_SPLIT_MIN", "1")
    args = (ctx, dtype, 1, 2, d, 90, 40, [600], [150])
    assert torch.equal(prefill_case(*args), prefill_case(*args))


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f16", 4, 256), ("f32", 2, 128), ("bf16", 8, 128)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_odd_values_stay_with_the_rows_that_attend_them(ctx, dtype, group, d, value):
    """A value that is not finite reaches the rows whose window or sinks hold it and no other:
    one inside the chunk, one at the window's edge, one among the sinks."""
    print(f"window prefill {dtype} group {group} d {d} with {value}", flush=True)
    for token in (205, 150, 2):
        prefill_case(ctx, dtype, 1, group, d, 40, 4, [180], [60], odd=(0, token, value))


def test_mixed_batch_of_decode_rows_and_chunks(ctx):
    prefill_case(ctx, "bf16", 2, 2, 128, 48, 4, [99, 0, 640, 255], [1, 33, 1, 64])


def test_two_windows_and_the_full_context_share_a_batch(ctx):
    """Layers alternate between two windows and none; each keeps its own answer."""
    lengths = [300, 77, 5]
    cache = Cache(ctx, "bf16", lengths, 2, 128, seed=4)
    pool = cache.to_device()
    cache.upload([n - 1 for n in lengths], [1] * 3)
    q = cache.randn(3, 4, 128)
    scale, qd = 1 / math.sqrt(128), q.cuda().flatten(1)
    for _ in range(2):
        for window in (20, None, 64, 10_000):
            out = torch.empty(3, 512, dtype=torch.bfloat16, device="cuda")
            if window is None:
                pool.attention(0, qd, 4, scale, out)
            else:
                pool.attention_window(0, qd, 4, scale, window, out, sinks=2)
            ctx.sync()
            for r, n in enumerate(lengths):
                t = seen(n - 1, window or 10_000, 2)
                at = cache.slots(cache.tables[r], t)
                want, bound = attention(q[r:r + 1], cache.k[0, at], cache.v[0, at], [np.arange(len(t))], scale)
                assert_within(out[r].view(1, 4, 128), want, bound, f"window {window} row {r}")
    pool.close()


def test_rotated_append_decode_is_its_parts(ctx):
    """ckv_rope_append_decode_window against ckv_rope, ckv_rope_append and the attention: the cache
    within one unit in the last place of a rotated element, the output as far as that moves it."""
    lengths = [400, 64, 130, 2]
    for dtype, d, rotary, gated in (("bf16", 128, 128, False), ("f16", 256, 64, True), ("f32", 128, 0, False),
                                    ("bf16", 128, 48, True)):
        got = []
        for parts in (False, True):
            cache = Cache(ctx, dtype, lengths, 2, d, seed=6)
            pool = cache.to_device()
            _, _, at = cache.upload([n - 1 for n in lengths], [1] * 4)
            q, k, v = (cache.randn(4, n, d).cuda().flatten(1) for n in (4, 2, 2))
            gate = cache.randn(4, 4, d).cuda().flatten(1) if gated else None
            out, scale = torch.empty_like(q), 1 / math.sqrt(d)
            if parts:
                rq = torch.empty_like(q)
                pool.rope(q, rq, 4, 1e4, rotary)
                pool.rope_append(0, k, v, 1e4, rotary)
                pool.attention_window(0, rq, 4, scale, 100, out, sinks=4, gate=gate)
            else:
                pool.rope_append_decode_window(0, k, v, q, 4, scale, 1e4, 100, out, sinks=4, rotary_dim=rotary, gate=gate)
            ctx.sync()
            cache.unchanged(but=at)
            got.append((out.float(), cache.kd[0, at].float(), cache.vd[0, at]))
            pool.close()
        (o1, k1, v1), (o2, k2, v2) = got
        eps = torch.finfo(cache.dtype).eps
        assert torch.equal(v1, v2)
        assert torch.all((k1 - k2).abs() <= eps * torch.maximum(k1.abs(), k2.abs()) + 1e-6)
        # rotated operands one step apart: a score moves by 2 eps |q| |k| scale at most, values are N(0, 1)
        room = 4 * eps * float((q.float().view(4, 4, d).norm(dim=-1)).max() * 20 / math.sqrt(d)) * 5
        assert torch.all((o1 - o2).abs() <= room)


def test_captured_decode_replays_and_cold_capture_is_refused(ctx):
    """A windowed decode captured after one eager call replays on new inputs; a capture before any
    such call is refused, and the batch still works after that."""
    from chibillm_amd import ckv
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    lengths = [700, 90, 333]
    cache = Cache(own, "bf16", lengths, 2, 128, seed=8)
    with torch.cuda.stream(stream):
        pool = cache.to_device()
        cache.upload([n - 1 for n in lengths], [1] * 3)
        q, k, v = (cache.randn(3, n, 128).cuda().flatten(1) for n in (4, 2, 2))
        out, scale = torch.empty_like(q), 1 / math.sqrt(128)

        def call():
            pool.append_decode_window(0, k, v, q, 4, scale, 60, out, sinks=4)

        stream.synchronize()
        cold = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cold, stream=stream):
            with pytest.raises(ckv.CkvError) as refused:
                call()
            out.zero_()  # the capture itself goes on
        assert refused.value.name == "ckv.invalid_argument"
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for seed in range(4):
            torch.manual_seed(seed)
            for x in (q, k, v):
                x.normal_()
            call()
            stream.synchronize()
            want = out.clone()
            out.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want)
    pool.close()
    own.close()


@pytest.mark.parametrize("dtype,d,chunks", [("bf16", 128, False), ("f32", 128, False), ("bf16", 64, False),
                                            ("bf16", 128, True), ("f32", 128, True), ("f16", 256, True)])
def test_captured_windows_keep_what_they_read(ctx, dtype, d, chunks):
    """Layers of two windows and more query heads captured into one graph: calls of other windows
    and of more heads afterwards, which take lists of their own and larger scratch, leave its
    replays as they were, on new inputs."""
    print(f"captured windows {dtype} d {d} chunks {chunks}", flush=True)
    from chibillm_amd import ckv
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    first, counts = ([900, 40, 0], [100, 1, 33]) if chunks else ([1500, 89, 0, 700], [1] * 4)
    rows, heads = sum(counts), 2
    cache = Cache(own, dtype, [f + c for f, c in zip(first, counts)], heads, d, seed=12)
    with torch.cuda.stream(stream):
        pool = cache.to_device()
        cache.upload(first, counts, slots=not chunks)
        q, k, v = (cache.randn(rows, n * heads, d).cuda().flatten(1) for n in (8, 1, 1))
        scale = 1 / math.sqrt(d)

        def layer(group, window, out):
            rows_q = q[:, :group * heads * d].contiguous() if group < 8 else q
            if chunks or group == 4:
                pool.attention_window(0, rows_q, group * heads, scale, window, out, sinks=4)
            else:
                pool.rope_append_decode_window(0, k, v, rows_q, group * heads, scale, 1e4, window, out, sinks=4)

        calls = [(2, 700), (2, 60), (4, 700), (2, 5000)]
        outs = [torch.empty(rows, g * heads * d, dtype=cache.dtype, device="cuda") for g, _ in calls]

        def layers():
            for (group, window), out in zip(calls, outs):
                layer(group, window, out)

        layers()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layers()
        wide = torch.empty(rows, 8 * heads * d, dtype=cache.dtype, device="cuda")
        for turn in range(3):
            for window in (33 + turn, 800 + turn, 400):
                layer(8, window, wide)
                layer(2, window, outs[0])
            for x in (q, k, v):
                x.normal_()
            layers()
            stream.synchronize()
            want = [out.clone() for out in outs]
            for out in outs:
                out.fill_(math.nan)
            graph.replay()
            stream.synchronize()
            for out, w, call in zip(outs, want, calls):
                assert torch.equal(out, w), f"replay {turn} of group {call[0]} window {call[1]}"
    pool.close()
    own.close()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("f32", 128)])
@pytest.mark.parametrize("window", [40, 10_000])
def test_a_refused_call_captures_nothing(ctx, dtype, d, window):
    """Under capture and before any eager call, also where the window covers every row: refused
    before the append, so that the graph leaves the cache as it was."""
    from chibillm_amd import ckv
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    lengths = [300, 7, 801]
    cache = Cache(own, dtype, lengths, 2, d, seed=13)
    with torch.cuda.stream(stream):
        pool = cache.to_device()
        _, _, at = cache.upload([n - 1 for n in lengths], [1] * 3)
        q, k, v = (cache.randn(3, n, d).cuda().flatten(1) for n in (16, 2, 2))
        out, scale, refused = torch.zeros_like(q), 1 / math.sqrt(d), 0
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out.add_(1)  # a graph has to hold something
            for call in (lambda: pool.append_decode_window(0, k, v, q, 16, scale, window, out, sinks=4),
                         lambda: pool.rope_append_decode_window(0, k, v, q, 16, scale, 1e4, window, out, sinks=4)):
                try:
                    call()
                except ckv.CkvError as e:
                    assert e.name == "ckv.invalid_argument"
                    refused += 1
        # rows of a plan that came with the batch and cuts none have nothing to upload
        assert refused == 2 or (window > 1000 and refused < 2)
        graph.replay()
        stream.synchronize()
        if refused == 2:
            cache.unchanged()
            assert torch.all(out == 1)
        else:
            cache.unchanged(but=at)
    pool.close()
    own.close()
