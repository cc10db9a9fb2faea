"""Windowed attention by calls that the other tests do not make: rows, gates and new tokens off 16-byte
boundaries (other kernels take them), the same row several times in a batch, batches without rows."""
import math

import numpy as np
import pytest
import torch

from tests.gpu_util import new_context
from tests.operator_ref import Cache, assert_within, attention, seen
from tests.test_gpu_axes import off_by_one

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def check(cache, out, q, gate, rows, window, sinks, scale, p_bits, what):
    """Each (sequence, position) of rows against what the cache on the device holds."""
    k, v = cache.kd[0].cpu(), cache.vd[0].cpu()
    for r, (s, p) in enumerate(rows):
        at = cache.slots(cache.tables[s], seen(p, window, sinks))
        want, bound = attention(q[r:r + 1], k[at], v[at], [np.arange(at.size)], scale, p_bits=p_bits)
        if gate is not None:
            g = torch.sigmoid(gate[r:r + 1].double())
            want, bound = want * g, bound * g + want.abs() * 16 * 2.0 ** -23
        assert_within(out[r].view(want.shape), want, bound, f"{what}: row {r}, position {p}")


@pytest.mark.parametrize("odd", ["queries", "output", "gate", "keys", "all"])
@pytest.mark.parametrize("dtype,heads,group,d", [("bf16", 2, 2, 128), ("f16", 1, 4, 256), ("f32", 2, 8, 128)])
def test_unaligned_rows(ctx, dtype, heads, group, d, odd):
    print(f"unaligned {odd} {dtype} {heads} x {group} d {d}", flush=True)
    lengths, window, sinks, scale = [300, 33, 70], 60, 4, 1 / math.sqrt(d)

    def place(name, t):
        return off_by_one(t) if odd in (name, "all") else t

    for first, counts in (([n - 1 for n in lengths], [1] * 3), ([250, 0, 69], [50, 33, 1])):
        cache = Cache(ctx, dtype, lengths, heads, d, seed=3)
        pool = cache.to_device()
        seq, pos, at = cache.upload(first, counts)
        n = len(pos)
        q, gate = cache.randn(n, heads * group, d), cache.randn(n, heads * group, d)
        k, v = cache.randn(n, heads, d), cache.randn(n, heads, d)
        args = [place("queries", q.cuda().flatten(1)), heads * group, scale, window,
                place("output", torch.full((n, heads * group * d), math.nan, dtype=cache.dtype, device="cuda"))]
        gd = place("gate", gate.cuda().flatten(1))
        kd, vd = place("keys", k.cuda().flatten(1)), place("keys", v.cuda().flatten(1))
        if n == 3:
            pool.append_decode_window(0, kd, vd, *args, sinks=sinks, gate=gd)
        else:
            pool.append(0, kd, vd)
            pool.attention_window(0, *args, sinks=sinks, gate=gd)
        ctx.sync()
        cache.unchanged(but=at)
        assert torch.equal(cache.kd[0, at].cpu(), k) and torch.equal(cache.vd[0, at].cpu(), v)
        keep = range(0, n, 1 if n == 3 else 5)
        check(cache, args[4][list(keep)], q[list(keep)], gate[list(keep)], [(seq[r], pos[r]) for r in keep], window, sinks,
              scale, 16, odd)
        pool.close()


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 1, 256), ("f16", 3, 96)])
def test_a_row_several_times(ctx, dtype, group, d):
    """The same row twice in a batch, a chunk twice, and positions out of order."""
    print(f"rows twice {dtype} group {group} d {d}", flush=True)
    lengths, window, sinks, scale = [400, 50], 45, 3, 1 / math.sqrt(d)
    cache = Cache(ctx, dtype, lengths, 2, d, seed=5)
    pool = cache.to_device()
    flat, starts = np.concatenate(cache.tables), [0, cache.tables[0].size]
    rows = [(0, 399), (0, 399), (1, 10), (0, 5)] + 2 * [(0, 300 + i) for i in range(40)] + [(1, 49), (0, 300)]
    seq, pos = np.array(rows).T
    pool.upload(flat, np.take(starts, seq), [cache.tables[s].size for s in seq], pos)
    q = cache.randn(len(rows), 2 * group, d)
    q[1], q[44:84] = q[0], q[4:44]
    out = torch.empty(len(rows), 2 * group * d, dtype=cache.dtype, device="cuda")
    pool.attention_window(0, q.cuda().flatten(1), 2 * group, scale, window, out, sinks=sinks)
    ctx.sync()
    assert torch.equal(out[0], out[1]) and torch.equal(out[4:44], out[44:84])
    keep = [0, 2, 3, 4, 20, 43, 84, 85]
    check(cache, out[keep], q[keep], None, [rows[r] for r in keep], window, sinks, scale, 16, "twice")
    pool.close()


def test_batches_without_rows(ctx):
    cache = Cache(ctx, "bf16", [40], 2, 128, seed=5)
    pool = cache.to_device()
    none = torch.empty(0, 512, dtype=torch.bfloat16, device="cuda")
    few = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    pool.upload(cache.tables[0], [], [], [], [])
    pool.upload_axes(np.zeros((3, 0)))
    pool.attention_window(0, none, 4, 0.1, 8, none, sinks=2)
    pool.append_decode_window(0, few, few, none, 4, 0.1, 8, none)
    pool.rope_append_decode_window(0, few, few, none, 4, 0.1, 1e4, 8, none)
    pool.rope_axes(none, none, 4, 1e4, [0] * 64)
    pool.rope_axes_append(0, none, none, 4, few, few, 1e4, [2] * 64)
    pool.compact([], [], [])
    ctx.sync()
    cache.unchanged()
    pool.close()
