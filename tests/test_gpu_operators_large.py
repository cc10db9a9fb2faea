"""Compaction and rotation on several axes at sizes whose launches take several heads in a workgroup or
in a thread (the CPU test "launch forms" has their number at these sizes), against 64 bits."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context
from tests.operator_ref import Cache, assert_within, frequencies, turned, turned_bound
from tests.test_gpu_axes import angles

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def check_compacted(cache, source, target, shift, theta, width):
    """The moves' rows against their definition, everything else as it was."""
    before = cache.k[:, source].clone()
    cache.v[:, target] = cache.v[:, source].clone()
    got = cache.kd.cpu()[:, target]
    cache.k[:, target] = got
    cache.unchanged()
    still = np.ones(source.size, bool) if shift is None else shift == 0
    assert torch.equal(got[:, still], before[:, still]) and torch.equal(got[..., width:], before[..., width:])
    if width:
        angle = torch.from_numpy(shift[:, None].astype(np.float64)) * frequencies(theta, width)
        for layer in range(cache.layers):
            want, bound = turned(before[layer], angle, width), turned_bound(before[layer], width)
            assert_within(got[layer][~still], want[~still], bound[~still], f"layer {layer}")


@pytest.mark.parametrize("fresh", [True, False])
@pytest.mark.parametrize("dtype,heads,d,rotary,layers,moves", [
    ("bf16", 8, 64, 64, 12, 6000),   # 8 heads a workgroup
    ("bf16", 8, 64, 64, 12, 3500),   # 4
    ("f32", 8, 64, 32, 12, 1800),    # 2
    ("f16", 8, 64, None, 12, 1000),  # 1
    ("f32", 4, 128, 128, 16, 4200),  # 4, two chunks of 32 tokens a run
    ("f16", 3, 256, 64, 2, 900),     # 3, two chunks
    ("f16", 6, 256, 64, 2, 900)])    # 3 of 6
def test_compaction_of_many_moves(ctx, dtype, heads, d, rotary, layers, moves, fresh):
    """Three sequences, the last of which makes the last run's chunk one that is not full; to fresh
    pages, where a run has as many moves as it takes, and towards the front."""
    print(f"compact {dtype} {heads} x {d} layers {layers} moves {moves} fresh {fresh}", flush=True)
    rng = np.random.RandomState(moves)
    want = [moves // 2, moves // 3, moves - moves // 2 - moves // 3 - 7]
    lengths = [2 * n + 9 for n in want]
    kept = [np.sort(rng.choice(n, m, replace=False)) for n, m in zip(lengths, want)]
    cache = Cache(ctx, dtype, lengths, heads, d, layers=layers, spare=sum(-(-m // 16) for m in want) + 2, seed=d)
    pool = cache.to_device()
    tables, at = cache.tables, 0
    if fresh:
        tables = []
        for m in want:
            tables.append(cache.free[at:at + -(-m // 16)])
            at += -(-m // 16)
    source = np.concatenate([cache.slots(t, x) for t, x in zip(cache.tables, kept)])
    target = np.concatenate([cache.slots(t, np.arange(x.size)) for t, x in zip(tables, kept)])
    shift = None if rotary is None else np.concatenate([np.arange(x.size) - x for x in kept])
    pool.compact(source, target, want, shift, 1e4, rotary or 0)
    ctx.sync()
    check_compacted(cache, source, target, shift, 1e4, rotary or 0)
    pool.close()


@pytest.mark.parametrize("dtype,heads,d,layers", [("bf16", 3, 128, 2), ("f32", 5, 64, 1), ("f16", 8, 64, 40)])
def test_long_chains_in_several_heads(ctx, dtype, heads, d, layers):
    """One token leaves: every move's source is the target of the one behind it. Chains through several
    chunks of several heads (an odd number of them, or many layers), cut or not, and turned."""
    print(f"chains {dtype} {heads} x {d} layers {layers}", flush=True)
    lengths = [700, 1500, 300]
    cache = Cache(ctx, dtype, lengths, heads, d, layers=layers, seed=9)
    pool = cache.to_device()
    kept = [np.delete(np.arange(n), x) for n, x in zip(lengths, (3, 500, 298))]
    source = np.concatenate([cache.slots(t, x) for t, x in zip(cache.tables, kept)])
    target = np.concatenate([cache.slots(t, np.arange(x.size)) for t, x in zip(cache.tables, kept)])
    shift = np.concatenate([np.arange(x.size) - x for x in kept])
    pool.compact(source, target, [x.size for x in kept], shift, 1e4)
    ctx.sync()
    check_compacted(cache, source, target, shift, 1e4, d)
    pool.close()


@pytest.mark.parametrize("dtype,q_heads,kv_heads,d,rotary,rows,sections", [
    ("bf16", 16, 8, 128, 128, 4200, [24, 20, 20]),  # heads a multiple of four
    ("bf16", 14, 7, 128, 48, 4700, [8, 8, 8]),      # a thread's four are queries and keys, the last's are one
    ("f16", 6, 3, 256, 64, 5500, [11, 11, 10]),
    ("f32", 5, 5, 64, 64, 13200, [16, 16])])
def test_axes_of_many_rows(ctx, dtype, q_heads, kv_heads, d, rotary, rows, sections):
    """Four heads a thread, alone (on a batch without slots, and in place) and with the append."""
    print(f"axes {dtype} {q_heads}+{kv_heads} x {d} rotary {rotary} rows {rows}", flush=True)
    theta, axis = 1e6, ckv.rope_pair_axes(sections, True)
    rng = np.random.RandomState(rows)
    positions = rng.randint(0, 5000, (len(sections), rows)).astype(np.uint32)
    positions[0, 0], positions[-1, -1] = 4294967295, 1_000_003
    cache = Cache(ctx, dtype, [rows], kv_heads, d, layers=2, seed=rows)
    pool = cache.to_device()
    q, k, v = cache.randn(rows, q_heads, d), cache.randn(rows, kv_heads, d), cache.randn(rows, kv_heads, d)
    angle = angles(positions, axis, theta, rotary)
    slack = (angle.abs() * 2.0 ** -50)[:, None]

    def check(got, x, what):
        bound = turned_bound(x, rotary)
        bound[..., :rotary] += torch.cat([slack, slack], -1) * x.double().abs().amax() * 2
        assert_within(got, turned(x, angle, rotary), bound, what)
        assert torch.equal(got[..., rotary:].cpu(), x[..., rotary:])

    cache.upload([0], [rows], slots=False)
    pool.upload_axes(positions)
    qd = q.cuda().flatten(1)
    alone = torch.full((rows + 2, q_heads * d), 3.0, dtype=q.dtype, device="cuda")
    pool.rope_axes(qd, alone, q_heads, theta, axis, rotary)
    place = qd.clone()
    pool.rope_axes(place, place, q_heads, theta, axis, rotary)
    _, _, at = cache.upload([0], [rows])
    pool.upload_axes(positions)
    out = torch.full((rows + 2, q_heads * d), 3.0, dtype=q.dtype, device="cuda")
    pool.rope_axes_append(1, qd, out, q_heads, k.cuda().flatten(1), v.cuda().flatten(1), theta, axis, rotary)
    ctx.sync()
    assert torch.all(out[rows:] == 3.0) and torch.all(alone[rows:] == 3.0)
    assert torch.equal(alone, out) and torch.equal(place, out[:rows]) and torch.equal(qd.cpu(), q.flatten(1))
    check(out[:rows].view(rows, q_heads, d), q, "queries")
    got = cache.kd[1, at]
    check(got, k, "keys")
    cache.k[1, at], cache.v[1, at] = got.cpu(), v
    cache.unchanged()
    pool.close()
