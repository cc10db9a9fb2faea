"""Rotation by positions on several axes, alone and fused with the append, against 64 bits:
axes at far positions, partial rotary widths, odd head counts, unaligned rows, in place."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context
from tests.operator_ref import Cache, assert_within, frequencies, turned, turned_bound

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def off_by_one(t):
    """A copy one element past a 16-byte boundary."""
    base = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    view = base[1:1 + t.numel()].view(t.shape)
    view.copy_(t)
    return view


def angles(positions, pair_axis, theta, rotary):
    at = torch.from_numpy(positions.astype(np.int64)).double()[torch.from_numpy(pair_axis.astype(np.int64))]
    return at.t() * frequencies(theta, rotary)  # [rows, pairs]


@pytest.mark.parametrize("rows", [1, 3, 65, 200])
@pytest.mark.parametrize("dtype,q_heads,kv_heads,d,rotary,theta,sections,interleaved", [
    ("bf16", 16, 8, 128, 0, 1e6, [24, 20, 20], True), ("f16", 8, 2, 256, 64, 1e7, [11, 11, 10], True),
    ("f32", 4, 2, 128, 0, 1e4, [16, 24, 24], False), ("bf16", 3, 1, 80, 32, 1e4, [16], False),
    ("f32", 1, 1, 64, 10, 500.0, [2, 1, 1, 1], True), ("bf16", 5, 5, 128, 48, 1e6, [12, 12], False),
    ("f16", 1, 1, 512, 512, 1e4, [100, 100, 56], False), ("bf16", 2, 1, 100, 0, 1e4, [30, 20], True)])
def test_axes_append(ctx, rows, dtype, q_heads, kv_heads, d, rotary, theta, sections, interleaved):
    print(f"axes {dtype} {q_heads}+{kv_heads} x {d} rotary {rotary} rows {rows}", flush=True)
    width = rotary or d
    pair_axis = ckv.rope_pair_axes(sections, interleaved)
    rng = np.random.RandomState(rows)
    positions = rng.randint(0, 2000, (len(sections), rows)).astype(np.uint32)
    positions[0, 0], positions[-1, -1] = 4294967295, 1_000_003  # as far as 32 bits go
    for shift in (lambda t: t, off_by_one):
        cache = Cache(ctx, dtype, [rows], kv_heads, d, layers=2, seed=rows)
        pool = cache.to_device()
        _, _, at = cache.upload([0], [rows])
        pool.upload_axes(positions)
        q, k, v = cache.randn(rows, q_heads, d), cache.randn(rows, kv_heads, d), cache.randn(rows, kv_heads, d)
        qd = shift(q.cuda().flatten(1))
        behind = torch.full((rows + 2, q_heads * d), 3.0, dtype=q.dtype, device="cuda")
        out = shift(behind)
        pool.rope_axes_append(1, qd, out, q_heads, shift(k.cuda().flatten(1)), shift(v.cuda().flatten(1)), theta,
                              pair_axis, rotary)
        place = qd.clone()
        pool.rope_axes(place, place, q_heads, theta, pair_axis, rotary)
        ctx.sync()
        cache.k[1, at], cache.v[1, at] = cache.kd[1, at].cpu(), v
        cache.unchanged()  # the values bit for bit, everything else as it was
        assert torch.all(out[rows:] == 3.0)
        assert torch.equal(place, out[:rows]) and torch.equal(qd.cpu(), q.flatten(1))
        # pow's own error: a frequency is within 2^-52 of its double
        angle = angles(positions, pair_axis, theta, width)
        slack = (angle.abs() * 2.0 ** -50)[:, None]
        for got, x in ((out[:rows].view(rows, q_heads, d), q), (cache.kd[1, at], k)):
            moved = torch.cat([slack, slack], -1) * x.double().abs().amax() * 2
            bound = turned_bound(x, width)
            bound[..., :width] += moved
            assert_within(got, turned(x, angle, width), bound, "rotated rows")
            assert torch.equal(got[..., width:].cpu(), x[..., width:])
        pool.close()


def test_equal_axes_are_ckv_rope(ctx):
    """With one position on every axis the rotation is ckv_rope's, within a step and what ckv_rope's
    32-bit angle is off (half a step of the angle, at most 2,000 radians here)."""
    rows, d = 40, 128
    cache = Cache(ctx, "f32", [rows], 2, d, seed=2)
    pool = cache.to_device()
    cache.upload([0], [rows])
    positions = np.arange(rows)
    pool.upload_axes(np.stack([positions] * 3))
    x = cache.randn(rows, 4, d).cuda().flatten(1)
    a, b = torch.empty_like(x), torch.empty_like(x)
    pool.rope(x, a, 4, 1e4)
    pool.rope_axes(x, b, 4, 1e4, ckv.rope_pair_axes([24, 20, 20], True))
    ctx.sync()
    # the angle in 32 bits: a step of the frequency and one of the product, of at most 39 radians
    assert float((a - b).abs().max()) <= float(x.abs().max()) * 2 * (39 * 2.0 ** -22 + 8 * 2.0 ** -23)
    pool.close()


def test_keys_alone_and_a_new_batch_forgets_the_axes(ctx):
    cache = Cache(ctx, "bf16", [20], 2, 128, seed=2)
    pool = cache.to_device()
    _, _, at = cache.upload([0], [20])
    k, v = cache.randn(20, 2, 128).cuda().flatten(1), cache.randn(20, 2, 128).cuda().flatten(1)
    axis = ckv.rope_pair_axes([64])
    with pytest.raises(ckv.CkvError) as e:
        pool.rope_axes_append(0, None, None, 0, k, v, 1e4, axis)
    assert e.value.name == "ckv.no_tables"
    pool.upload_axes(np.zeros((1, 20)))
    pool.rope_axes_append(0, None, None, 0, k, v, 1e4, axis)
    ctx.sync()
    assert torch.equal(cache.kd[0, at].flatten(1), k)  # at position 0 nothing turns
    cache.upload([0], [20])
    with pytest.raises(ckv.CkvError) as e:
        pool.rope_axes(k, k, 2, 1e4, axis)
    assert e.value.name == "ckv.no_tables"
    pool.close()
