"""The calls that were there before over pools held in 4 bits, and what prompts' attention takes batches
from: gated and fused forms, decode and tile calls by name, sequence tables, rotation on several axes."""
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


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 3, 64), ("f16", 4, 256)])
def test_calls_by_name(ctx, dtype, group, d):
    """ckv_decode_attention of a batch of tiles, ckv_prefill_attention of decode rows and of tiles: each
    row's attention, whichever kernel does it."""
    cache = ref.Cache(ctx, dtype, [140, 37, 5], 2, d, seed=31)
    cache.fill()
    for first, counts in (([100, 30, 0], [40, 7, 5]), ([139, 36, 4], [1, 1, 1])):
        cache.upload(first, counts, with_slots=False)
        q = cache.randn(sum(counts), 2 * group, d)
        x = q.cuda().flatten(1)
        for call, bits in ((cache.pool.decode, ref.decode_bits), (cache.pool.prefill, ref.tile_bits), (cache.pool.attention, ref.tile_bits)):
            out = torch.full_like(x, math.nan)
            call(0, x, 2 * group, 0.1, out)
            ref.assert_within(out, *cache.attended(q, 0.1, **bits(dtype)), f"{call.__name__} {counts}")
    cache.pool.close()


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 1, 64), ("f16", 3, 256)])
def test_gated_appends(ctx, dtype, group, d):
    cache = ref.Cache(ctx, dtype, [140, 37, 5], 2, d, seed=32)
    cache.fill()
    cache.upload([139, 36, 4], [1, 1, 1])
    q, k, v, gate = (cache.randn(3, n, d) for n in (2 * group, 2, 2, 2 * group))
    qd, kd, vd, gd = (x.cuda().flatten(1) for x in (q, k, v, gate))
    out = torch.full_like(qd, math.nan)
    cache.pool.append_decode_gated(0, kd, vd, qd, 2 * group, 0.1, gd, out)
    cache.keep(0, k, v)
    cache.check(0, "appended")
    ref.assert_within(out, *ref.gated(*cache.attended(q, 0.1, **ref.decode_bits(dtype)), gate), "gated")
    # rotated by the older call, gated
    rotation = ckv.Rotation(1e4, d // 2)
    positions = np.array([139, 36, 4])
    cache.pool.rope_append_decode(0, kd, vd, qd, 2 * group, 0.1, 1e4, out, d // 2, gate=gd)
    cache.keep(0, ref.rotated(k, positions, rotation)[0], v)
    cache.check(0, "rotated")
    q64, _ = ref.rotated(q, positions, rotation)
    want, bound = cache.attended(q64, 0.1, **ref.decode_bits(dtype))
    bound = bound + cache.attended(q64, 0.1, q_half=24 * ref.STEP32)[1]
    ref.assert_within(out, *ref.gated(want, bound, gate), "rotated and gated")
    cache.pool.close()


def test_axes_beside_a_pool_in_4_bits(ctx):
    """Rows rotated by positions on several axes do not touch the pool."""
    cache = ref.Cache(ctx, "bf16", [40], 2, 128, seed=33)
    cache.fill()
    cache.upload([0], [40], with_slots=False)
    q = cache.randn(40, 2, 128).cuda().flatten(1)
    cache.pool.upload_axes(np.arange(40)[None])
    by_axes, plain = torch.empty_like(q), torch.empty_like(q)
    cache.pool.rope_axes(q, by_axes, 2, 1e4, [0] * 64)
    cache.pool.rotate(ckv.Rotation(1e4), q, plain, 2)
    ref.assert_within(by_axes, *ref.rotated(q.view(40, 2, 128).cpu(), np.arange(40), ckv.Rotation(1e4)), "axes")
    ref.assert_within(plain, *ref.rotated(q.view(40, 2, 128).cpu(), np.arange(40), ckv.Rotation(1e4)), "rotate")
    cache.check(0, "as it was")
    cache.pool.close()


@pytest.mark.parametrize("dtype,group,d,fp4", [("bf16", 2, 128, False), ("bf16", 2, 128, True), ("f32", 1, 64, True), ("f16", 4, 256, False)])
def test_prompts_by_sequence_tables(ctx, dtype, group, d, fp4):
    """Prompts of a batch from the device's sequence tables, one of them as two items one after the
    other; then a chunk among them, which is refused; then prompts again."""
    heads, counts = 2, [70, 1, 33]
    pool = ckv.Pool(ctx, 1, 20, 16, heads, d, DTYPES[dtype], fp4=fp4)
    pool.reserve_sequences(6, 10)
    ids = [4, 0, 2]
    pages = [-(-c // 16) for c in counts]
    pool.update_sequences(np.repeat(ids, pages), np.concatenate([np.arange(p) for p in pages]), np.arange(sum(pages)), ids, pages)
    g = torch.Generator().manual_seed(34)
    n = sum(counts)
    q, k, v = (torch.randn(n, x, d, generator=g).to(DTYPES[dtype]) for x in (heads * group, heads, heads))
    qd, kd, vd = (x.cuda().flatten(1) for x in (q, k, v))
    want, at = [], 0
    for c in counts:
        s = slice(at, at + c)
        want.append(ref.attention(q[s], k[s], v[s], np.arange(1, c + 1), 0.1, **ref.tile_bits(dtype)))
        at += c
    want, bound = (torch.cat(x) for x in zip(*want))
    for items in (([4, 0, 2], [0, 0, 0], [70, 1, 33]), ([4, 4, 0, 2], [0, 40, 0, 0], [40, 30, 1, 33])):
        pool.upload_batch(*items, with_slots=False)
        out = torch.full_like(qd, math.nan)
        pool.prompt_attention(qd, kd, vd, heads * group, 0.1, out)
        ref.assert_within(out, want, bound, f"items {items[2]}")
    for items in (([4, 0, 2], [0, 3, 0], [70, 1, 33]), ([4, 2, 4], [0, 0, 40], [40, 33, 31])):
        pool.upload_batch(*items, with_slots=False)
        m = sum(items[2])
        with pytest.raises(ckv.CkvError) as refused:
            pool.prompt_attention(qd[:m], kd[:m], vd[:m], heads * group, 0.1, out[:m])
        assert refused.value.name == "ckv.invalid_argument"
    pool.close()


@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 1, 64)])
def test_the_same_row_twice_and_prompts_attended_by_pages(ctx, dtype, group, d):
    """A row of a batch twice, by decode and by tiles; a whole prompt through its pages is what the
    same rows, held, give without them, to their roundings."""
    cache = ref.Cache(ctx, dtype, [300, 40], 2, d, seed=35)
    k, v = cache.fill()
    lengths = np.array([t.size for t in cache.tables])
    at = np.array([0, 0, 1, 0])
    positions = np.array([255, 255, 39, 17])
    cache.rows = list(zip(at, positions))
    cache.pool.upload(np.concatenate(cache.tables), cache.starts[at], lengths[at], positions)
    q = cache.randn(4, 2 * group, d)
    out = torch.full_like(q.cuda().flatten(1), math.nan)
    cache.pool.attention(0, q.cuda().flatten(1), 2 * group, 0.1, out)
    for r, (i, p) in enumerate(cache.rows):
        slots = torch.from_numpy(cache.slots(i, range(p + 1)))
        want = ref.attention(q[r:r + 1], cache.k[0, slots], cache.v[0, slots], [p + 1], 0.1, **ref.tile_bits(dtype))
        ref.assert_within(out[r:r + 1], *want, f"row {r}")
    cache.upload([0, 0], [300, 40], with_slots=False)
    q = cache.randn(340, 2 * group, d)
    held = [x.flatten(1).to(cache.dtype).cuda() for x in cache.should()]
    for call in ("pages", "rows"):
        out = torch.full_like(q.cuda().flatten(1), math.nan)
        if call == "pages":
            cache.pool.attention(0, q.cuda().flatten(1), 2 * group, 0.1, out)
        else:
            cache.pool.prompt_attention(q.cuda().flatten(1), *held, 2 * group, 0.1, out)
        ref.assert_within(out, *cache.attended(q, 0.1, **ref.tile_bits(dtype)), call)
    cache.pool.close()
