"""Pools held in 4 bits: what appends, rotated appends, copies and gathers leave in them, exactly, at
the levels' borders, over every layout, and in pools past 4 GiB."""
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


def special(cache, n):
    """Rows with blocks of every kind among ordinary ones: zeros of both signs, the type's largest and
    smallest numbers, infinities, NaN, and numbers on the levels' borders."""
    x = cache.randn(n, cache.h, cache.d) * torch.exp2(torch.randint(-12, 13, (n, cache.h, cache.d // 32, 1), generator=cache.g)
                                                     ).expand(-1, -1, -1, 32).reshape(n, cache.h, cache.d).to(cache.dtype)
    b = x.view(n * cache.h, -1, 32)
    info = torch.finfo(cache.dtype)
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5] * 3 + [4.0, -0.0], dtype=cache.dtype)
    below = border - border * info.eps
    kinds = [torch.zeros(32), -torch.zeros(32), torch.full((32,), info.max), torch.full((32,), info.tiny),
             torch.full((32,), info.tiny * info.eps), border, -border, border * 2.0 ** -13, below, -border * (1 + info.eps),
             torch.cat([torch.full((1,), info.max), torch.zeros(31)]), torch.linspace(0, 1, 32) * info.tiny]
    for j, kind in enumerate(kinds):
        b[(5 * j) % b.shape[0], j % b.shape[1]] = kind.to(cache.dtype)
    if n > 4:
        b[1, 0, 7], b[2, 0, 31], b[3, 0, 0] = math.inf, -math.inf, math.nan
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,d,page,counts", [(1, 64, 16, [1]), (2, 128, 16, [17, 1, 40]), (3, 256, 32, [33, 64]),
                                                (8, 128, 64, [300, 5]), (5, 64, 4096, [70]), (4, 64, 16, [700])])
def test_appended_rows(ctx, dtype, heads, d, page, counts):
    """Every kind of block, read back exactly; tokens that no row wrote keep their bytes."""
    print(f"append {dtype} {heads} x {d} pages of {page} rows {counts}", flush=True)
    cache = ref.Cache(ctx, dtype, [n + 9 for n in counts], heads, d, page=page, layers=2, seed=1)
    cache.upload([3] * len(counts), counts)
    k, v = special(cache, len(cache.rows)), special(cache, len(cache.rows)).flip(0)
    cache.pool.append(1, k.cuda().flatten(1), v.cuda().flatten(1))
    cache.keep(1, k, v)
    cache.check(1, "appended")  # (what was not written reads as NaN)
    assert torch.isnan(cache.read(0)[0].float()).all()
    at = cache.bytes[0].numel() // 2
    assert all(bool((b[:at] == 255).all()) for b in cache.bytes)
    # rows again, in the middle of what is there
    cache.upload([4] + [0] * (len(counts) - 1), [1] + [0] * (len(counts) - 1))
    k, v = cache.randn(1, heads, d), cache.randn(1, heads, d)
    cache.pool.append(1, k.cuda().flatten(1), v.cuda().flatten(1))
    cache.keep(1, k, v)
    cache.check(1, "one more")
    cache.pool.close()


ROTATIONS = {
    "plain": dict(theta=1e4),
    "linear": dict(theta=1e6, scaling="linear", factor=3.0, layout="pairs"),
    "bands": dict(theta=5e5, scaling="bands", factor=8.0, low=1.0, high=4.0, original=8192),
    "yarn": dict(theta=1e6, scaling="yarn", factor=4.0, low=1.0, high=32.0, original=4096, layout="pairs"),
    "yarn of one factor": dict(theta=1e4, scaling="yarn", factor=1.0, low=1.0, high=32.0, original=512),
    "magnified": dict(theta=1e4, magnitude=1.75, layout="pairs"),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,q_heads,d,rotary,rows", [(2, 6, 128, 128, 37), (1, 1, 64, 64, 1), (3, 3, 64, 34, 90), (2, 0, 256, 64, 21),
                                                         (8, 16, 128, 128, 900), (1, 9, 256, 256, 40), (4, 4, 128, 2, 19)])
@pytest.mark.parametrize("kind", list(ROTATIONS))
def test_rotated_appends(ctx, dtype, heads, q_heads, d, rotary, rows, kind):
    """Keys turned in 64 bits and rounded once; held rows are the cache's; queries within the
    arithmetic's bound."""
    print(f"rotated append {dtype} {heads} {q_heads} {d} {rotary} {rows} {kind}", flush=True)
    rotation = ckv.Rotation(rotary_dim=rotary, **ROTATIONS[kind])
    cache = ref.Cache(ctx, dtype, [rows + 3], heads, d, seed=2)
    positions = cache.upload([2], [rows])
    q, k, v = cache.randn(rows, max(q_heads, 1), d), cache.randn(rows, heads, d), special(cache, rows)
    turned, kd = torch.empty_like(q.cuda()), k.cuda().flatten(1)
    held = [torch.empty_like(kd), torch.empty_like(kd)]
    cache.pool.rotate_append(0, rotation, q.cuda().flatten(1) if q_heads else None, turned.flatten(1) if q_heads else None, q_heads, kd,
                             v.cuda().flatten(1), *held)
    k64, _ = ref.rotated(k, positions, rotation)
    cache.keep(0, k64, v)
    cache.check(0, kind)
    for got, want in zip(held, (cache.k, cache.v)):
        want = want[0, cache.at]
        got = got.cpu().double().reshape(want.shape)
        assert torch.equal(got.nan_to_num(), want.nan_to_num()) and torch.equal(torch.isnan(got), torch.isnan(want))
    if q_heads:
        ref.assert_within(turned, *ref.rotated(q, positions, rotation), f"queries {kind}")
    cache.pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rotations_that_overflow_and_special_keys(ctx, dtype):
    """A rotated block that reaches 2^128, or with an infinity or NaN on either side of a pair, reads
    as NaN; others of the head do not."""
    cache = ref.Cache(ctx, dtype, [40], 2, 128, seed=3)
    rotation = ckv.Rotation(1e4)
    positions = cache.upload([0], [40])
    k, v = special(cache, 40), cache.randn(40, 2, 128)
    info = torch.finfo(cache.dtype)
    k[9, 0, 3] = k[9, 0, 67] = info.max  # a turn by 9 radians times 10000^(-6/128)
    k[10, 1, 100] = math.inf
    cache.pool.rotate_append(0, rotation, None, None, 0, k.cuda().flatten(1), v.cuda().flatten(1))
    k64, _ = ref.rotated(k, positions, rotation)
    cache.keep(0, k64, v)
    cache.check(0, "overflow")
    assert torch.isnan(cache.k[0, cache.at[10], 1, 96:]).all() and torch.isnan(cache.k[0, cache.at[10], 1, 32:64]).all()
    assert torch.isfinite(cache.k[0, cache.at[10], 1, 64:96]).all()
    cache.pool.close()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64), ("f16", 256)])
def test_the_older_rotated_calls(ctx, dtype, d):
    """ckv_rope_append is the rotation without scaling, bit for bit; ckv_rope turns queries."""
    cache = ref.Cache(ctx, dtype, [50], 2, d, layers=2, seed=4)
    positions = cache.upload([0], [50])
    q, k, v = cache.randn(50, 4, d), cache.randn(50, 2, d), cache.randn(50, 2, d)
    cache.pool.rope_append(0, k.cuda().flatten(1), v.cuda().flatten(1), 1e6, d // 2)
    rotation = ckv.Rotation(1e6, d // 2)
    cache.pool.rotate_append(1, rotation, None, None, 0, k.cuda().flatten(1), v.cuda().flatten(1))
    k64, _ = ref.rotated(k, positions, rotation)
    for layer in (0, 1):
        cache.keep(layer, k64, v)
        cache.check(layer, f"layer {layer}")
    out = torch.empty_like(q.cuda().flatten(1))
    cache.pool.rope(q.cuda().flatten(1), out, 4, 1e6, d // 2)
    # that call's angle is float(position) * float(theta^(-2j/rotary)): the exponent is off by half a
    # step (so the power by at most ln(theta) < 14 of them), the power by two, the product by half
    ref.assert_within(out, *ref.rotated(q, positions, rotation, 17 * 2.0 ** -24), "rope")
    cache.pool.close()


@pytest.mark.parametrize("dtype,odd", [("bf16", 1), ("f16", 3), ("f32", 1), ("bf16", 4)])
def test_rows_of_any_alignment(ctx, dtype, odd):
    cache = ref.Cache(ctx, dtype, [70], 2, 128, seed=5)
    cache.upload([0], [70])
    k, v = cache.randn(70, 2, 128), cache.randn(70, 2, 128)

    def apart(x):
        room = torch.empty(x.numel() + odd, dtype=x.dtype, device="cuda")
        room[odd:] = x.flatten().cuda()
        return room[odd:].view(x.shape[0], -1)

    held = [apart(torch.zeros_like(k)) for _ in range(2)]
    q, out = apart(k), apart(k)
    rotation = ckv.Rotation(1e4, 64, "pairs")
    cache.pool.rotate_append(0, rotation, q, out, 2, apart(k), apart(v), *held)
    k64, room = ref.rotated(k, range(70), rotation)
    cache.keep(0, k64, v)
    cache.check(0, "unaligned")
    for i, want in enumerate((cache.k, cache.v)):
        assert torch.equal(held[i].cpu().double().view(70, 2, 128), want[0, cache.at])
    ref.assert_within(out, k64, room, "unaligned queries")
    cache.pool.append(0, apart(v), apart(k))
    cache.keep(0, v, k)
    cache.check(0, "unaligned append")
    read = [apart(torch.zeros_like(k)) for _ in range(2)]
    cache.pool.gather(0, 0, cache.tables[0].size, 70, *read)
    assert torch.equal(read[0].cpu().double().view(70, 2, 128), cache.should()[0])
    cache.pool.close()


def test_copied_blocks(ctx):
    """Blocks copied in every layer as their bytes."""
    cache = ref.Cache(ctx, "bf16", [100], 3, 64, page=32, layers=3, spare=4, seed=6)
    for layer in range(3):
        cache.fill(layer)
    source, target = cache.tables[0][:3], cache.free[:3]
    cache.pool.copy_blocks(source, target)
    cache.tables[0] = np.concatenate([target, cache.tables[0][3:]])
    for t, s in zip(target, source):
        t, s = int(t) * 32, int(s) * 32
        cache.k[:, t:t + 32], cache.v[:, t:t + 32] = cache.k[:, s:s + 32].clone(), cache.v[:, s:s + 32].clone()
    cache.upload([0], [100], with_slots=False)
    for layer in range(3):
        cache.check(layer, f"layer {layer}")
    cache.pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_far_positions(ctx, dtype):
    """Angles at positions that 32-bit floats do not hold: a turn is off by at most what 2^32 times
    the 80-bit frequency's own rounding is, and a code changes only next to a border."""
    positions = np.array([2 ** 24 + 1, 2 ** 31 - 5, 2 ** 31 + 3, 2 ** 32 - 17, 123456789])
    heads, d, n = 2, 128, len(positions)
    cache = ref.Cache(ctx, dtype, [n], heads, d, seed=7)
    cache.upload([0], [n])
    pool = cache.pool
    # a batch whose positions no table covers: rows rotated without one
    rows = cache.randn(n, heads, d)
    for layout in ("halves", "pairs"):
        rotation = ckv.Rotation(1e6, 0, layout, "bands", 8.0, 1.0, 4.0, 8192)
        wide = ckv.Pool(ctx, 1, 2, 2 ** 31 - 1, 1, d, cache.dtype, *[torch.empty(16, device="cuda") for _ in range(2)])
        wide.upload([0, 1, 0], [0] * n, [3] * n, positions)
        out = torch.empty(n, heads * d, dtype=cache.dtype, device="cuda")
        wide.rotate(rotation, rows.cuda().flatten(1), out, heads)
        want, room = ref.rotated(rows, positions, rotation)
        ref.assert_within(out, want, room + 2.0 ** -28 * rows.abs().max().double(), f"far {layout}")
        wide.close()
    pool.close()


@pytest.mark.parametrize("dtype,heads,d,blocks", [("bf16", 8, 256, 270_000), ("f32", 1, 64, 8_500_000)])
def test_pools_past_four_gigabytes(ctx, dtype, heads, d, blocks):
    """Appends, gathers and attention where offsets pass 32 bits."""
    pool = ckv.Pool(ctx, 1, blocks, 16, heads, d, DTYPES[dtype], fp4=True)
    assert pool.buffers()[2] > 2 ** 32
    g = torch.Generator().manual_seed(8)
    table = np.array([blocks - 1, 3, blocks - 2, blocks // 2 + 1, 0])
    n = 75
    positions = np.arange(n)
    slots = table[positions // 16].astype(np.int64) * 16 + positions % 16
    pool.upload(table, [0] * n, [5] * n, positions, slots)
    k, v, q = (torch.randn(n, x, d, generator=g).to(DTYPES[dtype]) for x in (heads, heads, 2 * heads))
    pool.append(0, k.cuda().flatten(1), v.cuda().flatten(1))
    read = [torch.empty(n, heads * d, dtype=DTYPES[dtype], device="cuda") for _ in range(2)]
    pool.gather(0, 0, 5, n, *read)
    kept = [ref.held(x.double().flatten(1), dtype).view(x.shape) for x in (k, v)]
    for got, want in zip(read, kept):
        assert torch.equal(got.cpu().double().view(want.shape), want)
    out = torch.empty(n, 2 * heads * d, dtype=DTYPES[dtype], device="cuda")
    pool.attention(0, q.cuda().flatten(1), 2 * heads, 0.1, out)
    ref.assert_within(out, *ref.attention(q, *kept, positions + 1, 0.1, **ref.tile_bits(dtype)), "tiles")
    pool.upload(table, [0], [5], [n - 1], slots[-1:])
    one = torch.empty(1, 2 * heads * d, dtype=DTYPES[dtype], device="cuda")
    pool.attention(0, q[-1:].cuda().flatten(1), 2 * heads, 0.1, one)
    ref.assert_within(one, *ref.attention(q[-1:], *kept, [n], 0.1, **ref.decode_bits(dtype)), "decode")
    pool.close()


def test_what_is_refused(ctx):
    """Calls that have no 4-bit form say so and leave the pool as it was."""
    cache = ref.Cache(ctx, "bf16", [40], 2, 128, seed=9)
    cache.fill()
    pool, x = cache.pool, torch.zeros(40, 256, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros_like(x)
    for call in (lambda: pool.attention_window(0, x, 2, 1.0, 8, y), lambda: pool.element_offset(0, 0, 0, 0, 0),
                 lambda: pool.compact([1], [0], [1]), lambda: pool.checkpoint_pack([0], 16, x, y),
                 lambda: pool.append_decode_noalloc(0, x, x.clone(), x.clone(), 2, 1.0, y)):
        with pytest.raises(ckv.CkvError) as refused:
            call()
        assert refused.value.name == "tensor_op.unsupported_dtype"
    cache.check(0, "after refusals")
    pool.close()


def test_batches_without_rows(ctx):
    cache = ref.Cache(ctx, "f16", [20], 2, 128, seed=10)
    cache.fill()
    cache.upload([0], [0])
    none = torch.empty(0, 256, dtype=torch.float16, device="cuda")
    rotation = ckv.Rotation(1e4)
    cache.pool.append(0, none, none)
    cache.pool.rotate_append(0, rotation, none, none, 2, none, none, none, none)
    cache.pool.rotate_append_decode(0, rotation, none, none, none, 2, 1.0, none)
    cache.pool.attention(0, none, 2, 1.0, none)
    cache.pool.prompt_attention(none, none, none, 2, 1.0, none)
    cache.pool.rotate(rotation, none, none, 2)
    cache.check(0, "as it was")
    cache.pool.close()
