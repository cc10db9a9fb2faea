"""Scores that overflow to minus infinity over a pool held in 4 bits weigh nothing, wherever they stand
in a row."""
import pytest
import torch

from tests import fp4_ref as ref
from tests.gpu_util import force_plan, new_context

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("scale", [0.1, 1.0, -3.0])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64), ("bf16", 256), ("f32", 128)])
@pytest.mark.parametrize("lost,split", [(slice(0, 70), None), (slice(0, 70), "1"), (slice(0, 299), None), (slice(200, 260), "2")])
def test_scores_of_minus_infinity(ctx, monkeypatch, lost, split, dtype, d, scale, rows):
    """Of 300 tokens some have 2^100 in a feature where the query has 2^30 of the other sign: they are
    attended as if they were not there."""
    print(f"overflow {dtype} {d} {scale} {lost} {split} rows {rows}", flush=True)
    force_plan(monkeypatch, split)
    cache = ref.Cache(ctx, dtype, [300], 2, d, seed=40)
    k, v = cache.randn(300, 2, d), cache.randn(300, 2, d)
    k[:, :, 0] = 0
    k[lost, :, 0] = 2.0 ** 100
    cache.upload([0], [300])
    cache.pool.append(0, k.cuda().flatten(1), v.cuda().flatten(1))
    cache.keep(0, k, v)
    q = cache.randn(rows, 4, d)
    q[:, :, 0] = -2.0 ** 30 if scale > 0 else 2.0 ** 30
    cache.upload([300 - rows], [rows], with_slots=False)
    out = torch.empty(rows, 4 * d, dtype=cache.dtype, device="cuda")
    cache.pool.attention(0, q.cuda().flatten(1), 4, scale, out)
    there = torch.ones(300, dtype=torch.bool)
    there[lost] = False
    kept, values = (x[0, torch.from_numpy(cache.slots(0, range(300)))][there] for x in (cache.k, cache.v))
    seen = [int(there[:300 - rows + r + 1].sum()) for r in range(rows)]
    if min(seen) == 0:  # every score of the first rows: the sum of the weights is 0
        first = sum(n == 0 for n in seen)
        assert torch.isnan(out[:first].float()).all()
        q, out, seen = q[first:], out[first:], seen[first:]
    bits = ref.decode_bits(dtype) if rows == 1 else ref.tile_bits(dtype)
    ref.assert_within(out, *ref.attention(q, kept, values, seen, scale, **bits), "overflow")
    cache.pool.close()
