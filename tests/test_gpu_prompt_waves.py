"""Prompt attention of 128-wide 16-bit rows by workgroups of eight waves, as large launches run it, and
rows that lie more than 4 GiB apart, by four and by eight; against 64 bits."""
import math

import pytest
import torch

from tests import fp4_ref as ref
from tests.gpu_util import new_context
from tests.test_gpu_prompt import Prompts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group", [(2, 1), (2, 2), (1, 4), (1, 3), (2, 8)])
# (a workgroup has 256 / heads rows and eight stages of 32 keys: lengths on both sides of these)
@pytest.mark.parametrize("counts", [[1], [31, 32, 33, 1], [255, 64, 257], [288, 289], [512, 129, 1], [641], [319, 321]])
def test_eight_waves(ctx, monkeypatch, dtype, heads, group, counts):
    print(f"eight waves {dtype} {heads} x {group} {counts}", flush=True)
    monkeypatch.setenv("CKV_PREFILL_WAVES", "8")
    x = Prompts(ctx, dtype, counts, heads, 128, 41)
    q, k, v, gate = (x.randn(x.n, n, 128) for n in (heads * group, heads, heads, heads * group))
    qd, kd, vd, gd = (t.cuda().flatten(1) for t in (q, k, v, gate))
    out = torch.full_like(qd, math.nan)
    x.pool.prompt_attention(qd, kd, vd, heads * group, 0.09, out)
    want, bound = x.attended(q, k, v, 0.09)
    ref.assert_within(out, want, bound, "eight waves")
    out.fill_(math.nan)
    x.pool.prompt_attention(qd, kd, vd, heads * group, 0.09, out, gate=gd)
    ref.assert_within(out, *ref.gated(want, bound, gate), "gated")
    x.pool.close()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype,group", [("bf16", 1), ("f16", 2), ("bf16", 4)])
@pytest.mark.parametrize("at", [3, 290, 400])
def test_what_is_not_attended_weighs_nothing(ctx, monkeypatch, bad, dtype, group, at):
    """A value and a key that are not finite, in the first block, in a middle one and in the last, reach the
    rows behind them in their prompt alone."""
    print(f"not finite {dtype} {group} {bad} at {at}", flush=True)
    monkeypatch.setenv("CKV_PREFILL_WAVES", "8")
    counts = [60, 410, 33]
    x = Prompts(ctx, dtype, counts, 2, 128, 42)
    q, k, v = x.randn(x.n, 2 * group, 128), x.randn(x.n, 2, 128), x.randn(x.n, 2, 128)
    clean = x.attended(q, k, v, 0.1)
    row, end = 60 + at, 470
    k[row, 0, 5], v[row, 1, 9] = math.nan, bad
    out = torch.empty_like(q.cuda().flatten(1))
    x.pool.prompt_attention(*(t.cuda().flatten(1) for t in (q, k, v)), 2 * group, 0.1, out)
    got = out.cpu().view(x.n, 2 * group, 128)
    lost = torch.zeros(got.shape, dtype=torch.bool)
    lost[row:end, :group] = True  # a NaN score
    lost[row:end, group:, 9] = True
    assert not torch.isfinite(got[lost].float()).any()
    if math.isinf(bad):
        assert (got[row:end, group:, 9].double() == bad).all()
    ref.assert_within(torch.where(lost, 0, got), torch.where(lost, 0.0, clean[0]), torch.where(lost, 0.0, clean[1]), "the others")
    x.pool.close()


@pytest.mark.parametrize("gap", [8, 40])
def test_parts_of_wider_rows(ctx, monkeypatch, gap):
    monkeypatch.setenv("CKV_PREFILL_WAVES", "8")
    x = Prompts(ctx, "bf16", [300, 45], 2, 128, 43)
    wide = torch.full((x.n, 512 + 256 + 256 + gap), math.nan, dtype=x.dtype, device="cuda")
    q, k, v = x.randn(x.n, 4, 128), x.randn(x.n, 2, 128), x.randn(x.n, 2, 128)
    parts = [wide[:, :512], wide[:, 512:768], wide[:, 768:1024]]
    for part, t in zip(parts, (q, k, v)):
        part.copy_(t.flatten(1))
    out = torch.full((x.n, 512), math.nan, dtype=x.dtype, device="cuda")
    x.pool.prompt_attention(*parts, 4, 0.1, out)
    ref.assert_within(out, *x.attended(q, k, v, 0.1), "strided")
    x.pool.close()


def test_a_launch_that_takes_eight_waves_by_itself(ctx):
    """As many rows as give every compute unit two such workgroups (of 128 rows, for 8 of the heads)."""
    counts = [9000, 57, 3000]
    x = Prompts(ctx, "bf16", counts, 8, 128, 44)
    q, k, v = x.randn(x.n, 16, 128), x.randn(x.n, 8, 128), x.randn(x.n, 8, 128)
    qd, kd, vd = (t.cuda().flatten(1) for t in (q, k, v))
    out, again = torch.full_like(qd, math.nan), torch.full_like(qd, math.nan)
    x.pool.prompt_attention(qd, kd, vd, 16, 0.1, out)
    x.pool.prompt_attention(qd, kd, vd, 16, 0.1, again)
    assert torch.equal(out, again) and torch.isfinite(out).all()
    for first, rows in ((0, [0, 31, 32, 127, 128, 4999, 8959, 8999]), (9000, [0, 56]), (9057, [1, 255, 2999])):
        n = max(rows) + 1
        want = ref.attention(q[first:first + n][rows], k[first:first + n], v[first:first + n], [r + 1 for r in rows], 0.1,
                             **ref.tile_bits("bf16"))
        ref.assert_within(out[first:first + n][rows], *want, f"rows of the prompt at {first}")
    x.pool.close()


@pytest.mark.parametrize("waves", ["4", "8"])
@pytest.mark.parametrize("dtype,group", [("bf16", 1), ("f16", 2), ("bf16", 4), ("f16", 3)])
def test_rows_past_four_gigabytes(ctx, monkeypatch, waves, dtype, group):
    print(f"far rows {dtype} {group} waves {waves}", flush=True)
    monkeypatch.setenv("CKV_PREFILL_WAVES", waves)
    x = Prompts(ctx, dtype, [300, 1, 40], 1, 128, 45)
    wide = torch.full((x.n, 1 << 23), math.nan, dtype=x.dtype, device="cuda")
    assert wide.numel() * 2 > 2 ** 32
    q, k, v = x.randn(x.n, group, 128), x.randn(x.n, 1, 128), x.randn(x.n, 1, 128)
    keys, values = wide[:, 8:136], wide[:, -128:]
    keys.copy_(k.flatten(1))
    values.copy_(v.flatten(1))
    out = torch.full((x.n, group * 128), math.nan, dtype=x.dtype, device="cuda")
    x.pool.prompt_attention(q.cuda().flatten(1), keys, values, group, 0.1, out)
    ref.assert_within(out, *x.attended(q, k, v, 0.1), "far rows")
    x.pool.close()
