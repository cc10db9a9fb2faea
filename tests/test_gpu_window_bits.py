"""How many bits of a probability enter the product with V in the windowed prefill.

Outputs are rounded to the pool's type, which hides the rounding of probabilities where outputs
are as large as values. Here a row attends two keys of nearly equal scores whose values are v
and -v: the output is v tanh(d / 2), d the difference of the scores, small enough that its
own rounding is far below a probability's. Scores are exact in 32 bits: one product of two numbers
of eight bits, and a scale of a power of two."""
import numpy as np
import pytest
import torch

from tests.gpu_util import new_context
from tests.operator_ref import STEP32, Cache, assert_within

pytestmark = pytest.mark.gpu

SCALE, UNIT = 2.0 ** -4, 2.0 ** -19  # UNIT: the scores' grid, after the scale


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def rounded(x, bits):
    """x in 64 bits rounded to `bits` significant ones."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 2.0 ** bits) / 2.0 ** bits, e)


def scores(n):
    return np.random.RandomState(n).randint(0, 256, n).astype(np.float64) * UNIT


def room(p_bits):
    """What the definition allows besides the output's rounding, of |v| = 1: scores are exact and
    below 1, so that their exponential, the sum of two and the division are each within two steps
    of 2^-23 (fp16's, taken at 2^6 times, in an exponent that is rounded at 2^-22: 1.4 steps of the
    probability), a key range's weight within two; a probability of p_bits bits is off by at most
    2^-p_bits of itself in either of two keys."""
    return 8 * STEP32 + 2.0 ** -p_bits


def test_the_bound_tells_bits_apart():
    """On the CPU: probabilities rounded to 16 bits pass the bound of 16 and fail that of 22."""
    s = scores(300)
    d = s[1:] - s[:-1]
    p = rounded(np.exp(-np.abs(d)), 16)
    off = np.abs((1 - p) / (1 + np.exp(-np.abs(d))) - np.tanh(np.abs(d) / 2)).max()
    assert room(22) < off < room(16)


@pytest.mark.parametrize("dtype,group,d,p_bits", [
    ("bf16", 2, 128, 16), ("f16", 2, 128, 22), ("bf16", 8, 128, 16), ("f32", 2, 128, 32), ("f32", 8, 128, 32),
    ("bf16", 4, 256, 24), ("f16", 4, 256, 24), ("bf16", 2, 256, 24), ("bf16", 1, 256, 24), ("bf16", 8, 256, 24),
    ("f32", 2, 256, 32), ("bf16", 2, 64, 32), ("f16", 1, 80, 32)])
@pytest.mark.parametrize("split", ["1", "3"])
def test_probabilities_keep_their_bits(ctx, dtype, group, d, p_bits, split, monkeypatch):
    print(f"bits {dtype} group {group} d {d}: {p_bits}, {split} key ranges", flush=True)
    monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    monkeypatch.setenv("CKV_PREFILL_SPLIT_MIN", "1")
    n, first = 300, 0
    cache = Cache(ctx, dtype, [n], 1, d, seed=1)
    at = cache.slots(cache.tables[0], np.arange(n))
    s = scores(n)
    sign = torch.from_numpy(1.0 - 2.0 * (np.arange(n) % 2))
    side = torch.where(torch.arange(d) % 3 == 0, -1.0, 1.0).double()
    cache.k[0, at] = 0
    cache.k[0, at, :, 0] = torch.from_numpy(s / SCALE * 2.0 ** 8).to(cache.dtype)[:, None]
    assert torch.equal(cache.k[0, at, 0, 0].double(), torch.from_numpy(s / SCALE * 2.0 ** 8))
    cache.v[0, at] = (sign[:, None] * side).to(cache.dtype)[:, None]
    pool = cache.to_device()
    cache.upload([first], [n], slots=False)
    q = torch.zeros(n, group, d, dtype=cache.dtype)
    q[..., 0] = 2.0 ** -8
    out = torch.empty(n, group * d, dtype=cache.dtype, device="cuda")
    pool.attention_window(0, q.cuda().flatten(1), group, SCALE, 2, out, sinks=0)
    ctx.sync()
    mean = torch.cat([sign[:1], sign[1:] * torch.tanh(torch.from_numpy(s[1:] - s[:-1]) / 2)])
    want = (mean[:, None] * side)[:, None].expand(n, group, d)
    assert_within(out.view(n, group, d), want, torch.full((n, group, d), room(p_bits), dtype=torch.float64), "two keys")
    pool.close()
