"""How many bits of a probability enter the product with V in the windowed prefill.

Outputs are rounded to the pool's type, which hides the rounding of probabilities where outputs
are as large as values. Here a row attends a sink of score 0 and value 0 and two keys of nearly equal
scores below it whose values are v and -v: the output is the difference of their probabilities,
small enough that its own rounding is far below theirs. Scores are exact in 32 bits: sums of two
products of numbers of eight bits, and a scale of a power of two."""
import numpy as np
import pytest
import torch

from tests.gpu_util import new_context
from tests.operator_ref import ROUND, STEP32, Cache, assert_within

pytestmark = pytest.mark.gpu

SCALE, ROWS = 2.0 ** -4, 600


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def numbers():
    """Of each token its score's own part, r 2^-19 with r below 256; of each row what it takes from
    the scores of both, j 2^-8 with j below 256: probabilities from 0.36 to 1 of the sink's."""
    rng = np.random.RandomState(1)
    return rng.randint(0, 256, ROWS) * 2.0 ** -19, rng.randint(0, 256, ROWS) * 2.0 ** -8


def outputs(weight):
    """Of rows 2 on, for values of 1 at even tokens and -1 at odd ones, with weight(p) of each of
    the two entering the product with V."""
    own, taken = numbers()
    a, b = np.exp(own[1:-1] - taken[2:]), np.exp(own[2:] - taken[2:]) # tokens i - 1 and i of row i
    return (1 - 2 * (np.arange(2, ROWS) % 2)) * (weight(b) - weight(a)) / (1 + a + b)


def room(p_bits):
    """What 32-bit arithmetic may add to an output's rounding, of |v| = 1. Scores are exact. A
    probability's exponent is a product and a sum rounded at 2^-24 of at most 2 (fp16's, taken at 2^6
    times, at 2^-22), its exponential within two steps of 2^-23, a key range's weight within two, the
    sums and the division within two: 8 steps of each of two probabilities that make up at most
    2/3 of the sum. Rounded to p_bits bits a probability is off by 2^-p_bits of itself at most."""
    return (8 * STEP32 + 2.0 ** -p_bits) * 2 / 3


def bf16_terms(p, n):
    """p as the sum of n roundings to bf16, each of what those before it left."""
    left, total = torch.from_numpy(p).float(), torch.zeros(p.size)
    for _ in range(n):
        term = left.bfloat16().float()
        left, total = left - term, total + term
    return total.double().numpy()


def test_the_bound_tells_bits_apart():
    """On the CPU: probabilities as two bf16 terms pass the bound of 16 bits and fail that of 22 by
    more than the output's rounding; as three they pass that of 24."""
    exact = outputs(lambda p: p)
    slack = np.abs(exact) * ROUND[torch.bfloat16] * (1 + 1e-3)
    for terms, bits, passes in ((1, 8, True), (1, 16, False), (2, 16, True), (2, 22, False), (3, 24, True)):
        off = np.abs(outputs(lambda p: bf16_terms(p, terms)) - exact)
        assert (np.all(off <= room(bits))) if passes else np.any(off > room(bits) + 2 * slack)


@pytest.mark.parametrize("dtype,group,d,p_bits", [
    ("bf16", 2, 128, 16), ("f16", 2, 128, 22), ("bf16", 8, 128, 16), ("f32", 2, 128, 32), ("f32", 8, 128, 32),
    ("bf16", 4, 256, 24), ("f16", 4, 256, 24), ("bf16", 2, 256, 24), ("bf16", 1, 256, 24), ("bf16", 8, 256, 24),
    ("f32", 2, 256, 32), ("bf16", 2, 64, 32), ("f16", 1, 80, 32)])
@pytest.mark.parametrize("split", ["1", "3"])
def test_probabilities_keep_their_bits(ctx, dtype, group, d, p_bits, split, monkeypatch):
    print(f"bits {dtype} group {group} d {d}: {p_bits}, {split} key ranges", flush=True)
    monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    monkeypatch.setenv("CKV_PREFILL_SPLIT_MIN", "1")
    own, taken = numbers()
    cache = Cache(ctx, dtype, [ROWS], 1, d, seed=1)
    at = cache.slots(cache.tables[0], np.arange(ROWS))
    side = torch.where(torch.arange(d) % 3 == 0, -1.0, 1.0).double()
    sign = torch.from_numpy(1.0 - 2.0 * (np.arange(ROWS) % 2))
    k, v = torch.zeros(ROWS, d, dtype=torch.float64), sign[:, None] * side
    k[1:, 0], k[1:, 1] = torch.from_numpy(own[1:] / SCALE * 2.0 ** 8), 1.0
    v[0] = 0
    q = torch.zeros(ROWS, group, d, dtype=torch.float64)
    q[..., 0], q[..., 1] = 2.0 ** -8, torch.from_numpy(-taken / SCALE)[:, None]
    cache.k[0, at], cache.v[0, at] = k.to(cache.dtype)[:, None], v.to(cache.dtype)[:, None]
    qt = q.to(cache.dtype)
    assert torch.equal(cache.k[0, at, 0].double(), k) and torch.equal(qt.double(), q)
    pool = cache.to_device()
    cache.upload([0], [ROWS], slots=False)
    out = torch.empty(ROWS, group * d, dtype=cache.dtype, device="cuda")
    pool.attention_window(0, qt.cuda().flatten(1), group, SCALE, 2, out, sinks=1)
    ctx.sync()
    want = torch.from_numpy(outputs(lambda p: p))[:, None] * side
    want = want[:, None].expand(-1, group, d)
    assert_within(out.view(ROWS, group, d)[2:], want, torch.full(want.shape, room(p_bits), dtype=torch.float64), "rows")
    pool.close()
