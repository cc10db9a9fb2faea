"""Prompts of float rows whose numbers are near the type's smallest: terms of bf16 keep what is above its
own smallest number, products of floats all of it."""
import math

import pytest
import torch

from tests import fp4_ref as ref
from tests.gpu_util import new_context
from tests.test_gpu_prompt import Prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [-100, -112, -120, -126])
@pytest.mark.parametrize("heads,group,d,split", [(1, 2, 64, None), (2, 1, 128, None), (1, 4, 128, "4"), (1, 1, 256, None)])
def test_small_values(monkeypatch, heads, group, d, split, exponent):
    """Terms of a value leave at most half of bf16's smallest number, 2^-134, of it, and weights sum to 1;
    the output's own sum is of floats, whose smallest is 2^-149: half of it for each of 32 blocks of keys
    and of 10 ranges."""
    if split:
        monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
    ctx = new_context()
    x = Prompts(ctx, "f32", [300, 2], heads, d, 50)
    q, k, v = x.randn(x.n, heads * group, d), x.randn(x.n, heads, d), x.randn(x.n, heads, d)
    v = torch.ldexp(v.double(), torch.tensor(exponent)).float()
    out = torch.full_like(q.cuda().flatten(1), math.nan)
    x.pool.prompt_attention(*(t.cuda().flatten(1) for t in (q, k, v)), heads * group, 0.1, out)
    want, bound = x.attended(q, k, v, 0.1)
    ref.assert_within(out, want, bound + (0.0 if d == 256 else 2.0 ** -134) + 42 * 2.0 ** -150, f"values of 2^{exponent}")
    x.pool.close()
    ctx.close()
