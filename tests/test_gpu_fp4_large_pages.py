"""Pages of a 4-bit pool past 4 GiB are copied whole, and no other is touched."""
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context

pytestmark = pytest.mark.gpu


def test_copied_pages_past_four_gigabytes():
    ctx = new_context()
    heads, d, page, blocks = 8192, 256, 4096, 3
    size = page * heads * d * 17 // 32
    assert size > 2 ** 32
    caches = [torch.zeros(blocks * size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    # bytes at both ends of each page and all over it, another pattern for each
    at = torch.cat([torch.arange(4096), torch.arange(0, size - 1, 1_000_003), size - 4096 + torch.arange(4096)]).unique().cuda()
    marks = [[((at * 31 + 7 * b + 3 * c + 1) % 251).to(torch.uint8) for b in range(blocks)] for c in range(2)]
    for cache, mark in zip(caches, marks):
        for b in range(blocks):
            cache[b * size + at] = mark[b]
    pool = ckv.Pool(ctx, 1, blocks, page, heads, d, torch.bfloat16, *caches, fp4=True)
    assert pool.buffers()[2] == blocks * size
    print("copy page 1 to page 2", flush=True)
    pool.copy_blocks([1], [2])
    torch.cuda.synchronize()
    for cache, mark in zip(caches, marks):
        for b, source in ((0, 0), (1, 1), (2, 1)):
            assert torch.equal(cache[b * size + at], mark[source])
            assert int(cache[b * size:(b + 1) * size].count_nonzero()) == int(mark[source].count_nonzero())
    pool.close()
    ctx.close()
