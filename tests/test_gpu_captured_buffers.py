"""Buffers that grow after a capture stay with the pool whose calls were captured: its graphs read
the old ones, and they go when the pool goes."""
import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.operator_ref import Cache

pytestmark = pytest.mark.gpu


def grow(pool, blocks, entries):
    """A batch of one row whose table has so many entries: the pool's metadata buffer grows."""
    pool.upload(np.zeros(entries, np.uint32) + blocks - 1, [0], [entries], [5])


def cycle(own, stream, captured):
    """A pool whose metadata grows from 2 to 48 MB, behind a captured call or not; its allocations and
    frees from its making to its end."""
    before = own.allocations()
    cache = Cache(own, "bf16", [40], 2, 128, seed=1)
    pool = cache.to_device()
    cache.upload([39], [1])
    q = cache.randn(1, 4, 128).cuda().flatten(1)
    out = torch.empty_like(q)
    pool.attention_window(0, q, 4, 0.1, 20, out)
    stream.synchronize()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph, stream=stream):
            pool.attention_window(0, q, 4, 0.1, 20, out)
    for entries in (500_000, 3_000_000, 12_000_000):
        grow(pool, cache.blocks, entries)
    if captured:
        out.zero_()
        graph.replay()
        stream.synchronize()
        # the graph's lists are where they were; its batch is not this one, but its table is still read
        assert torch.equal(out, want)
        del graph
    pool.close()
    return own.allocations() - before


def test_buffers_that_grew_after_a_capture_go_with_the_pool():
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        for _ in range(8):  # until every staging slot of the context has its size
            plain = cycle(own, stream, False)
        for _ in range(3):
            assert cycle(own, stream, True) == plain  # every allocation has its free
        # a pool that captured nothing frees what it outgrows at once, though others did
        assert cycle(own, stream, False) == plain
    own.close()
