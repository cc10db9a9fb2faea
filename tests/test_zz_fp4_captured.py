"""Captured graphs over pools held in 4 bits: steps and chunks replayed on new inputs, with eager work of
their own between."""
import pytest
import torch

from chibillm_amd import ckv
from tests import fp4_ref as ref

pytestmark = pytest.mark.gpu

WIDE = pytest.param("f16", 4, 256, marks=pytest.mark.skip(
    reason="ended once in a GPU fault whose cause was not found: captures of such pools are refused"))


@pytest.mark.parametrize("counts", [[1, 1], [50, 9]])
@pytest.mark.parametrize("dtype,group,d", [("bf16", 2, 128), ("f32", 1, 64), WIDE])
def test_captured_steps_and_chunks(dtype, group, d, counts):
    """A step, or a chunk rotated, appended and attended; a batch's first tiles are refused under
    capture, which goes on."""
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    rotation = ckv.Rotation(1e5, 0, "pairs", "linear", 2.0)
    with torch.cuda.stream(stream):
        cache = ref.Cache(own, dtype, [1100, 60], 2, d, seed=20)
        cache.fill()
        pool, n = cache.pool, sum(counts)
        cache.upload([x - c for x, c in zip(cache.lengths, counts)], counts)
        q, k, v = (cache.randn(n, x, d).cuda().flatten(1) for x in (2 * group, 2, 2))
        out, turned = torch.empty_like(q), torch.empty_like(q)
        held = [torch.empty_like(k) for _ in range(2)]

        def call():
            if n == 2:
                pool.rotate_append_decode(0, rotation, k, v, q, 2 * group, 0.1, out, None, *held)
            else:
                pool.rotate_append(0, rotation, q, turned, 2 * group, k, v, *held)
                pool.attention(0, turned, 2 * group, 0.1, out)

        if n != 2:  # the work list is not made yet
            stream.synchronize()
            empty = torch.cuda.CUDAGraph()
            with torch.cuda.graph(empty, stream=stream):
                with pytest.raises(ckv.CkvError) as refused:
                    pool.attention(0, q, 2 * group, 0.1, out)
                assert refused.value.name == "ckv.invalid_argument"
                held[0].zero_()
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(4):
            for x in (q, k, v):
                x.normal_()
            call()
            stream.synchronize()
            want = [x.clone() for x in (out, *held)] + [b.clone() for b in cache.bytes]
            for x in (out, *held):
                x.zero_()
            graph.replay()
            stream.synchronize()
            for got, w in zip((out, *held, *cache.bytes), want):
                assert torch.equal(got, w)
        pool.close()
    own.close()
