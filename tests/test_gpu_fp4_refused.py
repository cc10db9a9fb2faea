"""4-bit pools of 256-wide heads once a call on them met a stream capture: appends and attention are
refused and their numbers stay readable."""
import pytest
import torch

from chibillm_amd import ckv
from tests import fp4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_a_wide_pool_that_met_a_capture(dtype):
    stream = torch.cuda.Stream()
    own = ckv.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        cache = ref.Cache(own, dtype, [90, 20], 2, 256, seed=30)
        cache.fill()
        pool = cache.pool
        cache.upload([80, 19], [10, 1])
        q, k, v = (cache.randn(11, n, 256).cuda().flatten(1) for n in (4, 2, 2))
        out = torch.zeros_like(q)
        rotation = ckv.Rotation(1e4)
        calls = [lambda: pool.attention(0, q, 4, 0.1, out), lambda: pool.append(0, k, v),
                 lambda: pool.rotate_append(0, rotation, q, out, 4, k, v),
                 lambda: pool.rope_append(0, k, v, 1e4)]
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(ckv.CkvError) as refused:
                pool.append(0, k, v)
            out.zero_()
        assert refused.value.name == "ckv.invalid_argument"
        for call in calls:
            with pytest.raises(ckv.CkvError) as refused:
                call()
            assert refused.value.name == "ckv.invalid_argument"
        stream.synchronize()
        assert not out.any()
        cache.check(0, "as it was")  # gathers are not refused
        pool.close()
    own.close()
