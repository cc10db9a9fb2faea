"""Layers past 4 GiB, whose page offsets take 64 bits in kernels of their own: a sequence's pages lie
on both sides of the line, and what the operators give there is what they give in a small pool, bit
for bit."""
import math

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests.gpu_util import new_context
from tests.operator_ref import Cache

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def bits(x):
    return x.contiguous().view({2: torch.int16, 4: torch.int32}[x.element_size()]).cpu()


@pytest.mark.parametrize("dtype,heads,d,groups", [
    ("bf16", 8, 128, (1, 2, 4, 8)), ("f16", 8, 128, (2, 8)), ("bf16", 4, 256, (1, 2, 4, 8)), ("f16", 4, 256, (4,)),
    ("f32", 4, 128, (1, 8))])
def test_a_layer_past_four_gigabytes(ctx, dtype, heads, d, groups, monkeypatch):
    print(f"far layer {dtype} {heads} x {d}", flush=True)
    lengths, got = [830, 40, 131], []
    cache = Cache(ctx, dtype, lengths, heads, d, spare=20, seed=31)
    page_bytes = PAGE * heads * d * cache.k.element_size()
    far = (2 ** 32 + 2 ** 28) // page_bytes
    # every other page of the small pool is one of the far pool's first, the others its last
    place = np.array([p // 2 if p % 2 == 0 else far - 1 - p // 2 for p in range(cache.blocks)], np.uint32)
    assert np.any(place[1::2].astype(np.uint64) * page_bytes > 2 ** 32) and far * page_bytes > 2 ** 32
    q_all = cache.randn(220, max(groups) * heads, d).cuda().flatten(1)
    k_all, v_all = (cache.randn(220, heads, d).cuda().flatten(1) for _ in range(2))
    scale, theta, axis = 1 / math.sqrt(d), 1e4, ckv.rope_pair_axes([d // 4, d // 4])
    for count, at_page in ((cache.blocks, np.arange(cache.blocks, dtype=np.uint32)), (far, place)):
        k = torch.empty(count, PAGE, heads * d, dtype=cache.dtype, device="cuda")
        v = torch.empty_like(k)
        pages = torch.from_numpy(at_page.astype(np.int64)).cuda()
        for dev, host in ((k, cache.k), (v, cache.v)):
            dev[pages] = host.view(cache.blocks, PAGE, heads * d).cuda()
        pool = ckv.Pool(ctx, 1, count, PAGE, heads, d, cache.dtype, k.view(-1), v.view(-1))
        tables = [at_page[t] for t in cache.tables]
        flat, starts = np.concatenate(tables), np.cumsum([0] + [t.size for t in tables[:-1]])

        def upload(first, counts):
            s = np.repeat(np.arange(len(counts)), counts)
            pos = np.concatenate([np.arange(f, f + c) for f, c in zip(first, counts)])
            slots = [int(tables[i][p // PAGE]) * PAGE + p % PAGE for i, p in zip(s, pos)]
            pool.upload(flat, starts[s], [tables[i].size for i in s], pos, slots)
            return len(pos)

        outs = []
        for split in (None, "1", "3"):
            if split:
                monkeypatch.setenv("CKV_PREFILL_SPLIT", split)
                monkeypatch.setenv("CKV_PREFILL_SPLIT_MIN", "1")
            n = upload([700, 0, 100], [130, 40, 31])
            for group in groups:
                q = q_all[:n, :group * heads * d].contiguous()
                for window, sinks in ((90, 20), (300, 0), (5000, 0)):
                    out = torch.full_like(q, 5.0)
                    pool.attention_window(0, q, group * heads, scale, window, out, sinks=sinks)
                    outs.append(out)
        monkeypatch.delenv("CKV_PREFILL_SPLIT")
        monkeypatch.delenv("CKV_PREFILL_SPLIT_MIN")
        n = upload([x - 1 for x in lengths], [1] * 3)
        pool.upload_axes(np.stack([np.arange(n), 3 * np.arange(n)]))
        q = q_all[:n, :2 * heads * d].contiguous()
        out, rotated = torch.empty_like(q), torch.empty_like(q)
        pool.append_decode_window(0, k_all[:n], v_all[:n], q, 2 * heads, scale, 77, out, sinks=4)
        pool.rope_axes_append(0, q, rotated, 2 * heads, k_all[n:2 * n], v_all[n:2 * n], theta, axis)
        outs += [out, rotated]
        keep = np.concatenate([np.arange(4), np.arange(400, 830)])
        slot = [int(tables[0][i // PAGE]) * PAGE + i % PAGE for i in range(830)]
        pool.compact(np.take(slot, keep), slot[:keep.size], [keep.size], np.arange(keep.size) - keep, theta)
        ctx.sync()
        got.append([bits(x) for x in outs] + [bits(k[pages]), bits(v[pages])])
        pool.close()
        del k, v, outs
        torch.cuda.empty_cache()
    for i, (small, other) in enumerate(zip(*got)):
        assert torch.equal(small, other), f"output {i}"
    assert torch.all(torch.isfinite(got[0][0].view(cache.dtype).float()))
