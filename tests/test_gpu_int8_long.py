"""pa_decode_int8 at the largest contexts that it takes (block tables of 2^27 entries),
and a captured step beside shorter ones."""
import numpy as np
import pytest
import torch

import int8_plain
from test_gpu_int8 import check, dev, i32, on_device, query

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MBS = (2 ** 31 - 4096) // 16 - 1  # the widest table


def test_ids_are_read_inside_the_widest_table(pa):
    """Many parts, the last of which begin where the steps that a wavefront looks ahead
    would pass 2^31 tokens; the context is short."""
    rng = np.random.default_rng(1)
    h, d, ctx, scale = 9, 32, 150, 0.02
    cache = int8_plain.random_cache(rng, 12, h, d)
    ids = np.arange(11, 1, -1)[None]
    tables = torch.zeros(1, MBS, dtype=torch.int32, device=DEV)
    tables[0, :10] = dev(ids[0])
    q, q64 = query(rng, 1, h, d)
    got = pa.decode_int8(q, on_device(pa, cache), tables, i32([ctx]), MBS * 16, scale=scale)
    want, tol = int8_plain.attention(cache, q64, ids, [ctx], [(0, ctx)], scale)
    check(got, want, tol)


@pytest.mark.parametrize("ctx", [2 ** 31 - 70000000, 2 ** 31 - 5000])
def test_parts_of_the_longest_contexts_are_merged(pa, ctx):
    """All scores 0 and values 1 or -1, the same at every token: out is the value (the
    sums are of multiples of 1 to 2^24 and, among 32 parts, off by 2^-20)."""
    d = 32
    cache = tuple(np.zeros(s, t) for s, t in (((2, 1, 16, d), np.int8), ((2, 1, d, 16), np.int8),
                                              ((2, 1), np.uint8), ((2, 1), np.uint8)))
    value = np.where(np.arange(d) % 3 == 0, -1, 1)
    cache[1][:] = value[:, None]
    cache[2][:] = cache[3][:] = 127
    tables = torch.ones(1, MBS, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, d, dtype=torch.bfloat16, device=DEV)
    out = pa.decode_int8(q, on_device(pa, cache), tables, i32([ctx]), MBS * 16)
    assert torch.equal(out[0, 0].float(), dev(value.astype(np.float32)))


def test_a_captured_step_keeps_its_workspace(pa):
    """A step captured for a capacity of 5000 tokens, replayed after eager steps of the
    same batch object at shorter capacities (which take more parts each)."""
    rng = np.random.default_rng(5)
    hq, hkv, d, nb, ctx = 32, 8, 128, 320, 4000
    cache = pa.PagedKvCache(1, hkv, d, nb, torch.int8, DEV)
    arrays = cache.int8(0)
    for x, y in zip((arrays.k, arrays.v, arrays.k_scales, arrays.v_scales),
                    int8_plain.random_cache(rng, nb, hkv, d)):
        x.copy_(dev(y))
    blocks = [list(range(nb - 1, 0, -1))]
    batch = pa.StepBatch()
    rows = [torch.randn(1, h, d, device=DEV).to(torch.bfloat16) for h in (hq, hkv, hkv)]

    def step(capacity):
        batch.set_capacity(capacity)
        batch.prepare(cache, [1], [ctx - 1], blocks)
        return batch.attention(cache, 0, *rows, scale=0.01)

    want = step(5000).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.attention(cache, 0, *rows, scale=0.01)
    for capacity in (4096, 4005, 4700):
        # (values up to 8, whose weights either step rounds by 2^-8, and out by 2^-8)
        got = step(capacity)
        torch.testing.assert_close(got.float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -4)
        used = [torch.full((1 << 20,), 7, dtype=torch.int32, device=DEV) for _ in range(8)]
        batch.set_capacity(5000)
        batch.prepare(cache, [1], [ctx - 1], blocks)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all((x == 7).all() for x in used)
