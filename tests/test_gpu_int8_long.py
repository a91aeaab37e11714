"""pa_decode_int8 at the largest contexts that it takes: block tables of 2^27 entries."""
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
