"""The int8 cache's attention where scales, queries and sizes are at their ends."""
import math

import numpy as np
import pytest
import torch

import int8_plain
from test_gpu_int8 import check, dev, i32, make_tables, on_device, on_host, query, rounded

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# the forms of a prefill launch: 64 rows a workgroup (few rows), 128, 256
@pytest.mark.parametrize("hq,hkv,d,new,past", [
    (4, 2, 32, [70, 9], [31, 0]), (4, 2, 64, [70, 9], [31, 0]), (6, 2, 96, [70, 9], [31, 0]),
    (4, 2, 128, [70, 9], [31, 0]), (2, 2, 192, [70, 9], [31, 0]), (2, 1, 256, [70, 9], [31, 0]),
    (32, 8, 64, [1999], [50]), (32, 8, 128, [1999], [50]), (32, 8, 128, [2001, 3001], [0, 40]),
])
def test_values_of_zero_and_tiny_ones_beside_others(pa, hq, hkv, d, new, past):
    """Blocks whose V is all zero (their scale byte is 1), tiny, of normal size and
    large, as pa_append_int8 writes them, in every mixture: a block's values do not
    change its keys' part in the denominator."""
    rng = np.random.default_rng(d + len(new))
    ctx = [a + b for a, b in zip(new, past)]
    counts = [-(-c // 16) for c in ctx]
    nb, total = sum(counts) + 2, sum(ctx)
    tables = make_tables(rng, counts, nb)
    cache = tuple(np.zeros_like(x) for x in int8_plain.random_cache(rng, nb, hkv, d))
    size = rng.choice([0.0, 2.0 ** -90, 2.0 ** -40, 2.0 ** -24, 1.0, 4.0], (total // 16 + 2, hkv, 1))
    size[0], size[1] = 0.0, 2.0 ** -90
    key = rng.standard_normal((total, hkv, d)).astype(np.float32)
    value = (1 + 0.1 * rng.standard_normal((total, hkv, d))).astype(np.float32)
    cu = np.cumsum([0] + ctx)
    at = 0
    for s, n in enumerate(ctx):
        for t in range(0, n, 16):
            value[cu[s] + t:min(cu[s] + t + 16, cu[s + 1])] *= size[at % len(size)]
            at += 1
    c = on_device(pa, cache)
    pa.append_int8(c, dev(key), dev(value), i32(tables), i32(cu), i32(ctx), max(ctx))
    cache = on_host(c)
    assert (cache[3] == 1).any() and ((cache[3] > 1) & (cache[3] < 40)).any()
    q, q64 = rounded(rng.standard_normal((sum(new), hq, d)), torch.bfloat16)
    scale = 1 / math.sqrt(d)
    got = pa.prefill_int8(q, c, i32(tables), i32(np.cumsum([0] + new)), i32(past), max(new),
                          scale=scale)
    rows = [(s, past[s] + i + 1) for s in range(len(new)) for i in range(new[s])]
    pick = np.arange(len(rows)) if len(rows) < 100 else rng.permutation(len(rows))[:12]
    want, tol = int8_plain.attention(cache, q64[pick], tables, ctx, [rows[i] for i in pick], scale)
    check(got[torch.from_numpy(pick).to(DEV)], want, tol)
    got = pa.decode_int8(q[:len(ctx)], c, i32(tables), i32(ctx), max(ctx), scale=scale)
    want, tol = int8_plain.attention(cache, q64[:len(ctx)], tables, ctx, list(enumerate(ctx)),
                                     scale)
    check(got, want, tol)
