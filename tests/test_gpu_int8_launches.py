"""The int8 cache's attention in every form that a launch may take: rows a workgroup,
parts, wavefronts, many sequences, a pool behind 4 GiB, scales near the ends."""
import math

import numpy as np
import pytest
import torch

import int8_plain
from test_gpu_int8 import check, dev, i32, make_tables, on_device, query

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def setup(rng, ctx, hq, hkv, d, total):
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 2
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    return cache, make_tables(rng, counts, nb), *query(rng, total, hq, d)


# 256 rows a workgroup: many tiles; 128: enough for the CUs; (64: the short chunks that
# are tested elsewhere).  head_dim 192 and 256 have one form.
@pytest.mark.parametrize("new,past", [([2001, 1, 3001, 990], [0, 77, 0, 1030]), ([1999], [50])])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 32), (32, 8, 64), (24, 8, 96), (32, 8, 128),
                                      (16, 8, 192), (16, 8, 256)])
def test_prefill_of_many_rows(pa, hq, hkv, d, new, past):
    rng = np.random.default_rng(d + len(new))
    ctx = [a + b for a, b in zip(new, past)]
    cache, tables, q, q64 = setup(rng, ctx, hq, hkv, d, sum(new))
    scale = 1 / math.sqrt(d) / 8
    cu = np.cumsum([0] + new)
    got = pa.prefill_int8(q, on_device(pa, cache), i32(tables), i32(cu), i32(past), max(new),
                          scale=scale)
    assert torch.isfinite(got).all()
    # the first and last rows of every sequence and some between
    pick = sorted({int(i) for s in range(len(new))
                   for i in (cu[s], cu[s + 1] - 1, *rng.integers(cu[s], cu[s + 1], 3))})
    seq = np.searchsorted(cu, pick, "right") - 1
    rows = [(int(s), past[s] + i - int(cu[s]) + 1) for s, i in zip(seq, pick)]
    want, tol = int8_plain.attention(cache, q64[pick], tables, ctx, rows, scale)
    check(got[torch.tensor(pick, device=DEV)], want, tol)


@pytest.mark.parametrize("hq,hkv,d,n", [(4, 2, 64, 300), (4, 1, 128, 257), (2, 1, 256, 140)])
def test_prefill_of_many_sequences(pa, hq, hkv, d, n):
    """More of them than a launch orders by length."""
    rng = np.random.default_rng(n)
    new = [int(x) for x in rng.integers(0, 40, n)]
    past = [int(x) for x in rng.integers(0, 60, n)]
    ctx = [a + b for a, b in zip(new, past)]
    cache, tables, q, q64 = setup(rng, ctx, hq, hkv, d, sum(new))
    scale = 1 / math.sqrt(d) / 8
    got = pa.prefill_int8(q, on_device(pa, cache), i32(tables), i32(np.cumsum([0] + new)),
                          i32(past), max(new), scale=scale)
    rows = [(s, past[s] + i + 1) for s in range(n) for i in range(new[s])]
    pick = np.arange(0, len(rows), 7)
    want, tol = int8_plain.attention(cache, q64[pick], tables, ctx, [rows[i] for i in pick], scale)
    check(got[torch.from_numpy(pick).to(DEV)], want, tol)


# one part and several, each with 8 wavefronts and with 4
@pytest.mark.parametrize("hq,hkv,d,ctx", [
    (4, 2, 64, [700, 3]), (8, 8, 128, [640, 0, 1, 639] * 10), (8, 4, 64, [100, 9000, 17] * 4),
    (4, 2, 96, [700, 31]), (8, 4, 128, [9000, 64, 1] * 4), (4, 2, 192, [5000, 300]),
    (8, 4, 256, [2000, 5] * 2), (8, 4, 32, [300, 31] * 40), (2, 2, 192, [600]),
])
def test_decode_parts(pa, hq, hkv, d, ctx):
    rng = np.random.default_rng(hq * d + len(ctx))
    cache, tables, q, q64 = setup(rng, ctx, hq, hkv, d, len(ctx))
    scale = 1 / math.sqrt(d) / 8
    got = pa.decode_int8(q, on_device(pa, cache), i32(tables), i32(ctx), max(ctx), scale=scale)
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(got, want, tol)


def test_a_pool_behind_4_gib(pa):
    """Blocks whose offsets pass 32 bits: appended to, read back and attended."""
    rng = np.random.default_rng(3)
    hq, hkv, d = 16, 8, 256
    nb = 140000  # 4.6 GB of codes each
    cache = pa.Int8Cache.empty(nb, hkv, d, DEV)
    far = np.arange(nb - 40, nb)
    tables = np.stack([rng.permutation(far[:20]), rng.permutation(far[20:])]).astype(np.int32)
    n = [300, 37]
    rows = [torch.from_numpy(rng.standard_normal((sum(n), hkv, d)).astype(np.float32)).to(DEV)
            for _ in range(2)]
    pa.append_int8(cache, *rows, i32(tables), i32([0, 300, 337]), i32(n), 300)
    # the same in a small pool
    small = pa.Int8Cache.empty(40, hkv, d, DEV)
    pa.append_int8(small, *rows, i32(tables - (nb - 40)), i32([0, 300, 337]), i32(n), 300)
    for a, b in ((cache.k, small.k), (cache.v, small.v), (cache.k_scales, small.k_scales),
                 (cache.v_scales, small.v_scales)):
        assert torch.equal(a[nb - 40:], b)
    assert not cache.k_scales[:nb - 40].any()
    for a, b in zip(pa.read_kv_int8(cache, i32(tables[0, :19]), 300),
                    pa.read_kv_int8(small, i32(tables[0, :19] - (nb - 40)), 300)):
        assert torch.equal(a, b) and a.abs().max() > 1
    q, _ = query(rng, 2, hq, d)
    out = [pa.decode_int8(q, c, i32(t), i32(n), 300)
           for c, t in ((cache, tables), (small, tables - (nb - 40)))]
    assert torch.equal(*out)
    q, _ = query(rng, 337, hq, d)
    out = [pa.prefill_int8(q, c, i32(t), i32([0, 300, 337]), i32([0, 0]), 300)
           for c, t in ((cache, tables), (small, tables - (nb - 40)))]
    assert torch.equal(*out)


@pytest.mark.parametrize("byte", [16, 60, 200, 240])
def test_values_of_any_size(pa, byte):
    """V's scales near the ends of what the header promises."""
    rng = np.random.default_rng(byte)
    hq, hkv, d, ctx = 4, 2, 64, [300, 97]
    cache = int8_plain.random_cache(rng, 30, hkv, d)
    cache[3][:] = byte + rng.integers(-3 if byte > 127 else 0, 1 if byte > 127 else 4,
                                      cache[3].shape)
    tables = make_tables(rng, [19, 7], 30)
    q, q64 = query(rng, 2, hq, d)
    c, scale = on_device(pa, cache), 0.02
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(pa.decode_int8(q, c, i32(tables), i32(ctx), 300, scale=scale), want, tol)
    check(pa.prefill_int8(q, c, i32(tables), i32([0, 1, 2]), i32([299, 96]), 1, scale=scale),
          want, tol)


def test_one_workspace_for_two_graphs(pa):
    """Two captured decodes that share a workspace, replayed in turn with other
    queries and contexts in their buffers, beside eager calls."""
    rng = np.random.default_rng(8)
    hq, hkv, d, ctx = 8, 2, 128, [3000, 1200]
    cache, tables, q0, _ = setup(rng, ctx, hq, hkv, d, 2)
    c, tab = on_device(pa, cache), i32(tables)
    need = pa.decode_int8_workspace_size(2, hq, hkv, d, 3000)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    q, lens, graphs = [q0.clone(), q0.clone()], [i32(ctx), i32(ctx)], []
    for i in range(2):
        pa.decode_int8(q[i], c, tab, lens[i], 3000, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pa.decode_int8(q[i], c, tab, lens[i], 3000, workspace=ws)
        graphs.append((g, out))
    for step in range(4):
        for i in range(2):
            new, _ = query(rng, 2, hq, d)
            n = i32([int(x) for x in rng.integers(1, 3001, 1)] + [1200 - step])
            q[i].copy_(new)
            lens[i].copy_(n)
            graphs[i][0].replay()
            want = pa.decode_int8(new, c, tab, n, 3000)
            torch.cuda.synchronize()
            assert torch.equal(graphs[i][1], want)
