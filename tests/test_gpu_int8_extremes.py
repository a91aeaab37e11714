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
    size = rng.choice([0.0, 2.0 ** -90, 2.0 ** -40, 2.0 ** -24, 1.0, 4.0],
                      (total // 16 + 2, hkv, 1))
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


@pytest.mark.parametrize("d", [64, 128, 256])
def test_scale_byte_0_reads_as_scale_0(pa, d):
    """V blocks of any codes under byte 0, beside others: their values are zeros, their
    keys are in the denominator."""
    rng = np.random.default_rng(d)
    hq, hkv, ctx = 4, 2, [200, 97, 40]
    cache = int8_plain.random_cache(rng, 30, hkv, d)
    zero = rng.random((30, hkv)) < 0.4
    tables = make_tables(rng, [13, 7, 3], 30)
    zero[tables[2, :3]] = True  # a sequence with no other
    cache[3][zero] = 0
    plain = (cache[0], np.where(zero[:, :, None, None], 0, cache[1]), cache[2], cache[3])
    q, q64 = query(rng, 3, hq, d)
    c, scale = on_device(pa, cache), 0.25 / math.sqrt(d)
    want, tol = int8_plain.attention(plain, q64, tables, ctx, list(enumerate(ctx)), scale)
    assert not want[2].any()
    check(pa.decode_int8(q, c, i32(tables), i32(ctx), 200, scale=scale), want, tol)
    check(pa.prefill_int8(q, c, i32(tables), i32([0, 1, 2, 3]), i32([x - 1 for x in ctx]), 1,
                          scale=scale), want, tol)


@pytest.mark.parametrize("byte", [1, 2, 94, 95, 96, 127, 249, 252, 253, 254])
@pytest.mark.parametrize("d", [32, 128, 256])
def test_every_value_scale_alone(pa, byte, d):
    """One key, so out is its value, in both kernels: powers of two to the first and
    the last scale."""
    rng = np.random.default_rng(byte)
    cache = int8_plain.random_cache(rng, 3, 2, d)
    cache[1][:] = rng.integers(-1, 2, cache[1].shape)
    cache[3][:] = byte
    q, _ = query(rng, 2, 4, d)
    c, tables = on_device(pa, cache), i32([[2], [1]])
    want = torch.stack([pa.read_kv_int8(c, i32([b]), 1)[1][0] for b in (2, 1)])
    want = want.repeat_interleave(2, 1)
    assert torch.equal(want.abs().amax((1, 2)), torch.full((2,), 2.0 ** (byte - 127), device=DEV))
    got = pa.prefill_int8(q, c, tables, i32([0, 1, 2]), i32([0, 0]), 1, scale=0.01)
    assert torch.equal(got.float(), want)
    assert torch.equal(pa.decode_int8(q, c, tables, i32([1, 1]), 1, scale=0.01).float(), want)


def test_masked_blocks_of_the_largest_values(pa):
    """An id outside the pool is replaced by block 0, here of the largest codes and
    scale: nothing of it shows."""
    rng = np.random.default_rng(3)
    hq, hkv, d, ctx = 4, 2, 64, [100, 33]
    cache = int8_plain.random_cache(rng, 12, hkv, d)
    cache[1][0], cache[3][0] = 127, 254
    tables = np.array([[1, -1, 2, 99, 3, 4, -5], [5, -1, 6, 0, 0, 0, 0]], np.int32)
    q, q64 = query(rng, 2, hq, d)
    c, scale = on_device(pa, cache), 0.02
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(pa.decode_int8(q, c, i32(tables), i32(ctx), 100, scale=scale), want, tol)
    check(pa.prefill_int8(q, c, i32(tables), i32([0, 1, 2]), i32([99, 32]), 1, scale=scale),
          want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 32), (4, 2, 64), (6, 2, 96), (4, 1, 128),
                                      (2, 1, 192), (2, 1, 256)])
@pytest.mark.parametrize("scale", [0.02, -0.02])
def test_infinite_queries_against_codes_of_one_sign(pa, hq, hkv, d, scale):
    """Rows with an infinity, whose scores may all be -inf: NaN, as pa.h says, and the
    rows beside them their values; zeros for one without keys."""
    rng = np.random.default_rng(d)
    new, past = [3, 40, 1, 70], [0, 0, 20, 33]
    ctx = [a + b for a, b in zip(new, past)]
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 1
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    tables = make_tables(rng, counts, nb)
    for s, sign in enumerate((1, -1, 1, -1)):  # dim 5 has codes of one sign
        for b in tables[s, :counts[s]]:
            cache[0][b, :, :, 5] = sign * (1 + np.abs(cache[0][b, :, :, 5] // 2))
    tables[2] = -1  # no keys
    q, q64 = query(rng, sum(new), hq, d)
    hit = rng.random(sum(new)) < 0.5
    hit[[0, 2, 3, 43]] = True
    for r in np.flatnonzero(hit):
        q[r, r % hq, 5] = q64[r, r % hq, 5] = math.inf if r % 3 else -math.inf
        if r % hq:
            q[r, 0, 5] = q64[r, 0, 5] = -q64[r, r % hq, 5]
    c = on_device(pa, cache)
    rows = [(s, past[s] + i + 1) for s in range(len(new)) for i in range(new[s])]
    want, tol = int8_plain.attention(cache, q64, tables, ctx, rows, scale)
    assert np.isnan(want).any() and not want[43].any()
    check(pa.prefill_int8(q, c, i32(tables), i32(np.cumsum([0] + new)), i32(past), max(new),
                          scale=scale), want, tol)
    last = np.cumsum(new) - 1
    check(pa.decode_int8(q[torch.from_numpy(last).to(DEV)], c, i32(tables), i32(ctx), max(ctx),
                         scale=scale), want[last], tol[last])


def test_key_scale_byte_0_reads_as_scale_0(pa):
    """Under byte 0 of K every score is 0, however large the query."""
    rng = np.random.default_rng(4)
    hq, hkv, d, ctx = 4, 2, 64, [100, 20]
    cache = int8_plain.random_cache(rng, 12, hkv, d)
    cache[2][:] = 0
    plain = (np.zeros_like(cache[0]), *cache[1:])
    tables = make_tables(rng, [7, 2], 12)
    q, q64 = query(rng, 2, hq, d)
    c, scale = on_device(pa, cache), 1.0
    want, tol = int8_plain.attention(plain, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(pa.decode_int8(q * 2.0 ** 118, c, i32(tables), i32(ctx), 100, scale=scale), want, tol)
    # (prefill's sums of q times codes are f32)
    check(pa.prefill_int8(q * 2.0 ** 100, c, i32(tables), i32([0, 1, 2]), i32([99, 19]), 1,
                          scale=scale), want, tol)


@pytest.mark.parametrize("power", [-126, -100, -60, 0, 60, 110])
def test_queries_and_key_scales_of_opposite_sizes(pa, power):
    """Queries of 2^power, keys of 70 * 2^-power: the scores are of normal size."""
    rng = np.random.default_rng(power + 200)
    hq, hkv, d, ctx = 4, 2, 64, [300, 97]
    cache = int8_plain.random_cache(rng, 30, hkv, d, 1.0)
    cache[2][:] = cache[2].astype(int) + 6 - power
    tables = make_tables(rng, [19, 7], 30)
    q = torch.from_numpy(rng.standard_normal((2, hq, d)) * 2.0 ** power).to(torch.bfloat16)
    c, scale = on_device(pa, cache), 1.2e-3
    want, tol = int8_plain.attention(cache, q.double().numpy(), tables, ctx,
                                     list(enumerate(ctx)), scale)
    check(pa.decode_int8(q.to(DEV), c, i32(tables), i32(ctx), 300, scale=scale), want, tol)


@pytest.mark.parametrize("sign", [1, -1])
def test_decode_rounds_a_query_to_2_to_the_minus_14_of_its_largest(pa, sign):
    """The largest with all its bits set and 63 values of 2^-13 of its power of two:
    rounded by 2^-14 of the largest each at most (here not at all), their products with
    two keys of 127 and -127 (and 0 for the largest) differ by 4: tanh(2) of the values
    1 and -1, off by the rounding of probabilities and out, 2^-8 each."""
    h = 2.0 ** -13
    q = torch.full((1, 1, 64), h, dtype=torch.bfloat16, device=DEV)
    q[0, 0, 0] = sign * (2 - 2.0 ** -7)
    cache = tuple(np.zeros(s, t) for s, t in (((1, 1, 16, 64), np.int8), ((1, 1, 64, 16), np.int8),
                                              ((1, 1), np.uint8), ((1, 1), np.uint8)))
    cache[0][0, 0, 0, 1:], cache[0][0, 0, 1, 1:] = 127, -127
    cache[1][0, 0, :, 0], cache[1][0, 0, :, 1] = 64, -64
    cache[2][:], cache[3][:] = 127, 121
    out = pa.decode_int8(q, on_device(pa, cache), i32([[0]]), i32([2]), 2,
                         scale=2 / (63 * 127 * h)).float()
    assert (out - math.tanh(2)).abs().max() <= 2.0 ** -7


@pytest.mark.parametrize("scale,spread", [(0.125, 0.0), (3.0, 0.0), (-0.1, 3.0), (0.0, 2.0),
                                          (1e-3, 40.0)])
def test_prefill_of_scales_far_apart(pa, scale, spread):
    """Peaked and flat softmaxes, a negative and a zero softmax scale, blocks whose
    scales are far apart, in chunks."""
    rng = np.random.default_rng(12)
    hq, hkv, d, new, past = 4, 2, 64, [70, 33], [230, 0]
    cache = int8_plain.random_cache(rng, 30, hkv, d, spread)
    if spread > 8:
        cache[2][:] = 121  # scores that are finite, values of any size
    tables = make_tables(rng, [19, 3], 30)
    q, q64 = query(rng, 103, hq, d)
    got = pa.prefill_int8(q, on_device(pa, cache), i32(tables), i32([0, 70, 103]), i32(past), 70,
                          scale=scale)
    rows = [(s, past[s] + i + 1) for s in range(2) for i in range(new[s])]
    want, tol = int8_plain.attention(cache, q64, tables, [300, 33], rows, scale)
    check(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d,ctx", [(4, 2, 64, [40, 300, 7]), (32, 8, 128, [1500, 3]),
                                          (2, 1, 256, [100, 17])])
def test_scores_below_the_floats(pa, hq, hkv, d, ctx):
    """A finite query against keys so large that all of a row's scores are below f32's
    range: NaN, not the 0 of a row without keys; where some key's score is a float, its
    value."""
    rng = np.random.default_rng(d)
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 1
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    cache[0][:] = -1 - np.abs(cache[0] // 2)
    cache[2][:] = 200
    tables = make_tables(rng, counts, nb)
    # the second sequence's first block: scores that are floats, the largest token 1's, 0
    cache[0][tables[1, 0], :, 1], cache[2][tables[1, 0]] = 0, 100
    tables[0, 0] = -1
    c = on_device(pa, cache)
    q = torch.full((len(ctx), hq, d), 2.0 ** 70, dtype=torch.bfloat16, device=DEV)
    want = np.full(q.shape, np.nan)
    v = int8_plain.values(cache[1], cache[3])[tables[1, 0], :, :, 1]
    want[1] = np.repeat(v, hq // hkv, 0)
    tol = 2.0 ** -7 * np.abs(want)
    check(pa.decode_int8(q, c, i32(tables), i32(ctx), max(ctx), scale=1.0), want, tol)
    check(pa.prefill_int8(q, c, i32(tables), i32(range(len(ctx) + 1)), i32([n - 1 for n in ctx]),
                          1, scale=1.0), want, tol)
    none = torch.full_like(i32(tables), -1)
    assert not pa.decode_int8(q, c, none, i32(ctx), max(ctx), scale=1.0).any()
