"""The int8 cache on the GPU: appending against the definition bit for bit, and
attention against a plain implementation in 64 bits with derived tolerances."""
import math

import numpy as np
import pytest
import torch

import int8_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if dtype is None else t.to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def on_device(pa, cache):
    return pa.Int8Cache(*(dev(x) for x in (cache[0], cache[1], cache[2], cache[3])))


def on_host(cache):
    return tuple(x.cpu().numpy() for x in (cache.k, cache.v, cache.k_scales, cache.v_scales))


def rounded(x, dtype):
    """x as the operator gets it: on the device, and its values in f64."""
    t = torch.from_numpy(np.asarray(x, np.float32)).to(dtype)
    return t.to(DEV), t.double().numpy()


def make_tables(rng, counts, nb, width=None):
    perm = rng.permutation(nb)
    out = np.full((len(counts), width or max(max(counts), 1)), 0, np.int32)
    at = 0
    for s, n in enumerate(counts):
        out[s, :n] = perm[at:at + n]
        at += n
    assert at <= nb
    return out


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,d", [(2, 64), (3, 96), (1, 256), (8, 128), (2, 32), (1, 192)])
@pytest.mark.parametrize("new,past", [
    ([1, 1, 1, 1], [0, 15, 16, 40]),          # a decode step
    ([5, 1, 16, 33, 0, 100], [0, 3, 7, 31, 9, 0]),
    ([2, 257], [1030, 15]),
])
def test_append_is_the_definition(pa, dtype, h, d, new, past):
    rng = np.random.default_rng(h * d + len(new))
    ctx = [a + b for a, b in zip(new, past)]
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 3
    tables = make_tables(rng, counts, nb)
    cache = int8_plain.random_cache(rng, nb, h, d)
    total = sum(new)
    # magnitudes from token to token, so that some blocks outgrow their scale
    mag = np.exp2(rng.uniform(-4, 5, (total, 1, 1)))
    key, k64 = rounded(rng.standard_normal((total, h, d)) * mag, dtype)
    value, v64 = rounded(rng.standard_normal((total, h, d)) * mag, dtype)
    cu = np.cumsum([0] + new)
    got = on_device(pa, cache)
    pa.append_int8(got, key, value, i32(tables), i32(cu), i32(ctx), max(new))
    want = int8_plain.append(cache, k64, v64, tables, cu, ctx, max(new))
    for a, b in zip(on_host(got), want):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_token_by_token(pa, dtype):
    """A sequence grown one token at a time, its magnitude drifting up and down:
    every step's codes and scales."""
    rng = np.random.default_rng(5)
    h, d, steps = 2, 64, 50
    tables = make_tables(rng, [4], 6)
    cache = int8_plain.random_cache(rng, 6, h, d)
    got = on_device(pa, cache)
    for t in range(steps):
        mag = 2.0 ** (3 * math.sin(t / 3))
        key, k64 = rounded(rng.standard_normal((1, h, d)) * mag, dtype)
        value, v64 = rounded(rng.standard_normal((1, h, d)) * mag, dtype)
        pa.append_int8(got, key, value, i32(tables), i32([0, 1]), i32([t + 1]), 1)
        cache = int8_plain.append(cache, k64, v64, tables, [0, 1], [t + 1], 1)
        for a, b in zip(on_host(got), cache):
            np.testing.assert_array_equal(a, b)


def test_append_values_at_the_edges(pa):
    """Largest values at and beside 127 * 2^e, subnormal, huge and zero ones,
    ties, infinities and NaN."""
    rng = np.random.default_rng(6)
    h, d = 1, 64
    tops = []
    for e in (-126, -100, -3, 0, 5, 100, 120):
        top = np.float32(127 * 2.0 ** e)
        tops += [top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0))]
    tops += [np.float32(x) for x in (0, 1e-45, 1e-39, 2.0 ** -126, 3.4028235e38, 1, 2, 254, 255)]
    n = len(tops)
    x = np.zeros((n, h, d), np.float32)
    for i, top in enumerate(tops):
        e = int8_plain.scale_exponent(float(top))
        x[i, 0, 0] = -top if i % 2 else top
        with np.errstate(over="ignore", under="ignore"):
            half = np.ldexp(rng.integers(-126, 126, d - 8) + 0.5, e).astype(np.float32)  # ties
        x[i, 0, 1:d - 7] = np.clip(half, -top, top)
        x[i, 0, d - 7:d - 3] = [np.nan, np.inf, -np.inf, -0.0]
    # one token at the start of a block each
    tables = np.arange(n, dtype=np.int32)[:, None]
    cache = int8_plain.random_cache(rng, n, h, d)
    key, k64 = rounded(x, torch.float32)
    value, v64 = rounded(-x, torch.float32)
    got = on_device(pa, cache)
    pa.append_int8(got, key, value, i32(tables), i32(range(n + 1)), i32([1] * n), 1)
    want = int8_plain.append(cache, k64, v64, tables, np.arange(n + 1), [1] * n, 1)
    for a, b in zip(on_host(got), want):
        np.testing.assert_array_equal(a, b)


def test_append_strided_and_unaligned_rows(pa):
    rng = np.random.default_rng(7)
    h, d, n = 2, 64, 37
    for dtype in DTYPES:
        for off, pad in ((0, 0), (1, 3), (2, 2), (4, 4), (64, 8)):
            wide, w64 = rounded(rng.standard_normal(n * (2 * h * d + pad) + off), dtype)
            k = wide[off:].view(n, -1)
            k64 = w64[off:].reshape(n, -1)
            cut = (slice(None), slice(0, h * d)), (slice(None), slice(h * d, 2 * h * d))
            key, value = (k[c].unflatten(1, (h, d)) for c in cut)
            tables = make_tables(rng, [4], 5)
            cache = int8_plain.random_cache(rng, 5, h, d)
            got = on_device(pa, cache)
            pa.append_int8(got, key, value, i32(tables), i32([0, n]), i32([n + 9]), n)
            want = int8_plain.append(cache, *(k64[c].reshape(n, h, d) for c in cut), tables,
                                     [0, n], [n + 9], n)
            for a, b in zip(on_host(got), want):
                np.testing.assert_array_equal(a, b)


def test_append_skips_what_it_cannot_place(pa):
    """Ids outside the pool, positions behind the table, contexts shorter than the
    call's tokens, and rows behind max_tokens: nothing else is touched."""
    rng = np.random.default_rng(8)
    h, d = 2, 64
    new, ctx = [40, 5, 9, 30, 12], [40, 3, 20, 70, 12]
    tables = np.array([[2, -1, 3], [4, 5, 0], [6, 99, 0], [7, 8, 9], [10, 0, 0]], np.int32)
    cache = int8_plain.random_cache(rng, 12, h, d)
    cu = np.cumsum([0] + new)
    key, k64 = rounded(rng.standard_normal((cu[-1], h, d)), torch.bfloat16)
    value, v64 = rounded(rng.standard_normal((cu[-1], h, d)), torch.bfloat16)
    for bound in (40, 10):
        got = on_device(pa, cache)
        pa.append_int8(got, key, value, i32(tables), i32(cu), i32(ctx), bound)
        want = int8_plain.append(cache, k64, v64, tables, cu, ctx, bound)
        for a, b in zip(on_host(got), want):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 96, 256])
def test_append_rotates(pa, dtype, d):
    """q and keys rotated: x1 c - x2 s and x2 c + x1 s with the angle's f32 product,
    sine and cosine within 2^-22, two products and a sum in f32: off by less than
    2^-21 (|x1| + |x2|), then one rounding (bf16 2^-8, f32 none besides; a code
    half a step)."""
    rng = np.random.default_rng(d)
    h, hq = 2, 6
    new, ctx = [1, 20, 3], [100000, 33, 3]
    tables = np.zeros((3, 6250), np.int32)
    tables[0, -1], tables[1, :3], tables[2, 0] = 1, [2, 3, 4], 5
    cache = int8_plain.random_cache(rng, 6, h, d)
    cu = np.cumsum([0] + new)
    t = int(cu[-1])
    pos = np.concatenate([np.arange(c - n, c) for n, c in zip(new, ctx)])
    inv = np.float32(1e4) ** -(np.arange(d // 2, dtype=np.float32) / np.float32(d // 2))
    q, q64 = rounded(rng.standard_normal((t, hq, d)), dtype)
    key, k64 = rounded(rng.standard_normal((t, h, d)), dtype)
    value, v64 = rounded(rng.standard_normal((t, h, d)), dtype)
    ang = (pos.astype(np.float32)[:, None] * inv[None]).astype(np.float64)[:, None]

    def turn(x):
        a, b = x[..., :d // 2], x[..., d // 2:]
        err = 2.0 ** -21 * (np.abs(a) + np.abs(b))
        return (np.concatenate([a * np.cos(ang) - b * np.sin(ang),
                                b * np.cos(ang) + a * np.sin(ang)], -1),
                np.concatenate([err, err], -1))

    got = on_device(pa, cache)
    pa.append_int8(got, key, value, i32(tables), i32(cu), i32(ctx), 20, q=q, inv_freq=dev(inv))
    rq, eq = turn(q64)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    assert np.all(np.abs(q.double().cpu().numpy() - rq) <= eq + half * (np.abs(rq) + eq))
    rk, ek = turn(k64)
    # the definition with the exact rotation: values and, but for the rounding, scales
    k, v, ks, vs = on_host(got)
    _, want_v, _, want_vs = int8_plain.append(cache, k64, v64, tables, cu, ctx, 20)
    np.testing.assert_array_equal(v, want_v)
    np.testing.assert_array_equal(vs, want_vs)
    val = int8_plain.values(k, ks)
    for i in range(t):
        s = int(np.searchsorted(cu, i, "right")) - 1
        blk = tables[s][pos[i] // 16]
        step = np.ldexp(1.0, ks[blk].astype(int) - 127)[:, None]
        assert np.all(np.abs(val[blk, :, pos[i] % 16] - rk[i]) <= 0.5 * step + ek[i])


def test_read_back(pa):
    rng = np.random.default_rng(9)
    for h, d, n in ((2, 64, 37), (3, 48, 1), (1, 128, 160)):
        cache = int8_plain.random_cache(rng, 12, h, d)
        ids = rng.permutation(12)[:-(-n // 16)].astype(np.int32)
        if len(ids) > 1:
            ids[1] = 12  # outside: zeros
        k, v = pa.read_kv_int8(on_device(pa, cache), i32(ids), n)
        kk, vv = int8_plain.values(cache[0], cache[2]), int8_plain.values(cache[1], cache[3])
        for t in range(n):
            b = ids[t // 16]
            wk = kk[b, :, t % 16] if b < 12 else np.zeros((h, d))
            wv = vv[b, :, :, t % 16] if b < 12 else np.zeros((h, d))
            np.testing.assert_array_equal(k[t].cpu().numpy(), wk.astype(np.float32))
            np.testing.assert_array_equal(v[t].cpu().numpy(), wv.astype(np.float32))


def check(got, want, tol):
    got = got.double().cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = np.abs(got - want) > tol
    assert not np.any(bad & ~nan), (np.abs(got - want)[bad].max(), tol[bad].min())


def query(rng, n, hq, d):
    """Queries with some channels larger than the rest."""
    x = rng.standard_normal((n, hq, d)) * np.where(rng.random(d) < 0.05, 12, 1)
    return rounded(x, torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (14, 2, 64), (8, 8, 128), (32, 8, 128),
                                      (6, 2, 96), (20, 1, 32), (34, 2, 192), (7, 1, 256)])
@pytest.mark.parametrize("ctx", [[1], [0, 1, 15, 16, 17, 63, 64, 65], [2051, 129], [255, 0, 700]])
def test_decode(pa, hq, hkv, d, ctx):
    rng = np.random.default_rng(hq * d + len(ctx))
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 2
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    tables = make_tables(rng, counts, nb)
    q, q64 = query(rng, len(ctx), hq, d)
    scale = 1 / math.sqrt(d) / 8  # codes are as large as any: keep the softmax soft
    got = pa.decode_int8(q, on_device(pa, cache), i32(tables), i32(ctx), max(ctx), scale=scale)
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (14, 2, 64), (8, 8, 128), (8, 2, 128),
                                      (6, 2, 96), (9, 1, 32), (3, 1, 192), (7, 1, 256)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([17, 1, 0, 64], [0, 40, 5, 63]),
                                      ([130, 3], [77, 260]), ([65, 16, 15], [0, 0, 1])])
def test_prefill(pa, hq, hkv, d, new, past):
    rng = np.random.default_rng(hq * d + len(new))
    ctx = [a + b for a, b in zip(new, past)]
    counts = [-(-c // 16) for c in ctx]
    nb = sum(counts) + 2
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    tables = make_tables(rng, counts, nb)
    q, q64 = query(rng, sum(new), hq, d)
    scale = 1 / math.sqrt(d) / 8
    got = pa.prefill_int8(q, on_device(pa, cache), i32(tables), i32(np.cumsum([0] + new)),
                          i32(past), max(new), scale=scale)
    rows = [(s, past[s] + i + 1) for s in range(len(new)) for i in range(new[s])]
    want, tol = int8_plain.attention(cache, q64, tables, ctx, rows, scale)
    check(got, want, tol)


def test_attention_masks(pa):
    """Table ids outside the pool contribute nothing (a row of only such gives
    zeros), blocks that are not attended may hold any scale byte, a query row that
    is not finite gives NaN and leaves the others alone."""
    rng = np.random.default_rng(11)
    hq, hkv, d = 6, 2, 64
    nb = 40
    cache = int8_plain.random_cache(rng, nb, hkv, d)
    tables = make_tables(rng, [9, 9, 9], nb - 1)
    cache[2][tables[0, 5:]] = 255  # behind the context
    cache[3][tables[0, 5:]] = 255
    tables[1, :5] = [-1, nb, 1 << 30, -(1 << 31), nb + 7]
    tables[2] = -1
    cache[2][0], cache[3][0] = 255, 255  # what an id outside the pool is replaced by
    tables[tables == 0] = nb - 1
    ctx = [80, 130, 144]
    q, q64 = query(rng, 3, hq, d)
    q[0, 1, 3], q64[0, 1, 3] = float("nan"), np.nan
    q[1, 4, 60], q64[1, 4, 60] = float("inf"), np.inf
    scale = 0.02
    c = on_device(pa, cache)
    got = pa.decode_int8(q, c, i32(tables), i32(ctx), 144, scale=scale)
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(got, want, tol)
    # the same rows as the last of chunks of one token
    got = pa.prefill_int8(q, c, i32(tables), i32([0, 1, 2, 3]), i32([x - 1 for x in ctx]), 1,
                          scale=scale)
    check(got, want, tol)


@pytest.mark.parametrize("scale,spread", [(0.125, 0.0), (3.0, 0.0), (-0.1, 3.0), (0.0, 2.0),
                                          (1e-3, 40.0)])
def test_scales_far_apart(pa, scale, spread):
    """Peaked and flat softmaxes, a negative and a zero softmax scale, blocks whose
    scales are far apart."""
    rng = np.random.default_rng(12)
    hq, hkv, d, ctx = 4, 2, 64, [300, 97]
    cache = int8_plain.random_cache(rng, 30, hkv, d, spread)
    if spread > 8:
        cache[2][:] = 121  # scores that are finite, values of any size
    tables = make_tables(rng, [19, 7], 30)
    q, q64 = query(rng, 2, hq, d)
    got = pa.decode_int8(q, on_device(pa, cache), i32(tables), i32(ctx), 300, scale=scale)
    want, tol = int8_plain.attention(cache, q64, tables, ctx, list(enumerate(ctx)), scale)
    check(got, want, tol)
