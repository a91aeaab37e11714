"""Plain forms of the int8 cache's operators, in 64 bits on the host (numpy)."""
import math

import numpy as np

BLOCK = 16


def scale_exponent(amax):
    """The least integer e >= -126 with amax <= 127 * 2^e."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax / 127)[1] - 1)  # amax / 127 = m 2^x, 0.5 <= m < 1
        while amax > 127 * 2.0 ** e:
            e += 1
    return e


def encode(x, e):
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.clip(np.rint(np.ldexp(np.where(np.isnan(x), 0, x), -e)), -127, 127)
    return y.astype(np.int8)


def append(cache, key, value, tables, cu, ctx, max_tokens):
    """pa_append_int8's definition on numpy arrays (k, v, k_scales, v_scales),
    returned changed."""
    k, v, ks, vs = (x.copy() for x in cache)
    nb = k.shape[0]
    for s in range(len(ctx)):
        n = int(cu[s + 1] - cu[s])
        start = int(ctx[s]) - n
        n = min(n, max_tokens)
        if n <= 0 or start < 0:
            continue
        for b in range(start // BLOCK, (start + n - 1) // BLOCK + 1):
            blk = int(tables[s][b]) if b < len(tables[s]) else -1
            if not 0 <= blk < nb:
                continue
            first, last = max(start - b * BLOCK, 0), min(start + n - b * BLOCK, BLOCK)
            rows = slice(int(cu[s]) + b * BLOCK + first - start,
                         int(cu[s]) + b * BLOCK + last - start)
            for x, codes, scales, minor in ((key, k, ks, False), (value, v, vs, True)):
                for h in range(k.shape[1]):
                    y = x[rows, h].astype(np.float64)
                    finite = np.abs(y[np.isfinite(y)])
                    e = scale_exponent(float(finite.max()) if finite.size else 0.0)
                    c = codes[blk, h].T if minor else codes[blk, h]
                    if first > 0:
                        old = int(scales[blk, h]) - 127
                        e = max(e, old)
                        c[:first] = np.rint(np.ldexp(c[:first].astype(np.float64), old - e))
                    c[first:last] = encode(y, e)
                    scales[blk, h] = e + 127
    return k, v, ks, vs


def values(codes, scales):
    """f64 values of codes [NB, H, ...] and scale bytes [NB, H]."""
    return np.ldexp(codes.astype(np.float64), scales.astype(np.int64)[:, :, None, None] - 127)


def random_cache(rng, nb, h, d, spread=2.0):
    """A filled cache whose blocks' magnitudes differ by factors of up to
    2^(2 * spread), each with one code at least of 64 and more, as a written one."""
    k = rng.integers(-127, 128, (nb, h, BLOCK, d)).astype(np.int8)
    v = rng.integers(-127, 128, (nb, h, d, BLOCK)).astype(np.int8)
    e = [np.rint(rng.uniform(-spread, spread, (nb, h))).astype(int) for _ in range(2)]
    return k, v, (e[0] + 121).astype(np.uint8), (e[1] + 121).astype(np.uint8)


def attention(cache, q, tables, lens, rows, scale):
    """Attention of query rows q [R, Hq, D] (f64 of what the operator gets):
    rows[r] = (sequence, keys attended).  Returns the exact output and how far an
    output may be from it:
      - q rounded by d = 2^-14 of its row's largest: a score moves by at most
        eps = scale * d * sum |k|, a probability by a factor within e^(+-2 eps), an
        output by (e^(2 eps) - 1) * 2 max |v|;
      - a score's f32 product and its exponential: 2^-21 of its size besides;
      - a probability times the V scale in bf16: 2^-8 of it, so 2^-8 A of an
        output, A = sum p |v| / sum p;
      - f32 sums over n keys: (n + 64) 2^-24 A;
      - the output in bf16: 2^-8 of it."""
    k_all, v_all = values(cache[0], cache[2]), values(cache[1], cache[3])
    nb, hkv, _, d = k_all.shape
    hq = q.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for r, (s, n) in enumerate(rows):
        n = min(n, len(tables[s]) * BLOCK)
        keys = [(int(tables[s][t // BLOCK]), t % BLOCK) for t in range(n)]
        keys = [(b, t) for b, t in keys if 0 <= b < nb]
        if not keys:
            continue
        blk, off = (np.array(x) for x in zip(*keys))
        for h in range(hq):
            kv = h // (hq // hkv)
            k, v = k_all[blk, kv, off], v_all[blk, kv, :, off]
            if not np.all(np.isfinite(q[r, h])):
                out[r, h] = np.nan
                continue
            x = k @ q[r, h] * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[r, h] = p @ v
            a = p @ np.abs(v)
            eps = abs(scale) * 2.0 ** -14 * np.abs(q[r, h]).max() * np.abs(k).sum(1).max()
            eps += 2.0 ** -21 * (np.abs(x).max() * 1.4427 + 1)
            tol[r, h] = (math.expm1(2 * eps) * 2 * np.abs(v).max() + 2.0 ** -8 * a +
                         (n + 64) * 2.0 ** -24 * a + 2.0 ** -8 * np.abs(out[r, h]) + 1e-37)
    return out, tol
