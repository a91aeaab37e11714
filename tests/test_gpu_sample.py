"""pa_sample on the GPU: the very tokens of the definition in 64 bits.

The kernel's weights are off by less than 2^-48 of themselves and half a unit of
2^-min(51, 62 - b), b = ceil(log2 cols), so a running sum over n tokens is off by less
than 2^-48 of the total and n 2^-(63 - b) or, for 1024 columns and fewer, n 2^-52;
numpy's by n 2^-53 of it at most, and half of that over runs of equal steps.  Where u or p is
nearer than that (over the total, which is 1 or more) to a border between two
tokens, the tokens on both sides are right."""
import numpy as np
import pytest
import torch

import sample_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(x, dtype):
    return torch.tensor(np.asarray(x), dtype=dtype, device=DEV)


def run(pa, logits, u, t=None, k=None, p=None, m=None):
    f = torch.float32
    return pa.sample(logits, dev(u, f), temperature=None if t is None else dev(t, f),
                     top_k=None if k is None else dev(k, torch.int32),
                     top_p=None if p is None else dev(p, f),
                     min_p=None if m is None else dev(m, f)).cpu().numpy()


def check(pa, logits, u, t=None, k=None, p=None, m=None):
    rows, cols = logits.shape
    got = run(pa, logits, u, t, k, p, m)
    x = logits.double().cpu().numpy()
    bits = max(1, int(np.ceil(np.log2(cols)))) if cols > 1 else 1
    for r in range(rows):
        # the settings as the kernel gets them
        one = [float(np.float32(v[r])) if v is not None else d
               for v, d in ((u, 0.0), (t, 1.0), (p, 1.0), (m, 0.0))]
        kk = int(k[r]) if k is not None else 0
        want = {sample_plain.draw(x[r], one[0], one[1], kk, one[2], one[3])}
        gap, total = sample_plain.margin(x[r], one[0], one[1], kk, one[2], one[3])
        near = 2.0 ** -46 + cols * (2.0 ** -(63 - bits) / total + 2.0 ** -52)
        if gap <= near:
            want |= {sample_plain.draw(x[r], one[0] + a * near, one[1], kk, one[2] + b * near,
                                       one[3]) for a in (-1, 1) for b in (-1, 0, 1)}
        assert got[r] in want, (r, got[r], want, one, kk)


def rows_of(rng, rows, cols, dtype, spread=2.5):
    x = torch.from_numpy((spread * rng.standard_normal((rows, cols))).astype(np.float32))
    return x.to(DEV).to(dtype)


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 17), (64, 1000), (33, 4097),
                                       (7, 32000), (300, 513), (9, 50257), (32, 151936)])
def test_all_settings(pa, dtype, rows, cols):
    rng = np.random.default_rng(rows + cols)
    logits = rows_of(rng, rows, cols, dtype)
    u = rng.random(rows).astype(np.float32)
    t = rng.choice([0.0, 0.2, 0.7, 1.0, 1.5, 4.0], rows)
    k = rng.choice([0, 1, 2, 5, 50, 1000, cols, 2 * cols], rows)
    p = rng.choice([1.0, 0.99, 0.9, 0.5, 0.05], rows)
    m = rng.choice([0.0, 0.01, 0.2], rows)
    check(pa, logits, u, t, k, p, m)
    check(pa, logits, u)
    check(pa, logits, u, t)
    check(pa, logits, u, t, k=k)
    check(pa, logits, u, t, p=p)
    check(pa, logits, u, t, m=m)
    check(pa, logits, u, t, k=k, m=m)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_values(pa, dtype):
    """Ties everywhere: whole rows of one value, a few values, thresholds among
    equal ones, zeros of both signs."""
    rng = np.random.default_rng(2)
    rows, cols = 48, 20011
    x = rng.integers(-3, 4, (rows, cols)).astype(np.float32)
    x[:8] = 1.5
    x[8:16] = np.where(rng.random((8, cols)) < 0.5, 0.0, -0.0)
    x[16:24, ::7] = 9.0
    logits = torch.from_numpy(x).to(DEV).to(dtype)
    u = rng.random(rows).astype(np.float32)
    k = rng.choice([0, 3, 100, 5000, 19000], rows)
    p = rng.choice([1.0, 0.97, 0.31], rows)
    check(pa, logits, u, np.full(rows, 0.83), k, p)


def test_many_values_beside_an_outlier(pa):
    """All but one of the values in one interval: their threshold is found by reading
    the row again."""
    rng = np.random.default_rng(3)
    rows, cols = 12, 70001
    x = (1e-3 * rng.standard_normal((rows, cols))).astype(np.float32)
    x[:, 17] = 60.0
    x[6:, 17] = 4.0
    logits = torch.from_numpy(x).to(DEV)
    u = rng.random(rows).astype(np.float32)
    t = np.array([20.0, 30.0] * 6)
    k = np.array([0, 30000, 60000, 2, 9000, 0] * 2)
    p = np.array([0.9, 1.0, 0.8, 0.99, 0.4, 0.7] * 2)
    check(pa, logits, u, t, k, p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_special_values(pa, dtype):
    """Rows with most values masked by -inf or the type's lowest value, NaN, +inf, no
    value at all."""
    rng = np.random.default_rng(4)
    rows, cols = 40, 9001
    x = (2 * rng.standard_normal((rows, cols))).astype(np.float32)
    low = float(torch.finfo(dtype).min)
    hit = rng.random((rows, cols)) < 0.97
    x[:10][hit[:10]] = -np.inf
    x[10:20][hit[10:20]] = low
    x[20:25][hit[20:25]] = np.nan
    x[25, :] = -np.inf
    x[26, :] = np.nan
    x[27, :] = low
    x[28, 5:8] = np.inf
    x[29, :] = np.inf
    x[30, :] = -np.inf
    x[30, 77] = -3.0
    x[31, 12] = np.float32(low) * -1
    logits = torch.from_numpy(x).to(DEV).to(dtype)
    u = rng.random(rows).astype(np.float32)
    t = rng.choice([0.0, 0.5, 1.0, 2.0], rows)
    t[25:33] = [1, 1, 1, 0.5, 1, 1, 1, 0]
    k = rng.choice([0, 0, 3, 40, 700], rows)
    p = rng.choice([1.0, 0.9, 0.3], rows)
    m = rng.choice([0.0, 0.1], rows)
    check(pa, logits, u, t, k, p, m)
    assert run(pa, logits, u, t, k, p, m)[25] == 0 == run(pa, logits, u, t, k, p, m)[26]


def test_settings_at_their_ends(pa):
    """Temperatures from tiny to infinite, p and m outside their ranges, u at 0, 1,
    outside and NaN."""
    rng = np.random.default_rng(5)
    cols = 3001
    x = rows_of(rng, 1, cols, torch.float32)
    h = x.double().cpu().numpy()[0]
    ts = [1e-30, 1e-3, 3e38, float("inf"), -1.0, float("nan"), 1e-45]
    got = run(pa, x.repeat(len(ts), 1), [0.37] * len(ts), ts)
    want = [sample_plain.draw(h, float(np.float32(0.37)), float(np.float32(t))) for t in ts]
    assert list(got) == want
    ps = [0.0, -1.0, 1e-40, 1.0, 2.0, float("nan")]
    got = run(pa, x.repeat(len(ps), 1), [0.73] * len(ps), p=ps)
    top, free = int(np.argmax(h)), sample_plain.draw(h, float(np.float32(0.73)))
    assert list(got) == [top] * 3 + [free] * 3
    ms = [1.0, 5.0, float("inf"), -1.0, float("nan")]
    got = run(pa, x.repeat(len(ms), 1), [0.73] * len(ms), m=ms)
    assert list(got) == [top] * 3 + [free] * 2
    us = [0.0, -1.0, float("nan"), 1.0, 7.0, float("inf")]
    order, _ = sample_plain.kept(h, 1.0, 20, 1.0, 0.0)
    got = run(pa, x.repeat(len(us), 1), us, k=[20] * len(us))
    assert list(got) == [order[0]] * 3 + [order[-1]] * 3
    ks = [-5, cols, 1 << 30, -(1 << 31)]
    got = run(pa, x.repeat(len(ks), 1), [0.73] * len(ks), k=ks)
    assert list(got) == [free] * 4


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(pa, dtype):
    rng = np.random.default_rng(6)
    for cols, pad, off in ((1000, 0, 1), (1001, 7, 3), (5003, 1, 0), (31, 2, 5), (4096, 8, 8)):
        rows = 9
        flat = rows_of(rng, 1, rows * (cols + pad) + off, dtype)[0]
        flat[:off] = 1e4  # what is not a row's is not drawn
        logits = flat[off:].view(rows, cols + pad)
        logits[:, cols:] = 1e4
        check(pa, logits[:, :cols], rng.random(rows).astype(np.float32), np.full(rows, 0.9),
              rng.choice([0, 7, 300], rows), rng.choice([1.0, 0.8], rows))


def test_frequencies(pa):
    """Tokens of evenly spaced u come as often as their probabilities say."""
    x = torch.log(torch.tensor([[0.5, 0.125, 0.25, 0.125]], device=DEV))
    n = 4096
    u = (np.arange(n) + 0.5) / n
    got = run(pa, x.repeat(n, 1), u)
    # the logits are off by 2^-24, the borders by a few of that: less than one u
    assert list(np.bincount(got, minlength=4)) == [2048, 512, 1024, 512]
    assert np.all(np.diff(got) >= 0)  # in the order of the columns
    got = run(pa, x.repeat(n, 1), u, k=[2] * n)
    assert list(np.bincount(got, minlength=4)) == [2731, 0, 1365, 0]


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_launch_and_four_agree(pa, dtype):
    """Many rows take their steps in one launch, few long ones in four: the same
    tokens."""
    rng = np.random.default_rng(7)
    rows, cols = 600, 12007
    x = (2.5 * rng.standard_normal((rows, cols))).astype(np.float32)
    x[:60] = rng.integers(-3, 4, (60, cols))
    x[60:80] = 1.5
    x[80:120][rng.random((40, cols)) < 0.97] = -np.inf
    x[120:140, 5] = 60.0
    x[140:160][rng.random((20, cols)) < 0.5] = np.nan
    logits = torch.from_numpy(x).to(DEV).to(dtype)
    s = (rng.random(rows).astype(np.float32), rng.choice([0.0, 0.3, 1.0, 20.0], rows),
         rng.choice([0, 1, 40, 9000], rows), rng.choice([1.0, 0.9, 0.4], rows),
         rng.choice([0.0, 0.05], rows))
    got = run(pa, logits, *s)
    few = [run(pa, logits[i:i + 100], *(v[i:i + 100] for v in s)) for i in range(0, rows, 100)]
    np.testing.assert_array_equal(got, np.concatenate(few))


@pytest.mark.parametrize("cols", [8191, 8192, 8193])
def test_short_rows_at_the_limit(pa, cols):
    """Ties, masks, an outlier over values in one interval and odd strides, in rows
    that take one launch and just not."""
    rng = np.random.default_rng(cols)
    rows = 24
    x = (2.5 * rng.standard_normal((rows, cols))).astype(np.float32)
    x[:6] = rng.integers(-3, 4, (6, cols))
    x[6:10] = 1e-3 * x[6:10]
    x[6:10, 3] = 60.0
    x[10:14][rng.random((4, cols)) < 0.99] = -np.inf
    x[14] = np.nan
    x[15, 8:10] = np.inf
    flat = torch.full((rows * (cols + 3) + 1,), 1e4, device=DEV)
    logits = flat[1:].view(rows, cols + 3)[:, :cols]
    logits.copy_(torch.from_numpy(x))
    u = rng.random(rows).astype(np.float32)
    t = np.where(np.arange(rows) // 2 == 3, 30.0, rng.choice([0.4, 1.0], rows))
    check(pa, logits, u, t, rng.choice([0, 3, 50, 5000], rows), rng.choice([1.0, 0.8], rows),
          rng.choice([0.0, 0.02], rows))
    check(pa, logits, u, t)
    # settings at their ends
    h = x[20].astype(np.float64)
    one = logits[20:21].expand(7, cols)
    ts = [1e-30, 1e-3, 3e38, float("inf"), -1.0, float("nan"), 1e-45]
    want = [sample_plain.draw(h, float(np.float32(0.37)), float(np.float32(v))) for v in ts]
    assert list(run(pa, one, [0.37] * 7, ts)) == want
    top, free = int(np.argmax(h)), sample_plain.draw(h, float(np.float32(0.73)))
    ps = [0.0, -1.0, 1e-40, 1.0, 2.0, float("nan"), 1.5]
    assert list(run(pa, one, [0.73] * 7, p=ps)) == [top] * 3 + [free] * 4


def test_graphs_share_a_workspace(pa):
    """Two captured draws, long rows and short ones, with one workspace, replayed in
    turn over changing logits and numbers beside eager calls."""
    rng = np.random.default_rng(8)
    rows = 5
    ws = torch.empty(pa.sample_workspace_size(rows), dtype=torch.uint8, device=DEV)
    bufs, graphs = [], []
    for cols in (30011, 700):
        x, u = rows_of(rng, rows, cols, torch.bfloat16), dev(rng.random(rows), torch.float32)
        opts = dict(temperature=dev([0.8] * rows, torch.float32),
                    top_k=dev([0, 50, 3, 0, 999], torch.int32),
                    top_p=dev([0.9, 0.9, 1.0, 1.0, 0.3], torch.float32))
        pa.sample(x, u, workspace=ws, **opts)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pa.sample(x, u, workspace=ws, **opts)
        bufs.append((x, u, opts))
        graphs.append((g, out))
    for _ in range(4):
        for (x, u, opts), (g, out) in zip(bufs, graphs):
            x.copy_(rows_of(rng, *x.shape, x.dtype))
            u.copy_(dev(rng.random(rows), torch.float32))
            g.replay()
            want = pa.sample(x, u, **opts)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
