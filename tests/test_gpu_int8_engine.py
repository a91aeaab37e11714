"""The int8 cache and the sampler as an engine uses them: one step's operators
together, the batch object, captured steps, streams, and generation."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

import int8_plain
import sample_plain
from test_gpu_int8 import check, i32, make_tables, on_host, rounded

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_step_together(pa):
    """Chunks, then single tokens, appended, attended and, over a vocabulary, drawn:
    each operator on what the ones before it left, against the plain forms."""
    rng = np.random.default_rng(1)
    hq, hkv, d, vocab = 8, 2, 64, 3000
    lens = [45, 16, 3, 130]
    counts = [-(-(n + 3) // 16) for n in lens]
    nb = sum(counts) + 1
    tables = make_tables(rng, counts, nb)
    cache = pa.Int8Cache.empty(nb, hkv, d, DEV)
    plain = on_host(cache)
    head, head64 = rounded(rng.standard_normal((vocab, hq * d)) / 8, torch.bfloat16)
    scale = 1 / math.sqrt(d)
    new, ctx = list(lens), list(lens)
    for step in range(4):
        cu = np.cumsum([0] + new)
        t = int(cu[-1])
        key, k64 = rounded(2 * rng.standard_normal((t, hkv, d)), torch.bfloat16)
        value, v64 = rounded(rng.standard_normal((t, hkv, d)), torch.bfloat16)
        q, q64 = rounded(2 * rng.standard_normal((t, hq, d)), torch.bfloat16)
        pa.append_int8(cache, key, value, i32(tables), i32(cu), i32(ctx), max(new))
        plain = int8_plain.append(plain, k64, v64, tables, cu, ctx, max(new))
        for a, b in zip(on_host(cache), plain):
            np.testing.assert_array_equal(a, b)
        if step == 0:
            out = pa.prefill_int8(q, cache, i32(tables), i32(cu), i32([0] * 4), max(new))
        else:
            out = pa.decode_int8(q, cache, i32(tables), i32(ctx), max(ctx))
        rows = [(s, ctx[s] - new[s] + i + 1) for s in range(4) for i in range(new[s])]
        check(out, *int8_plain.attention(plain, q64, tables, ctx, rows, scale))
        last = out[torch.tensor(cu[1:] - 1, device=DEV)].reshape(4, -1)
        logits = last @ head.t()
        u = rng.random(4).astype(np.float32)
        settings = [(0.8, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.7, 0.05), (1.5, 7, 1.0, 0.0)]
        t_, k_, p_, m_ = (np.array(x) for x in zip(*settings))
        f = torch.float32
        got = pa.sample(logits, torch.tensor(u, device=DEV),
                        temperature=torch.tensor(t_, dtype=f, device=DEV),
                        top_k=i32(k_.tolist()), top_p=torch.tensor(p_, dtype=f, device=DEV),
                        min_p=torch.tensor(m_, dtype=f, device=DEV)).tolist()
        x = logits.double().cpu().numpy()
        want = [sample_plain.draw(x[r], float(u[r]), *(float(np.float32(v)) if i != 1 else v
                                                       for i, v in enumerate(settings[r])))
                for r in range(4)]
        assert got == want
        new, ctx = [1] * 4, [c + 1 for c in ctx]


@pytest.mark.parametrize("rotate", [False, True])
def test_batch_attention_is_the_operators(pa, rotate):
    """StepBatch.attention on an int8 cache: what append_int8 and the attention of
    the step give, bit for bit, for a prompt step, a mixed one and decode steps that
    advance on the device."""
    rng = np.random.default_rng(2)
    layers, hq, hkv, d, nb = 2, 6, 2, 64, 40
    cache = pa.PagedKvCache(layers, hkv, d, nb, torch.int8, DEV)
    mine = pa.Int8Cache.empty(nb, hkv, d, DEV)
    blocks = [list(map(int, x)) for x in np.split(rng.permutation(nb)[:36], 3)]
    tables = np.array(blocks, np.int32)
    inv = torch.from_numpy(pa.rope_inv_freq(d, 1e4)).to(DEV) if rotate else None
    batch = pa.StepBatch()
    ctx = [0, 0, 0]
    for step, new in enumerate([[20, 7, 100], [1, 30, 1], [1, 1, 1], [1, 1, 1], [1, 1, 1]]):
        if step < 4:
            batch.prepare(cache, new, ctx, blocks)
        else:
            batch.advance(cache)
        past, ctx = ctx, [a + b for a, b in zip(ctx, new)]
        t = sum(new)
        # q, k and v as views of one projection
        rows = torch.randn(t, (hq + 2 * hkv) * d, device=DEV).to(torch.bfloat16)
        def views(x):
            return [y.unflatten(1, (-1, d)) for y in x.split([hq * d, hkv * d, hkv * d], 1)]
        q, k, v = views(rows.clone())
        out = batch.attention(cache, 1, q, k, v, inv)
        q2, k2, v2 = views(rows.clone())
        cu = i32(np.cumsum([0] + new))
        pa.append_int8(mine, k2, v2, i32(tables), cu, i32(ctx), max(new),
                       q=q2 if rotate else None, inv_freq=inv)
        got = cache.int8(1)
        for a, b in zip(on_host(got), on_host(mine)):
            np.testing.assert_array_equal(a, b)
        q2 = q2.contiguous()
        if step >= 2:
            want = pa.decode_int8(q2, mine, i32(tables), i32(ctx), max(ctx))
        else:
            want = pa.prefill_int8(q2, mine, i32(tables), cu, i32(past), max(new))
        assert torch.equal(out, want)
    assert not cache.key_cache(0).any() and not cache.int8(0).k_scales.any()
    k, v = cache.read_kv(1, blocks[2], ctx[2])
    wk, wv = pa.read_kv_int8(mine, i32(blocks[2]), ctx[2])
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert cache.block_hashes(1) == {}
    row = torch.zeros(hkv, d, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: cache.write_kv(0, 0, 0, row, row),
                 lambda: cache.write_kv_batch(0, 0, 0, row[None], row[None]),
                 lambda: cache.write_prefill_kv(0, [0], [0], 1, row[None], row[None])):
        with pytest.raises(pa.PaError):
            call()


def test_captured_step_replays(pa):
    """Append, attend and draw in one graph, replayed with eager work between, and
    every replay against the same step eagerly."""
    rng = np.random.default_rng(3)
    b, hq, hkv, d, vocab = 5, 4, 2, 64, 5000
    nb, most = 200, 600
    tables = i32(make_tables(rng, [38] * b, nb))
    start = [590, 3, 65, 15, 300]
    cu = i32(range(b + 1))
    f = torch.float32
    opts = dict(temperature=torch.full((b,), 0.9, device=DEV),
                top_k=i32([0, 50, 5, 0, 1000]),
                top_p=torch.tensor([0.9, 0.95, 1, 0.5, 0.99], dtype=f, device=DEV))
    head = torch.randn(vocab, hq * d, device=DEV).to(torch.bfloat16) / 4
    buf = dict(q=torch.empty(b, hq, d, dtype=torch.bfloat16, device=DEV),
               k=torch.empty(b, hkv, d, dtype=torch.bfloat16, device=DEV),
               v=torch.empty(b, hkv, d, dtype=torch.bfloat16, device=DEV),
               u=torch.empty(b, device=DEV), ctx=i32(start))

    def step(cache):
        pa.append_int8(cache, buf["k"], buf["v"], tables, cu, buf["ctx"], 1)
        out = pa.decode_int8(buf["q"], cache, tables, buf["ctx"], most)
        logits = pa.linear(out.view(b, -1), head)
        return out, pa.sample(logits, buf["u"], **opts)

    caches = [pa.Int8Cache.empty(nb, hkv, d, DEV) for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(0)
    full = [torch.randn(sum(start), hkv, d, device=DEV).to(torch.bfloat16) for _ in range(2)]
    at = i32(np.cumsum([0] + start))
    for c in caches:
        pa.append_int8(c, *full, tables, at, i32(start), max(start))

    def feed(i):
        for name in ("q", "k", "v"):
            buf[name].copy_(torch.randn(buf[name].shape, generator=g, device=DEV))
        buf["u"].copy_(torch.rand(b, generator=g, device=DEV))
        buf["ctx"].copy_(i32([n + i + 1 for n in start]))

    feed(0)
    step(caches[0])
    step(caches[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for i in range(1, 7):
        feed(i)
        graph.replay()
        want = step(caches[1])  # eager, between the replays
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w), i
        for a, w in zip(on_host(caches[0]), on_host(caches[1])):
            np.testing.assert_array_equal(a, w)


def test_two_streams(pa):
    """Steps of two batches on streams of their own give what they give alone."""
    rng = np.random.default_rng(4)
    hq, hkv, d = 8, 1, 128
    jobs = []
    for ctx in ([3000, 10], [700, 1500, 2]):
        counts = [-(-c // 16) for c in ctx]
        tables = i32(make_tables(rng, counts, sum(counts)))
        cache = pa.Int8Cache.empty(sum(counts), hkv, d, DEV)
        rows = [torch.randn(sum(ctx), hkv, d, device=DEV).to(torch.bfloat16) for _ in range(2)]
        q = torch.randn(len(ctx), hq, d, device=DEV).to(torch.bfloat16)
        x = torch.randn(len(ctx), 60000, device=DEV)
        jobs.append((cache, rows, tables, i32(np.cumsum([0] + ctx)), i32(ctx), max(ctx), q, x,
                     torch.rand(len(ctx), device=DEV)))

    def run(job):
        cache, rows, tables, cu, ctx, most, q, x, u = job
        pa.append_int8(cache, *rows, tables, cu, ctx, most)
        p = torch.full((len(u),), 0.9, device=DEV)
        return pa.decode_int8(q, cache, tables, ctx, most), pa.sample(x, u, top_p=p)

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(run(j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.fixture(scope="module")
def small(pa):
    from vllm_lite_amd import e2e
    cfg = e2e.ModelConfig(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=32, inter=512,
                          vocab=1008, rope_theta=1e4)
    return e2e, cfg


@pytest.mark.parametrize("pack", ["", "pack", "pack_mx"])
def test_engine_generates(pa, small, pack):
    """Captured steps give the tokens of eager ones; equal seeds give equal tokens,
    other seeds others; a temperature of 0 and a top-k of 1 are greedy.  (Contexts of
    one 64-token step: no sum's order depends on the launch.)"""
    e2e, cfg = small
    w = e2e.Weights(cfg, seed=3, device=DEV)
    if pack:
        getattr(w, pack)()
    rng = np.random.default_rng(1)
    prompts = [list(rng.integers(0, cfg.vocab, n)) for n in (7, 30, 16, 40)]
    S = e2e.Sampling
    mixed = [S(0.8, 20, 0.9), S(0.0), S(1.0, 0, 0.95, 0.02), S(1.3)]

    def run(graph, **kw):
        return e2e.Engine(cfg, w, 64, DEV, graph=graph, kv_dtype=torch.int8).generate(
            prompts, 12, **kw)[0]

    greedy = run(False)
    assert torch.equal(greedy, run(True))
    assert torch.equal(greedy, run(True, sampling=S(0.0)))
    assert torch.equal(greedy, run(False, sampling=S(2.0, 1), seed=8))
    a = run(False, sampling=mixed, seed=5)
    assert torch.equal(a, run(True, sampling=mixed, seed=5))
    assert torch.equal(a[1], greedy[1])
    assert not torch.equal(a, run(True, sampling=mixed, seed=6))
    with pytest.raises(ValueError):
        run(False, sampling=mixed[:2])


def test_engine_bf16_cache_samples(pa, small):
    e2e, cfg = small
    w = e2e.Weights(cfg, seed=3, device=DEV)
    w.pack()
    prompts = [[1, 2, 3], [5] * 20]
    runs = [e2e.Engine(cfg, w, 64, DEV, graph=g).generate(
        prompts, 9, sampling=e2e.Sampling(0.9, 100), seed=2)[0] for g in (False, True)]
    assert torch.equal(*runs)


def test_engine_logits_near_the_bf16_cache(pa, small):
    """The same engine over an int8 and a bf16 cache.  A code is off by at most half a
    step, a step at most 2^-6 of its block's largest value, which for normal values
    (D = 32, blocks of 512) is about 3.3 of their root mean square: an error of at most
    3.3 * 2^-6 / sqrt(12) = 1.5% of it at the root mean square in K and in V each, the
    scores' errors averaging over a head's dims; with bf16's own roundings beside
    them, two layers' and the head's, logits within 10% (their norm)."""
    e2e, cfg = small
    w = e2e.Weights(cfg, seed=4, device=DEV)
    rng = np.random.default_rng(6)
    seqs = [rng.integers(0, cfg.vocab, n).tolist() for n in (5, 70, 33)]
    blocks = [list(range(10 * i, 10 * i + 10)) for i in range(3)]
    lens = [len(s) for s in seqs]
    tokens = torch.tensor([t for s in seqs for t in s], device=DEV)
    last = torch.tensor(np.cumsum(lens) - 1, device=DEV)
    out = []
    for dtype in (torch.int8, torch.bfloat16):
        eng = e2e.Engine(cfg, w, 64, DEV, kv_dtype=dtype)
        eng.batch.prepare(eng.cache, lens, [0] * 3, blocks)
        out.append([eng.forward(tokens, last)])
        for i in range(3):
            eng.batch.prepare(eng.cache, [1] * 3, [n + i for n in lens], blocks)
            out[-1].append(eng.forward(torch.tensor([3, 4, 5], device=DEV), None))
    for a, b in zip(*out):
        assert ((a - b).norm(dim=1) / b.norm(dim=1)).max().item() < 0.1
        assert F.cosine_similarity(a, b).min().item() > 0.995
