"""The MXFP8 operators together: an MLP of the four, each against 64 bits on
what the one before it wrote; captured and replayed; on another stream; and the
engine in MXFP8 against a forward pass with the same quantisation in f32."""
import math

import pytest
import torch
import torch.nn.functional as F

import mx_plain as plain
from test_gpu_mx import (EPS, gated_reference, gen, hidden_states, near_bf16, norm_reference,
                         product, same_as_definition, weight)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def mlp_weights(pa, g, hidden, inter):
    return weight(pa, g, 2 * inter, hidden), weight(pa, g, hidden, inter)


def mlp(pa, x, add, g, gu, down, total):
    h = pa.rms_norm_mx(x, g, EPS, add=add, residual_out=total)
    act = pa.linear_mx(h, gu, act=pa.ops.ACT_SILU_MUL, mx_out=True)
    return h, act, pa.linear_mx(act, down, residual=total)


@pytest.mark.parametrize("rows,hidden,inter", [(1, 896, 4864), (32, 896, 4864), (33, 300, 544),
                                               (333, 896, 4864), (2100, 640, 1056)])
def test_mlp(pa, rows, hidden, inter):
    gn = gen(rows, hidden, inter)
    x, add = (hidden_states(gn, rows, hidden, torch.bfloat16) for _ in range(2))
    g = (1 + 0.1 * torch.randn(hidden, generator=gn, device=DEV)).to(torch.bfloat16)
    gu, down = mlp_weights(pa, gn, hidden, inter)
    total = torch.empty_like(x)
    h, act, out = mlp(pa, x, add, g, gu, down, total)
    s, y = norm_reference(x, add, g)
    assert torch.equal(total.double(), s)
    same_as_definition(h, y)
    y, err = gated_reference(plain.dequantize(h)[:, :hidden], plain.weight_values(gu), inter)
    plain.assert_rounds(act, y, err)
    y, err = product(plain.dequantize(act)[:, :inter], plain.weight_values(down))
    near_bf16(out, y + s, err + (y.abs() + err + s.abs()) * 2.0 ** -24)
    # attention's output, as it is quantised in front of the O projection
    same_as_definition(pa.quantize_mx(x), x.double())


@pytest.mark.parametrize("rows", [7, 200])
def test_mlp_captured(pa, rows):
    """Replayed on new inputs in the same buffers, with eager work in between:
    every replay equals the eager result."""
    hidden, inter = 640, 1056
    gn = gen(rows)
    g = torch.ones(hidden, device=DEV, dtype=torch.bfloat16)
    gu, down = mlp_weights(pa, gn, hidden, inter)
    x, add = (hidden_states(gn, rows, hidden, torch.bfloat16) for _ in range(2))
    total = torch.empty_like(x)
    mlp(pa, x, add, g, gu, down, total)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, act, out = mlp(pa, x, add, g, gu, down, total)
    for _ in range(4):
        x.copy_(hidden_states(gn, rows, hidden, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        again = torch.empty_like(x)
        h2, act2, out2 = mlp(pa, x, add, g, gu, down, again)
        assert torch.equal(total, again) and torch.equal(out, out2)
        for a, b in ((h, h2), (act, act2)):
            assert torch.equal(a.codes, b.codes)
            assert torch.equal(plain.row_scales(a), plain.row_scales(b))


def test_mlp_on_two_streams(pa):
    """Two runs at once on streams of their own, with the same weights."""
    hidden, inter, rows = 640, 1056, 300
    gn = gen(9)
    g = torch.ones(hidden, device=DEV, dtype=torch.bfloat16)
    gu, down = mlp_weights(pa, gn, hidden, inter)
    xs = [hidden_states(gn, rows, hidden, torch.bfloat16) for _ in range(4)]
    want = [mlp(pa, xs[2 * i], xs[2 * i + 1], g, gu, down, torch.empty_like(xs[0]))[2]
            for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    totals = [torch.empty_like(xs[0]) for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = mlp(pa, xs[2 * i], xs[2 * i + 1], g, gu, down, totals[i])[2]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- the engine ------------------------------------------------------------


def mx(y):
    """f32 rows through MXFP8 and back."""
    v, s = plain.quantize(y.double())
    v = v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    return v[:, :y.shape[1]].float()


def reference_logits(cfg, w, tokens, inv_freq):
    """The last token's logits, f32 but for the MXFP8 operands."""
    hq, hkv, d = cfg.heads, cfg.kv_heads, cfg.head_dim
    f = {k: [plain.weight_values(m).float() for m in v] if isinstance(v, list)
         else plain.weight_values(v).float() for k, v in w.mx.items()}
    x = w.embed.float()[tokens]
    t = len(tokens)
    ang = torch.arange(t, device=DEV, dtype=torch.float32)[:, None] * inv_freq[None]
    cos, sin = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def rope(z):
        z1, z2 = z.chunk(2, -1)
        return torch.cat([z1 * cos - z2 * sin, z2 * cos + z1 * sin], -1)

    def norm(z):  # the norm weights are ones
        if cfg.norm == "layer":
            return F.layer_norm(z, (z.shape[-1],), None, None, cfg.eps)
        return z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + cfg.eps)

    mask = torch.full((t, t), float("-inf"), device=DEV).triu(1)
    for i in range(cfg.layers):
        qkv = mx(norm(x)) @ f["qkv"][i].T + w.bqkv[i].float()
        q = rope(qkv[:, :hq * d].view(t, hq, d)).transpose(0, 1)
        k = rope(qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)).repeat_interleave(hq // hkv, 1)
        v = qkv[:, (hq + hkv) * d:].view(t, hkv, d).repeat_interleave(hq // hkv, 1)
        s = torch.matmul(q.contiguous(), k.permute(1, 2, 0).contiguous()) / math.sqrt(d) + mask
        a = torch.matmul(s.softmax(-1), v.transpose(0, 1).contiguous())
        x = x + mx(a.transpose(0, 1).reshape(t, hq * d)) @ f["o"][i].T
        gu = mx(norm(x)) @ f["gu"][i].T
        x = x + mx(F.silu(gu[:, :cfg.inter]) * gu[:, cfg.inter:]) @ f["down"][i].T
    return mx(norm(x[-1:])) @ f["lm_head"].T


def written_out(pa, eng, tokens, last):
    """The engine's step over its prepared batch, operator by operator."""
    c, w, mx = eng.cfg, eng.w, eng.w.mx
    t, hq, hkv, d = tokens.shape[0], c.heads, c.kv_heads, c.head_dim
    x = w.embed[tokens]

    def norm(z, wt):
        if c.norm == "rms":
            return pa.rms_norm_mx(z, wt, c.eps)
        return pa.quantize_mx(pa.layer_norm(z, wt, c.eps))

    for i in range(c.layers):
        qkv = pa.linear_mx(norm(x, w.ln1[i]), mx["qkv"][i], bias=w.bqkv[i])
        q, k, v = (z.contiguous().view(t, -1, d) for z in qkv.split([hq * d, hkv * d, hkv * d], 1))
        a = eng.batch.attention(eng.cache, i, q, k, v, eng.inv_freq, d ** -0.5)
        x = pa.linear_mx(pa.quantize_mx(a.reshape(t, -1)), mx["o"][i], residual=x)
        act = pa.linear_mx(norm(x, w.ln2[i]), mx["gu"][i], act=pa.ops.ACT_SILU_MUL, mx_out=True)
        x = pa.linear_mx(act, mx["down"][i], residual=x)
    x = x if last is None else x[last]
    return pa.linear_mx(norm(x, w.norm), mx["lm_head"]).float()


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_engine_logits(pa, norm):
    """Prefill and decode logits: those of the operators written out one by one,
    bit for bit, and near the f32 forward pass with the same quantisation.  How
    near: the engine keeps bf16 where the pass keeps f32, so values next to a
    border get other codes, which moves the values behind them, and so on; at
    most until the codes of both are independent roundings.  A rounding to
    E4M3 is off by 2.6e-2 of the values at the root mean square (a step of 2^-4
    to 2^-3 of the value over sqrt(12)), two independent ones differ by sqrt(2)
    times that, and nine of them (four products in each of two layers and the
    head) add up to 3 sqrt(2) 2.6e-2 = 0.11."""
    from vllm_lite_amd import e2e
    cfg = e2e.ModelConfig(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=32, inter=544,
                          vocab=1000, norm=norm)
    w = e2e.Weights(cfg, seed=5, device=DEV)
    w.pack_mx()
    eng = e2e.Engine(cfg, w, num_blocks=64, device=DEV)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 70, 33)]
    blocks = [list(range(10 * i, 10 * i + 10)) for i in range(3)]

    def check(tokens, last):
        logits = eng.forward(tokens, last)
        assert torch.equal(logits, written_out(pa, eng, tokens, last))
        for row, seq in zip(logits, seqs):
            ref = reference_logits(cfg, w, torch.tensor(seq, device=DEV), eng.inv_freq)[0]
            assert ((row - ref).norm() / ref.norm()).item() < 0.11

    lens = [len(s) for s in seqs]
    eng.batch.prepare(eng.cache, lens, [0] * 3, blocks)
    check(torch.tensor([t for s in seqs for t in s], device=DEV),
          torch.tensor([sum(lens[:i + 1]) - 1 for i in range(3)], device=DEV))
    for step in range(2):
        new = torch.randint(0, cfg.vocab, (3,), generator=g).tolist()
        eng.batch.prepare(eng.cache, [1] * 3, [len(s) for s in seqs], blocks)
        seqs = [s + [t] for s, t in zip(seqs, new)]
        check(torch.tensor(new, device=DEV), None)


def test_engine_generates(pa):
    """Captured decode steps give the tokens of eager ones, at the benchmark's
    architecture (fewer layers)."""
    from vllm_lite_amd import e2e
    cfg = e2e.qwen25_05b()
    cfg.layers = 3
    w = e2e.Weights(cfg, seed=6, device=DEV)
    w.pack_mx()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist()
               for n in (3, 64, 17, 100, 33)]
    eager, _ = e2e.Engine(cfg, w, 64, DEV, graph=False).generate(prompts, 12)
    graphed, _ = e2e.Engine(cfg, w, 64, DEV, graph=True).generate(prompts, 12)
    assert torch.equal(eager, graphed)
