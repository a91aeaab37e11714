"""End-to-end decoder around the paged-attention path.

A Qwen2.5-0.5B-shaped causal LM (24 layers, hidden 896, 14 / 2 heads x 64,
SwiGLU 4864, RoPE theta 1e6, vocab 151,936, tied embeddings) with random bf16
weights, run the way the reference's CausalLm runs it
(crates/model/src/causal_lm/model/mod.rs:143-164, decoder block
crates/model/src/components/decoder_block/mod.rs:157-198), but batched: one
StepBatch per engine step, and per layer
    residual add + norm         pa_rms_norm | pa_layer_norm
    Q and K|V projections       two projections over row slices of the fused
      (+ bias)                  QKV weight, so q comes out contiguous
    RoPE + KV write + attention StepBatch.attention (pa_batch_attention)
    O projection
    residual add + norm         pa_rms_norm | pa_layer_norm
    gate|up projection + SwiGLU pa_linear's fused epilogue (small batches) or
                                a GEMM then pa_silu_mul
    down projection
Projections of batches of at most SKINNY_ROWS rows (decode steps, the LM head
over the last tokens) run in pa_linear over weights repacked once at load
time (pa_linear_pack: every MFMA operand fragment one contiguous kilobyte);
larger batches (prefill chunks) run in pa_linear's tiled GEMM over the
row-major weights (gate|up with its SwiGLU epilogue).  With RMSNorm and
weights packed with the norm weights folded in (Weights.pack()), a decode step
runs the fused layer of Engine._forward_fused: five launches per layer (the
QKV projection with RoPE and the KV write in its epilogue, attention, O, gate|up
+ SwiGLU, and the down projection split over K by pa_linear's workspace), the
residual adds in the O and down epilogues.  Decode steps after the first are
one replay each of a captured step that advances the batch by a token on the
device (pa_batch_advance; the block tables hold the whole generation).
With weights quantised by Weights.pack_mx() every step runs the decoder block
in MXFP8 (Engine._forward_mx): half the bytes of the projections' weights, the
matrix cores at their FP8 rate.
The norm is chosen explicitly by ModelConfig.norm: "rms" (RMSNorm, what the
benchmark configuration states) or "layer" (the zero-bias LayerNorm the
reference's CausalLm constructs for these models,
crates/model/src/qwen3/model.rs:19,
crates/model/src/components/decoder_block/factory.rs:42-46).  Norm weights
start at 1, every other weight is N(0, 0.02).
"""
import dataclasses
import math
import time

import torch
import torch.nn.functional as F

from . import ops
from .kv_cache import PagedKvCache, StepBatch


SKINNY_ROWS = 64


@dataclasses.dataclass
class ModelConfig:
    layers: int = 24
    hidden: int = 896
    heads: int = 14
    kv_heads: int = 2
    head_dim: int = 64
    inter: int = 4864
    vocab: int = 151936
    rope_theta: float = 1e6
    eps: float = 1e-6
    norm: str = "rms"  # "rms" | "layer" (zero-bias LayerNorm)


def qwen25_05b():
    return ModelConfig()


class Weights:
    """Random weights of the configuration (bf16 on the device)."""

    def __init__(self, cfg, seed=4, device="cuda", dtype=torch.bfloat16):
        self.cfg = cfg
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) * 0.02).to(dtype)

        h, d = cfg.hidden, cfg.head_dim
        qkv = (cfg.heads + 2 * cfg.kv_heads) * d
        self.embed = w(cfg.vocab, h)
        self.ln1 = [torch.ones(h, dtype=dtype, device=device) for _ in range(cfg.layers)]
        self.ln2 = [torch.ones(h, dtype=dtype, device=device) for _ in range(cfg.layers)]
        self.wqkv = [w(qkv, h) for _ in range(cfg.layers)]
        self.bqkv = [w(qkv) for _ in range(cfg.layers)]
        self.wo = [w(h, cfg.heads * d) for _ in range(cfg.layers)]
        self.wgu = [w(2 * cfg.inter, h) for _ in range(cfg.layers)]
        self.wd = [w(h, cfg.inter) for _ in range(cfg.layers)]
        self.norm = torch.ones(h, dtype=dtype, device=device)
        self.packed = None
        self.mx = None

    def pack(self, fold_rms=True):
        """Repacks the weights pa_linear reads (QKV as separate Q and K|V row
        blocks, O, gate|up, the tied embedding as LM head) into its fragment
        layout; the row-major tensors stay for the tiled GEMM of prompt chunks.  fold_rms:
        fold each RMSNorm weight into the columns of the projection after it
        (ln1 into Q and K|V, ln2 into gate|up, the final norm into the LM head),
        for the engine's fused decode step (pa_linear normalises its input
        rows itself)."""
        def fits(wt):  # shapes pa_linear_pack takes
            return wt.shape[0] % 16 == 0 and wt.shape[1] % 32 == 0

        n = len(self.wqkv)
        nq = self.wo[0].shape[1]
        ln1 = self.ln1 if fold_rms else [None] * n
        ln2 = self.ln2 if fold_rms else [None] * n
        blocks = {"qkv": [(x, g) for x, g in zip(self.wqkv, ln1)],
                  "q": [(x[:nq], g) for x, g in zip(self.wqkv, ln1)],
                  "kv": [(x[nq:], g) for x, g in zip(self.wqkv, ln1)],
                  "o": [(x, None) for x in self.wo],
                  "gu": [(x, g) for x, g in zip(self.wgu, ln2)],
                  "down": [(x, None) for x in self.wd]}
        p = {name: [ops.PackedWeight(x, col_scale=g) for x, g in ws]
             for name, ws in blocks.items() if all(fits(x) for x, _ in ws)}
        if fold_rms and self.cfg.head_dim % 32 == 0 and self.cfg.hidden % 32 == 0:
            # the fused QKV weight for pa_linear_rope_cache (RoPE and the KV
            # write in the projection's epilogue)
            c = self.cfg
            p["qkv_rope"] = [ops.PackedWeight(x, col_scale=g,
                                              rope_heads=(c.heads, c.kv_heads, c.head_dim))
                             for x, g in zip(self.wqkv, ln1)]
        if fits(self.embed):
            p["lm_head"] = ops.PackedWeight(self.embed, col_scale=self.norm if fold_rms else None)
        p["rms_folded"] = fold_rms
        self.packed = p

    def pack_mx(self):
        """Quantises the projections' weights and the tied LM head to MXFP8
        (ops.MxWeight); engines made with these weights then run in MXFP8.  The
        row-major tensors stay (the embedding rows are read from them)."""
        self.mx = {"qkv": [ops.MxWeight(x) for x in self.wqkv],
                   "o": [ops.MxWeight(x) for x in self.wo],
                   "gu": [ops.MxWeight(x) for x in self.wgu],
                   "down": [ops.MxWeight(x) for x in self.wd],
                   "lm_head": ops.MxWeight(self.embed)}

    def nbytes(self):
        """Bytes of the model's weights (row-major; a step reads each once)."""
        ts = [self.embed, self.norm]
        for lst in (self.ln1, self.ln2, self.wqkv, self.bqkv, self.wo, self.wgu, self.wd):
            ts += lst
        return sum(t.numel() * t.element_size() for t in ts)


class Engine:
    """Batched greedy generation over one paged KV cache."""

    def __init__(self, cfg, weights, num_blocks, device="cuda", graph=True):
        """graph: capture one decode step's forward in a HIP graph and replay
        it for the following steps (the batch is re-prepared on the host
        before every replay; see StepBatch.set_capacity)."""
        self.cfg, self.w, self.device = cfg, weights, torch.device(device)
        self.graph = graph
        self.cache = PagedKvCache(cfg.layers, cfg.kv_heads, cfg.head_dim, num_blocks,
                                  torch.bfloat16, device)
        self.batch = StepBatch()
        self.inv_freq = torch.from_numpy(ops.rope_inv_freq(cfg.head_dim, cfg.rope_theta)).to(
            self.device)
        self.free = list(range(num_blocks))
        self.scale = 1.0 / math.sqrt(cfg.head_dim)
        if cfg.norm not in ("rms", "layer"):
            raise ValueError(f"unknown norm {cfg.norm!r}")
        self._norm = ops.rms_norm if cfg.norm == "rms" else ops.layer_norm
        # pa_linear's K split of the down projection (the one long-K
        # projection), sized for every skinny batch; zeroed once here, every
        # call leaves it zeroed
        ws = max(ops.linear_workspace_size(r, cfg.hidden, cfg.inter)
                 for r in range(1, SKINNY_ROWS + 1))
        self.linear_ws = (torch.zeros(ws, dtype=torch.uint8, device=self.device)
                          if ws else None)

    def forward(self, tokens, logit_rows):
        """One step over the prepared batch: tokens [T] (int64, device) ->
        logits of the rows logit_rows [R, vocab] (f32; None: every row, as
        in a decode step)."""
        return self._logits(tokens, logit_rows).float()

    def next_tokens(self, tokens, logit_rows):
        """Greedy next token of each row of logit_rows (int64 [R]): pa_argmax
        over the bf16 logits, argmax_logits's rule."""
        return ops.argmax(self._logits(tokens, logit_rows))

    def _logits(self, tokens, logit_rows):
        """forward's logits in the model dtype (bf16)."""
        c, w = self.cfg, self.w
        if w.mx is not None:
            return self._forward_mx(tokens, logit_rows)
        t = tokens.shape[0]
        hq, hkv, d = c.heads, c.kv_heads, c.head_dim
        skinny = t <= SKINNY_ROWS

        def linear(inp, weight, bias=None, packed=None):
            if skinny and packed is not None:
                return ops.linear(inp, packed, bias)
            return ops.linear(inp.contiguous(), weight, bias)

        pk = w.packed or {}

        def packed(name, layer):
            return pk[name][layer] if name in pk else None

        if (skinny and pk.get("rms_folded") and c.norm == "rms" and
                all(name in pk for name in ("qkv", "o", "gu", "lm_head"))):
            return self._forward_fused(tokens, logit_rows)

        x = F.embedding(tokens, w.embed)          # residual stream [T, hidden]
        h = torch.empty_like(x)
        add = None
        nq = hq * d
        for layer in range(c.layers):
            self._norm(x, w.ln1[layer], c.eps, add=add, out=h)
            wqkv, bqkv = w.wqkv[layer], w.bqkv[layer]
            if skinny and packed("q", layer) is not None:
                q = ops.linear(h, packed("q", layer), bqkv[:nq]).view(t, hq, d)
                kv = ops.linear(h, packed("kv", layer), bqkv[nq:])
                k = kv[:, :hkv * d].view(t, hkv, d)
                v = kv[:, hkv * d:].view(t, hkv, d)
            else:
                # one projection for Q, K and V; attention takes strided
                # views of its rows
                qkv = ops.linear(h, wqkv, bqkv)
                q = qkv[:, :nq].view(t, hq, d)
                k = qkv[:, nq:nq + hkv * d].view(t, hkv, d)
                v = qkv[:, nq + hkv * d:].view(t, hkv, d)
            attn = self.batch.attention(self.cache, layer, q, k, v, self.inv_freq, self.scale)
            o = linear(attn.view(t, nq), w.wo[layer], packed=packed("o", layer))
            self._norm(x, w.ln2[layer], c.eps, add=o, out=h)
            gu = packed("gu", layer) if skinny else None
            act = ops.linear(h, gu if gu is not None else w.wgu[layer], act=ops.ACT_SILU_MUL)
            add = linear(act, w.wd[layer])
        self._norm(x, w.norm, c.eps, add=add, out=h)
        rows = h if logit_rows is None else h[logit_rows]
        lm = pk.get("lm_head") if rows.shape[0] <= SKINNY_ROWS else None
        return ops.linear(rows.contiguous(), lm if lm is not None else w.embed)

    def _forward_fused(self, tokens, logit_rows):
        """Decode-step forward with the RMSNorms folded into the projections:
        per layer the fused QKV projection (normalising its input rows, ln1
        folded into the packed weight) with RoPE and the KV-cache write in
        its epilogue (pa_batch_qkv_rope_cache; without a "qkv_rope" pack, the
        projection, then RoPE + the KV write in the attention call),
        attention reading q as a strided view of its rows, O added into the
        residual stream in place, gate|up + SwiGLU (ln2 folded), down (K
        split over workgroups) added into the residual stream; the final
        norm is folded into the LM head.  Five launches per layer instead of
        nine."""
        c, w, pk = self.cfg, self.w, self.w.packed
        t = tokens.shape[0]
        hq, hkv, d = c.heads, c.kv_heads, c.head_dim
        nq = hq * d
        x = F.embedding(tokens, w.embed)  # residual stream [T, hidden]
        for layer in range(c.layers):
            if "qkv_rope" in pk:
                # one QKV projection with RoPE and the KV write in its
                # epilogue; attention reads q as a strided view of its rows
                qkv = self.batch.qkv_rope_cache(self.cache, layer, x, pk["qkv_rope"][layer],
                                                w.bqkv[layer], self.inv_freq, rms_eps=c.eps)
                q = qkv[:, :nq].view(t, hq, d)
                attn = self.batch.attention(self.cache, layer, q, None, None, None, self.scale)
            else:
                # one QKV projection; q, k, v are strided views of its rows
                qkv = ops.linear(x, pk["qkv"][layer], w.bqkv[layer], rms_eps=c.eps)
                q = qkv[:, :nq].view(t, hq, d)
                k = qkv[:, nq:nq + hkv * d].view(t, hkv, d)
                v = qkv[:, nq + hkv * d:].view(t, hkv, d)
                attn = self.batch.attention(self.cache, layer, q, k, v, self.inv_freq,
                                            self.scale)
            ops.linear(attn.view(t, nq), pk["o"][layer], out=x, add_to_out=True)
            act = ops.linear(x, pk["gu"][layer], act=ops.ACT_SILU_MUL, rms_eps=c.eps)
            if "down" in pk:
                ops.linear(act, pk["down"][layer], out=x, add_to_out=True,
                           workspace=self.linear_ws)
            else:
                ops.linear(act, w.wd[layer], out=x, add_to_out=True)
        rows = x if logit_rows is None else x[logit_rows].contiguous()
        return ops.linear(rows, pk["lm_head"], rms_eps=c.eps)

    def _norm_mx(self, x, weight):
        """The configured norm of the rows of x, as MXFP8 rows."""
        if self.cfg.norm == "rms":
            return ops.rms_norm_mx(x, weight, self.cfg.eps)
        return ops.quantize_mx(ops.layer_norm(x, weight, self.cfg.eps))

    def _forward_mx(self, tokens, logit_rows):
        """_logits with the projections in MXFP8: per layer the norm writes the
        QKV projection's rows, attention's output is quantised for the O
        projection, the gate|up projection's SwiGLU epilogue writes the down
        projection's rows, and O and down add into the residual stream."""
        c, w, mx = self.cfg, self.w, self.w.mx
        t = tokens.shape[0]
        hq, hkv, d = c.heads, c.kv_heads, c.head_dim
        nq = hq * d
        x = F.embedding(tokens, w.embed)  # residual stream [T, hidden]
        for layer in range(c.layers):
            h = self._norm_mx(x, w.ln1[layer])
            qkv = ops.linear_mx(h, mx["qkv"][layer], bias=w.bqkv[layer])
            q = qkv[:, :nq].view(t, hq, d)
            k = qkv[:, nq:nq + hkv * d].view(t, hkv, d)
            v = qkv[:, nq + hkv * d:].view(t, hkv, d)
            attn = self.batch.attention(self.cache, layer, q, k, v, self.inv_freq, self.scale)
            ops.linear_mx(ops.quantize_mx(attn.view(t, nq)), mx["o"][layer], residual=x, out=x)
            h = self._norm_mx(x, w.ln2[layer])
            act = ops.linear_mx(h, mx["gu"][layer], act=ops.ACT_SILU_MUL, mx_out=True)
            ops.linear_mx(act, mx["down"][layer], residual=x, out=x)
        rows = x if logit_rows is None else x[logit_rows].contiguous()
        return ops.linear_mx(self._norm_mx(rows, w.norm), mx["lm_head"])

    def generate(self, prompts, max_new):
        """Greedy generation for every prompt (lists of token ids).  Returns
        (generated ids [B, max_new] on the host, {"prefill_s", "decode_s"})."""
        b = len(prompts)
        lens = [len(p) for p in prompts]
        blocks = []
        for n in lens:
            need = (n + max_new + 15) // 16
            if need > len(self.free):
                raise RuntimeError("KV pool exhausted")
            blocks.append([self.free.pop() for _ in range(need)])
        try:
            torch.cuda.synchronize(self.device)
            t0 = time.perf_counter()
            self.batch.prepare(self.cache, lens, [0] * b, blocks)
            tokens = torch.tensor([x for p in prompts for x in p], dtype=torch.int64,
                                  device=self.device)
            last = torch.tensor([sum(lens[:i + 1]) - 1 for i in range(b)], device=self.device)
            nxt = self.next_tokens(tokens, last)
            out = [nxt]
            torch.cuda.synchronize(self.device)
            t1 = time.perf_counter()
            rows = None  # decode steps: one token per sequence, every row's logits
            self.batch.set_capacity(max(lens) + max_new if self.graph else 0)
            graph = None
            hist = None  # graph path: generated ids [max_new, B], written by the replays
            for step in range(1, max_new):
                if not self.graph or step == 1:
                    # eager (also the warm-up of every launch the graph records)
                    self.batch.prepare(self.cache, [1] * b, [n + step - 1 for n in lens],
                                       blocks)
                    nxt = self.next_tokens(nxt, rows)
                    out.append(nxt)
                    continue
                if graph is None:
                    # The captured step advances the batch by one token on
                    # the device (the tables hold every block of the
                    # generation), feeds its tokens to the next replay and
                    # stores them in row `row` of hist: a replay is the whole
                    # step, with no host work between replays.
                    hist = torch.empty(max_new, b, dtype=torch.int64, device=self.device)
                    hist[:step] = torch.stack(out, 0)
                    row = torch.full((1,), step, dtype=torch.int64, device=self.device)
                    static_tok = nxt.clone()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        self.batch.advance(self.cache)
                        static_out = self.next_tokens(static_tok, rows)
                        static_tok.copy_(static_out)
                        hist.index_copy_(0, row, static_out[None])
                        row.add_(1)
                graph.replay()
            gen = (hist.t() if hist is not None else torch.stack(out, 1)).cpu()
            t2 = time.perf_counter()
        finally:
            self.batch.set_capacity(0)
            for blk in blocks:
                self.free.extend(blk)
        return gen, {"prefill_s": t1 - t0, "decode_s": t2 - t1}
