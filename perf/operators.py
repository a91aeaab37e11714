"""A decoder block's projections in MXFP8 (E4M3 codes, one power-of-two scale per
32 columns): quantising rows, RMSNorm with the residual's addition and an MXFP8
output, the product of MXFP8 rows with MXFP8 weights (bias or residual in the
epilogue, bf16 out; SwiGLU in the epilogue, MXFP8 out), and an MLP that chains
the three.  Sizes are those of bench.py's configurations (layers of 896 / 4864
with 14 / 2 heads x 64; 4096 wide with 32 / 8 heads x 128) and generic ones.

Layout of MXFP8 rows [rows, cols]: codes [rows, Kp], Kp = cols rounded up to
128 (zeros behind cols); scales [Kp / 128][R][4] bytes, 2^(byte - 127), R = rows
rounded up to 16.  Of weights: fragments of 16 rows x 128 columns, see pack().

A case is a dict of plain values; `kind` names the operator.
"""
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
EPS = 1e-6
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
own = False


def package():
    """The vllm-lite_amd directory as the package vllm_lite_amd."""
    if "vllm_lite_amd" not in sys.modules:
        where = os.path.join(ROOT, "vllm-lite_amd")
        spec = importlib.util.spec_from_file_location(
            "vllm_lite_amd", os.path.join(where, "__init__.py"),
            submodule_search_locations=[where])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["vllm_lite_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["vllm_lite_amd"]


def listed():
    return [
        # The attention output of a decode step of 32 requests, before the O
        # projection: the smallest call, all latency.
        dict(name="quantize_decode", kind="quantize", dtype="bf16", rows=32, cols=896, pad=0),
        # The same of a large prompt batch.
        dict(name="quantize_prompt", kind="quantize", dtype="bf16", rows=7569, cols=4096, pad=0),
        # The norm in front of a decode step's QKV or gate|up projection.
        dict(name="norm_decode", kind="norm", dtype="bf16", rows=32, cols=896, add=True),
        # ... of a large prompt batch.
        dict(name="norm_prompt", kind="norm", dtype="bf16", rows=7569, cols=4096, add=True),
        # f32 rows of a width off every vector, the first norm of a model (no addition).
        dict(name="norm_f32_odd", kind="norm", dtype="f32", rows=617, cols=2050, add=False),
        # The QKV projection of a decode step of 32 requests (18 heads x 64, with bias).
        dict(name="qkv_decode", kind="linear", rows=32, n=1152, k=896, epi="bias"),
        # The down projection of a decode step of a wide layer, added to the residual.
        dict(name="down_decode", kind="linear", rows=17, n=4096, k=12288, epi="residual"),
        # The QKV projection of a mixed step (48 heads x 128, with bias).
        dict(name="qkv_mixed", kind="linear", rows=618, n=6144, k=4096, epi="bias"),
        # The O projection of a large prompt batch, added to the residual.
        dict(name="o_prompt", kind="linear", rows=7569, n=4096, k=4096, epi="residual"),
        # gate|up of a decode step.
        dict(name="swiglu_decode", kind="swiglu", rows=32, n=4864, k=896),
        # gate|up of four 512-token chunks of a wide layer: the largest.
        dict(name="swiglu_prompt", kind="swiglu", rows=2048, n=12288, k=4096),
        # The MLP over one request's prompt: norm, gate|up, down, one after another.
        dict(name="mlp_prompt", kind="mlp", rows=333, cols=896, inter=4864),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "linear", "linear", "swiglu", "mlp"])
    if kind in ("quantize", "norm"):
        cols = _log_int(rng, 33, 12288)
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f32"]), cols=cols,
                    rows=_log_int(rng, 1, min(8192, 33554432 // cols)))
        if kind == "quantize":
            # rows of a wider buffer, as the columns of a fused projection's output
            case["pad"] = rng.choice([0, 0, rng.randint(1, 999)])
        else:
            case["add"] = rng.random() < 0.7
        return case
    most = 10 ** 11  # products of one call
    if kind == "linear":
        n, k = _log_int(rng, 5, 16384), _log_int(rng, 32, 12288)
        return dict(kind=kind, n=n, k=k, rows=_log_int(rng, 1, min(8192, most // (n * k))),
                    epi=rng.choice(["none", "bias", "residual"]))
    if kind == "swiglu":
        n, k = 32 * _log_int(rng, 1, 384), _log_int(rng, 32, 8192)
        return dict(kind=kind, n=n, k=k, rows=_log_int(rng, 1, min(8192, most // (2 * n * k))))
    cols, inter = rng.choice([(896, 4864), (_log_int(rng, 64, 4096), 32 * _log_int(rng, 4, 300))])
    return dict(kind=kind, cols=cols, inter=inter,
                rows=_log_int(rng, 1, min(4096, most // (3 * cols * inter))))


def _up(n, m):
    return -(-n // m) * m


# ---- plain forms -----------------------------------------------------------


def quantize(y):
    """f32 rows [rows, cols] -> codes [rows, Kp] (E4M3), scale bytes [rows, Kp / 32]."""
    rows, cols = y.shape
    y = torch.nn.functional.pad(y, (0, _up(cols, 128) - cols)).view(rows, -1, 32)
    mag = y.abs()
    mag = torch.where(torch.isfinite(mag), mag, 0.0)
    # amax = m 2^x, 0.5 <= m < 1, and 448 = 0.875 2^9
    m, x = torch.frexp(mag.amax(-1))
    e = torch.where(m == 0, -127, x - 9 + (m > 0.875).to(x.dtype)).clamp(min=-127)
    t = torch.ldexp(y, -e[..., None])
    t = torch.where(torch.isfinite(t), t, torch.nan)
    return t.to(E4M3).view(rows, -1), (e + 127).to(torch.uint8)


def by_column(scales):
    """Scale bytes [rows, Kp / 32] -> [Kp / 128, rows, 4], the rows' order in memory."""
    rows = scales.shape[0]
    return scales.view(rows, -1, 4).permute(1, 0, 2).contiguous()


def values(codes, scales):
    """E4M3 codes [rows, Kp] and scale bytes [rows, Kp / 32] -> f32 values."""
    s = torch.ldexp(torch.ones((), device=codes.device), scales.to(torch.int32) - 127)
    return (codes.float().view(*scales.shape, 32) * s[..., None]).view(codes.shape)


def pack(codes, scales):
    """Codes [Np, Kp] and scale bytes [Np, Kp / 32] of a weight -> fragments
    [Np / 16, Kp / 128][8 chunks of 16 columns][16 rows][16 bytes] and their
    scales [Np / 16, Kp / 128][16 rows][4 blocks]."""
    np_, kp = codes.shape
    c = codes.view(torch.uint8).view(np_ // 16, 16, kp // 128, 8, 16)
    s = scales.view(np_ // 16, 16, kp // 128, 4)
    return c.permute(0, 2, 3, 1, 4).contiguous(), s.permute(0, 2, 1, 3).contiguous()


def mx_out(y):
    codes, scales = quantize(y)
    return codes, by_column(scales).view(E8M0)


def rows_values(s, x="x"):
    """The values of MXFP8 rows as prepare() holds them."""
    scales = s[x + "_scales"][:, :s["rows"]].permute(1, 0, 2).reshape(s["rows"], -1)
    return values(s[x].view(E4M3), scales)


def plain_norm(s):
    total = s["x"]
    if s["add"] is not None:
        total = (total.float() + s["add"].float()).to(total.dtype)
    t = total.float()
    return total, t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * s["g"].float()


def plain_linear(x, w, n):
    return x @ values(w["codes"].view(E4M3), w["scales"])[:n].t()


def plain_swiglu(x, w, n):
    gu = plain_linear(x, w, 2 * n)
    return gu[:, :n] * torch.sigmoid(gu[:, :n]) * gu[:, n:]


def plain(s):
    kind, n = s["kind"], s.get("n")
    if kind == "quantize":
        return mx_out(s["x"].float())
    if kind == "norm":
        total, y = plain_norm(s)
        codes, scales = mx_out(y)
        return (codes, scales, total) if s["add"] is not None else (codes, scales)
    if kind == "swiglu":
        return mx_out(plain_swiglu(rows_values(s), s["w"], n))
    if kind == "linear":
        y = plain_linear(rows_values(s), s["w"], n)
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(torch.bfloat16)
    total, y = plain_norm(s)
    act = plain_swiglu(values(*quantize(y)), s["gu"], s["inter"])
    y = plain_linear(values(*quantize(act)), s["down"], s["cols"])
    return total, (y + total.float()).to(torch.bfloat16)


# ---- the framework's calls -------------------------------------------------


def whole(mx):
    return mx.codes.view(E4M3), mx.scales[:, :mx.rows].view(E8M0)


def weight(pa, w):
    return pa.MxWeight.from_packed(w["packed"], w["packed_scales"], w["rows"], w["cols"])


def framework(s):
    pa, kind = package(), s["kind"]
    if kind == "quantize":
        return whole(pa.quantize_mx(s["x"]))
    if kind in ("norm", "mlp"):
        total = torch.empty_like(s["x"]) if s["add"] is not None else None
        h = pa.rms_norm_mx(s["x"], s["g"], EPS, add=s["add"], residual_out=total)
        if kind == "norm":
            return (*whole(h), total) if total is not None else whole(h)
        act = pa.linear_mx(h, weight(pa, s["gu"]), act=pa.ops.ACT_SILU_MUL, mx_out=True)
        return total, pa.linear_mx(act, weight(pa, s["down"]), residual=total)
    x = pa.MxRows(s["x"], s["x_scales"], s["rows"], s["k"])
    if kind == "swiglu":
        return whole(pa.linear_mx(x, weight(pa, s["w"]), act=pa.ops.ACT_SILU_MUL, mx_out=True))
    return pa.linear_mx(x, weight(pa, s["w"]), bias=s["bias"], residual=s["residual"])


# ---- inputs ----------------------------------------------------------------


def _activations(g, rows, cols, dtype):
    """Hidden states: normal values, a few channels an order of magnitude larger."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= 1 + 15 * (torch.rand(cols, generator=g, device=DEV) < 0.01)
    return x.to(dtype)


def _mx_rows(y):
    codes, scales = quantize(y)
    scales = torch.nn.functional.pad(by_column(scales), (0, 0, 0, -y.shape[0] % 16))
    return codes.view(torch.uint8), scales.contiguous()


def _weight(g, rows, cols):
    """A weight as the engine keeps it (fragments), and in rows for the plain form."""
    w = torch.randn(rows, cols, generator=g, device=DEV) / math.sqrt(cols)
    codes, scales = quantize(torch.nn.functional.pad(w, (0, 0, 0, -rows % 16)))
    packed, packed_scales = pack(codes, scales)
    return dict(codes=codes.view(torch.uint8), scales=scales, packed=packed.view(-1),
                packed_scales=packed_scales.view(-1), rows=rows, cols=cols)


def _vector(g, n, dtype, mean=0.0):
    return (mean + 0.1 * torch.randn(n, generator=g, device=DEV)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s, kind, rows = dict(case), case["kind"], case["rows"]
    dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[case.get("dtype", "bf16")]
    if kind == "quantize":
        s["x"] = _activations(g, rows, case["cols"] + case["pad"], dtype)[:, :case["cols"]]
    elif kind in ("norm", "mlp"):
        s["x"] = _activations(g, rows, case["cols"], dtype)
        s["add"] = (_activations(g, rows, case["cols"], dtype) if case.get("add", True) else None)
        s["g"] = _vector(g, case["cols"], dtype, 1.0)
        if kind == "mlp":
            s["gu"] = _weight(g, 2 * case["inter"], case["cols"])
            s["down"] = _weight(g, case["cols"], case["inter"])
    else:
        s["x"], s["x_scales"] = _mx_rows(_activations(g, rows, case["k"], torch.float32))
        s["w"] = _weight(g, case["n"] * (2 if kind == "swiglu" else 1), case["k"])
        if kind == "linear":
            n, bf16 = case["n"], torch.bfloat16
            s["bias"] = _vector(g, n, bf16) if case["epi"] == "bias" else None
            s["residual"] = (_activations(g, rows, n, bf16) if case["epi"] == "residual"
                             else None)
    return s


def run(state):
    if own:
        return framework(state)
    return plain(state)


def work(case):
    rows, kind = case["rows"], case["kind"]
    size = 2 if case.get("dtype", "bf16") == "bf16" else 4
    mx = 33 / 32  # bytes a value: the code and its share of a scale
    if kind == "quantize":
        return {"bytes": rows * case["cols"] * (size + mx), "flops": 0}

    def norm(cols, add):
        return rows * cols * (size * (3 if add else 1) + mx) + cols * size

    if kind == "norm":
        return {"bytes": norm(case["cols"], case["add"]), "flops": 5 * rows * case["cols"]}
    if kind == "linear":
        n, k = case["n"], case["k"]
        more = {"none": 0, "bias": 2 * n, "residual": 2 * rows * n}[case["epi"]]
        return {"bytes": (rows + n) * k * mx + 2 * rows * n + more, "flops": 2 * rows * n * k}
    if kind == "swiglu":
        n, k = case["n"], case["k"]
        return {"bytes": (rows + 2 * n) * k * mx + rows * n * mx, "flops": 4 * rows * n * k}
    cols, inter = case["cols"], case["inter"]
    # x, add, their sum and the output, and the weights
    return {"bytes": 2 * 4 * rows * cols + 3 * inter * cols * mx, "flops": 6 * rows * cols * inter}


# ---- the definition in 64 bits ---------------------------------------------


def _table():
    """The 256 values of E4M3."""
    v = []
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = math.nan if b & 127 == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v.append(-x if b & 128 else x)
    return torch.tensor(v, dtype=torch.float64, device=DEV)


def _exact_mx(y, rounded=True):
    """Values over their scale (rounded to codes, or as they are) and scales of
    f64 rows, the rows padded to 128 columns."""
    rows, cols = y.shape
    wide = torch.zeros(rows, _up(cols, 128), dtype=torch.float64, device=y.device)
    wide[:, :cols] = y
    t = wide.reshape(rows, -1, 32)
    top = torch.nan_to_num(t, 0.0, 0.0, 0.0).abs().amax(-1)
    scale = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-127))
    scale = torch.where(top > 448 * scale, 2 * scale, scale)
    scale = torch.where((top <= 224 * scale) & (scale > 2.0 ** -127), scale / 2, scale)
    t = t / scale[..., None]
    if not rounded:
        return t.reshape(rows, -1), scale
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    step = torch.where(t.abs() >= 16 * step, 2 * step, step)
    step = torch.where((t.abs() < 8 * step) & (step > 2.0 ** -9), step / 2, step)
    codes = (t / step).round() * step
    return codes.reshape(rows, -1), scale


def _exact_out(y, rounded=True):
    codes, scale = _exact_mx(y, rounded)
    return codes, scale.reshape(len(y), -1, 4).transpose(0, 1)


def _exact_values(codes, scale_bytes):
    c = _table()[codes.view(torch.uint8).long()]
    s = torch.exp2(scale_bytes.double() - 127)
    return (c.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _exact_rows(s):
    b = s["x_scales"][:, :s["rows"]].transpose(0, 1).flatten(1)
    return _exact_values(s["x"], b)


def _exact_norm(s):
    t = s["x"].double()
    if s["add"] is not None:
        t = (t + s["add"].double()).to(s["x"].dtype).double()
    r = (t.pow(2).sum(1) / t.shape[1] + EPS).sqrt()
    return t, t / r[:, None] * s["g"].double()


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_out(s["x"].double())
    if kind == "norm":
        t, y = _exact_norm(s)
        return (*_exact_out(y), t) if case["add"] else _exact_out(y)

    def product(x, w, n):
        return torch.matmul(x, _exact_values(w["codes"], w["scales"])[:n].T)

    def swiglu(x, w, n):
        g, u = product(x, w, 2 * n).split(n, dim=1)
        return g / (1 + torch.exp(-g)) * u

    if kind == "swiglu":
        # as a bf16 result: before the rounding to the output's bits
        return _exact_out(swiglu(_exact_rows(s), s["w"], case["n"]), rounded=False)
    if kind == "linear":
        y = product(_exact_rows(s), s["w"], case["n"])
        for more in (s["bias"], s["residual"]):
            y = y if more is None else y + more.double()
        return y
    t, y = _exact_norm(s)

    def as_mx(v):
        codes, scale = _exact_mx(v)
        return (codes.unflatten(1, (-1, 32)) * scale[..., None]).flatten(1)

    act = swiglu(as_mx(y), s["gu"], case["inter"])
    return t, product(as_mx(act), s["down"], case["cols"]) + t
