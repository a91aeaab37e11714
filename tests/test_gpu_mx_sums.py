"""The sums of every kernel of pa_linear_mx to the last bit: exact integers, in
every epilogue; and what random values are off by."""
import pytest
import torch

import mx_plain as plain
from mx_sums import cancel, gate_scale, integers, silu_ends, totals
from test_gpu_mx import DEV, KERNELS, KERNELS_GATED, gen, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epi", ["none", "bias", "residual", "both"])
@pytest.mark.parametrize("m,n,k", list(KERNELS) + [(5, 40, 4865), (64, 70, 4000), (300, 99, 4999)])
def test_exact_sums(pa, m, n, k, epi):
    g = gen(m, n, k, epi)
    x, w = integers(g, m, n, k, DEV, same_rows=epi == "bias")
    t = totals(x, w)
    bias = res = None
    if epi == "bias":
        bias = cancel(t[0])
    if epi == "both":
        bias = torch.randint(-99, 100, (n,), generator=g, device=DEV).to(torch.bfloat16)
    more = t if bias is None else t + bias.double()
    if epi in ("residual", "both"):
        res = cancel(more)
        more = more + res.double()
    out = pa.linear_mx(pa.quantize_mx(x), pa.MxWeight(w), bias=bias, residual=res)
    assert torch.equal(out, more.to(torch.bfloat16))


def round_at(y, scales):
    """E4M3 values of y at scale bytes [rows, Kp / 32]."""
    wide = torch.nn.functional.pad(y, (0, 32 * scales.shape[1] - y.shape[1]))
    t = wide * torch.exp2(127 - scales.double()).repeat_interleave(32, 1)
    _, e = torch.frexp(t)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return (t / step).round() * step


def between(mx, lo, hi):
    """Codes and scales of rows between lo and hi, which round alike or to
    neighbours."""
    got, scales = plain.row_values(mx)[0], plain.row_scales(mx)
    s_lo, s_hi = (plain.quantize(v)[1].int() for v in (torch.minimum(lo.abs(), hi.abs()),
                                                       torch.maximum(lo.abs(), hi.abs())))
    s = scales.int()
    assert ((s >= s_lo) & (s <= s_hi)).all()
    a, b = round_at(lo, s), round_at(hi, s)
    bad = (got < a) | (got > b) | torch.isnan(got)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("m,n,k", list(KERNELS_GATED) + [(5, 32, 4865), (40, 96, 4000),
                                                         (300, 64, 4999)])
def test_exact_gates(pa, m, n, k):
    g = gen(m, n, k)
    x, w = integers(g, m, 2 * n, k, DEV)
    scale = gate_scale(k)
    t = totals(x, w) * scale
    gate, up = t[:, :n], t[:, n:]
    assert gate.abs().max() < 80
    lo, hi = silu_ends(gate, up)
    xq, wq = pa.quantize_mx(x), pa.MxWeight(w * scale)
    out = pa.linear_mx(xq, wq, act=pa.ops.ACT_SILU_MUL)
    assert ((out >= lo.to(torch.bfloat16)) & (out <= hi.to(torch.bfloat16))).all()
    between(pa.linear_mx(xq, wq, act=pa.ops.ACT_SILU_MUL, mx_out=True), lo, hi)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_gates_far_below_zero(pa, m):
    """The error of e^-g grows with |g|.  Below -87.3, where 1 / (1 + e^-g) is
    below the normal floats, the result is 0 or the formula's."""
    n, k = 32, 128
    gates = torch.tensor([-1, -2, -4, -8, -16, -20, -24, -32, -40, -48, -56, -60, -64, -72, -80,
                          -88], device=DEV).float().repeat(2)
    x = torch.zeros(m, k, device=DEV)
    x[:, 0] = 1
    w = torch.zeros(2 * n, k, device=DEV)
    w[:n, 0], w[n:, 0] = gates, 3
    gate, up = gates.double().expand(m, n), torch.full((m, n), 3., dtype=torch.float64, device=DEV)
    lo, hi = silu_ends(gate, up)
    hi = torch.where(gate < -87.3, 0., hi)
    out = pa.linear_mx(pa.quantize_mx(x), pa.MxWeight(w), act=pa.ops.ACT_SILU_MUL)
    assert ((out >= lo.to(torch.bfloat16)) & (out <= hi.to(torch.bfloat16))).all()


def tops(v):
    """The largest magnitude of each 16 columns."""
    pad = -v.shape[1] % 16
    return torch.nn.functional.pad(v.abs(), (0, pad)).view(len(v), -1, 16).amax(-1)


@pytest.mark.parametrize("m,n,k", list(KERNELS) + [(32, 1000, 4864), (333, 896, 4864),
                                                   (300, 512, 16384)])
def test_error_of_random_products(pa, m, n, k):
    """The root of the mean square of what products of normal values are off by.
    Each of 16 aligned products loses less than 2^-13 of the largest (cut off
    towards zero: their signs are as random as the values', and the losses of
    one output, at most spread evenly over that range, add up as the root of
    their squares): sqrt(16 / 3) 2^-13 of each group's.  Adding the K / 16 groups
    in f32 is less than 2^-24 of the largest sum each, far less; and the residual
    leaves outputs of at most 2^-8 of the products, rounded to 2^-8 of that."""
    g = gen(m, n, k, "random")
    x = pa.quantize_mx(torch.randn(m, k, generator=g, device=DEV))
    w = weight(pa, g, n, k)
    xv, wv = plain.dequantize(x)[:, :k], plain.weight_values(w)
    ref = xv @ wv.t()
    res = cancel(ref)
    out = pa.linear_mx(x, w, residual=res).double()
    want = ref + res.double()
    square = (tops(xv).pow(2) @ tops(wv).pow(2).t()).mean() * (16 / 3 * 2.0 ** -26)
    square = square + want.pow(2).mean() * 2.0 ** -16 + ref.pow(2).mean() * (k / 16 * 2.0 ** -48)
    assert (out - want).pow(2).mean() <= square
    assert (out - want).abs().max() <= 16 * square.sqrt()
