"""The MXFP8 operators against their definitions in 64 bits (mx_plain.py), at
the sizes, layouts and values where they can go wrong."""
import zlib

import pytest
import torch

import mx_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float32]
EPS = 1e-6


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def hidden_states(g, rows, cols, dtype=torch.float32):
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= 1 + 20 * (torch.rand(cols, generator=g, device=DEV) < 0.02)
    return x.to(dtype)


def same_as_definition(mx, y):
    """Codes and scales of values that need no rounding before them: equal."""
    v, s = plain.quantize(y)
    got, _ = plain.row_values(mx)
    assert torch.equal(plain.row_scales(mx), s)
    assert torch.equal(torch.nan_to_num(got, 1e9), torch.nan_to_num(v, 1e9))


SIZES = [(2500, 130), (2048, 2300), (1, 1), (1, 32), (3, 31), (2, 33), (16, 128), (17, 129),
         (5, 896), (64, 1000), (33, 2048), (7, 2049), (4, 4096), (5, 5000), (3, 8200), (2, 12289),
         (1000, 40), (4099, 96), (4100, 700)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(pa, rows, cols, dtype):
    x = hidden_states(gen(rows, cols), rows, cols, dtype)
    same_as_definition(pa.quantize_mx(x), x.double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strided_and_misaligned(pa, dtype):
    wide = hidden_states(gen(1), 37, 513, dtype)
    for lo, hi in ((0, 512), (1, 301), (3, 500), (509, 513)):
        x = wide[:, lo:hi]
        same_as_definition(pa.quantize_mx(x), x.double())
    one = wide[5:6, 7:200]
    same_as_definition(pa.quantize_mx(one), one.double())


def test_quantize_values(pa):
    """Every magnitude: powers of two around the scale's borders, ties between
    codes, subnormal floats and codes, zeros, the largest floats."""
    v = []
    for e in (-149, -148, -140, -136, -127, -126, -120, -10, -1, 0, 1, 8, 100, 127):
        for m in (1.0, 1.0 + 2.0 ** -23, 1.0625, 1.125, 1.1875, 1.5, 1.75, 1.75 + 2.0 ** -23,
                  2.0 - 2.0 ** -23):
            v.append(m * 2.0 ** e)
    v = torch.tensor(v, dtype=torch.float64).to(torch.float32)
    v = torch.cat([v, -v, torch.zeros(2)]).to(DEV)
    # each as the largest of its block, over blocks of its own fractions
    frac = torch.cat([torch.tensor([1.0]), 2.0 ** -torch.arange(0, 21).float(),
                      torch.tensor([0.9375, 0.53125, 0.28125, 0.0009765625, 3e-4, 1e-5, 0., -0.,
                                    -0.71875, -0.3])])[:32].to(DEV)
    x = v[:, None] * frac
    same_as_definition(pa.quantize_mx(x.contiguous()), x.double())
    # every half step between codes is a tie
    t = torch.arange(0, 1025, device=DEV).float() * 2.0 ** -10
    t = torch.cat([t, torch.arange(1, 449, device=DEV).float(), t * 448])
    x = torch.cat([t, -t, t.new_zeros(-2 * len(t) % 31)]).view(-1, 31)
    x = torch.cat([torch.full((len(x), 1), 448.0, device=DEV), x], 1)
    same_as_definition(pa.quantize_mx(x), x.double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_non_finite(pa, dtype):
    """NaN and infinities become NaN codes and leave the rest of their block."""
    x = hidden_states(gen(2), 6, 96, dtype)
    x[0, 3] = float("nan")
    x[1, 40] = float("inf")
    x[2, 95] = -float("inf")
    x[3, :32] = float("nan")
    x[4] = float("inf")
    same_as_definition(pa.quantize_mx(x), x.double())


def test_outputs_stay_in_their_rows(pa):
    """The scales of the rows behind the last and what follows the arrays stay."""
    rows, cols = 21, 300
    x = hidden_states(gen(3), rows, cols)
    codes = torch.full((rows + 3, 384), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((3 * 32 * 4 + 64,), 0xCD, dtype=torch.uint8, device=DEV)
    out = pa.MxRows(codes[:rows], scales[:3 * 32 * 4].view(3, 32, 4), rows, cols)
    assert pa.quantize_mx(x, out=out) is out
    same_as_definition(out, x.double())
    assert (codes[rows:] == 0xAB).all() and (scales[3 * 32 * 4:] == 0xCD).all()
    assert (out.scales[:, rows:] == 0xCD).all()
    w = torch.ones(cols, device=DEV)
    out.scales[:, :rows] = 0
    pa.rms_norm_mx(x, w, EPS, out=out)
    assert (codes[rows:] == 0xAB).all() and (out.scales[:, rows:] == 0xCD).all()


# ---- RMSNorm ---------------------------------------------------------------


def norm_reference(x, add, w):
    """The sum as it is stored, and the row's result in 64 bits, of which the
    kernel's codes are."""
    s = x.double() if add is None else (x.float() + add.float()).to(x.dtype).double()
    return s, s / (s.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w.double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("rows,cols", SIZES + [(2, 16000), (2, 20000), (2100, 200), (2065, 4097)])
def test_rms_norm(pa, rows, cols, dtype, with_add):
    g = gen(rows, cols, with_add)
    x = hidden_states(g, rows, cols, dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(dtype)
    add = hidden_states(g, rows, cols, dtype) if with_add else None
    s, y = norm_reference(x, add, w)
    before = x.clone()
    total = torch.empty_like(x) if with_add else None
    mx = pa.rms_norm_mx(x, w, EPS, add=add, residual_out=total)
    assert torch.equal(x, before)
    if with_add:
        assert torch.equal(total.double(), s)
    same_as_definition(mx, y)
    # in place: the same sum and the same codes
    mx2 = pa.rms_norm_mx(x, w, EPS, add=add)
    assert torch.equal(mx.codes, mx2.codes)
    assert torch.equal(plain.row_scales(mx), plain.row_scales(mx2))
    assert torch.equal(x.double(), s)


def test_rms_norm_special_rows(pa):
    """A row of zeros, one of the smallest values, one with an infinity, one
    with a NaN, one whose squares pass f32, a weight that makes a value do so:
    as the formula has them."""
    x = torch.ones(6, 256, device=DEV)
    x[0] = 0
    x[1] = 1e-30
    x[2, 7] = float("inf")
    x[3, 200] = float("nan")
    x[4] = 1e30
    w = torch.ones(256, device=DEV)
    v = plain.dequantize(pa.rms_norm_mx(x, w, EPS))
    assert (v[0] == 0).all()
    # 1e-30 / sqrt(eps): within half a step of 2^-4
    assert ((v[1] / 1e-27 - 1).abs() <= 2.0 ** -4).all()
    assert torch.isnan(v[2, 7]) and (torch.cat([v[2, :7], v[2, 8:]]) == 0).all()
    assert torch.isnan(v[3]).all()
    assert (v[4] == 1).all()
    w[9] = 2.0 ** 127
    x[5, 9] = 4
    v = plain.dequantize(pa.rms_norm_mx(x, w, EPS))
    assert torch.isnan(v[5, 9]) and (torch.cat([v[5, :9], v[5, 10:]]) > 0.9).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm_misaligned(pa, dtype):
    """Contiguous tensors that start one element behind a 16-byte border."""
    rows, cols = 9, 333
    g = gen(4)

    def odd(n):
        return torch.randn(n + 1, generator=g, device=DEV).to(dtype)[1:]

    x, add, w = odd(rows * cols).view(rows, cols), odd(rows * cols).view(rows, cols), odd(cols)
    s, y = norm_reference(x, add, w)
    same_as_definition(pa.rms_norm_mx(x, w, EPS, add=add), y)
    assert torch.equal(x.double(), s)


# ---- products --------------------------------------------------------------


def weight(pa, g, n, k, dtype=torch.bfloat16):
    return pa.MxWeight((torch.randn(n, k, generator=g, device=DEV) * k ** -0.5).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 40), (100, 896), (3, 2050), (33, 5000)])
def test_pack(pa, n, k, dtype):
    w = hidden_states(gen(n, k), n, k, dtype)
    mx = pa.MxWeight(w)
    v, s = plain.quantize(w.double())
    ref = (v.view(n, -1, 32) * torch.exp2(s.double() - 127)[..., None]).view(n, -1)
    assert not ref[:, k:].any()
    assert torch.equal(plain.weight_values(mx), ref[:, :k])
    # the rows and columns behind the last are zero codes
    np_ = plain.up(n, 16)
    codes = mx.codes.view(np_ // 16, -1, 8, 16, 16).permute(0, 3, 1, 2, 4).reshape(np_, -1)
    assert not codes[n:].any() and not codes[:, k:].any()


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (896, 300)])
def test_from_packed(pa, n, k):
    """A weight from its packed arrays, whose sizes are the library's."""
    w = pa.MxWeight(hidden_states(gen(n, k), n, k))
    lib = pa._lib.load()
    assert w.codes.numel() == lib.pa_mx_weight_bytes(n, k)
    assert w.scales.numel() == lib.pa_mx_scale_bytes(n, k)
    again = pa.MxWeight.from_packed(w.codes, w.scales, n, k)
    x = pa.quantize_mx(hidden_states(gen(3), 5, k))
    assert torch.equal(pa.linear_mx(x, again), pa.linear_mx(x, w))
    for codes, scales, rows, cols in (
            (w.codes[:-1], w.scales, n, k), (w.codes, w.scales[1:], n, k),
            (w.codes, w.scales, n, k + 128), (w.codes[:0], w.scales[:0], 0, k),
            (w.codes.cpu(), w.scales, n, k), (w.codes.view(torch.int8), w.scales, n, k)):
        with pytest.raises(ValueError):
            pa.MxWeight.from_packed(codes, scales, rows, cols)


def product(x, w):
    """The product in 64 bits, and what it may be off.  The matrix instructions
    align the (exact) products of 16 consecutive columns to the largest of them
    and keep 13 binary places below its leading one: 16 products each lose less
    than 2^-13 of the largest, which is at most the product of the largest
    magnitudes of both operands.  (Measured on the instructions with one small
    product between two large ones of opposite sign: within 16 columns it is
    kept down to 2^-13 of them, beside other columns to 2^-23.)  The groups'
    sums are added in f32: fewer than K roundings of at most the sum of all
    magnitudes."""
    def tops(v):
        pad = -v.shape[1] % 16
        return torch.nn.functional.pad(v.abs(), (0, pad)).view(len(v), -1, 16).amax(-1)

    err = tops(x) @ tops(w).t() * (16 * 2.0 ** -13)
    return x @ w.t(), err + x.abs() @ w.abs().t() * (x.shape[1] * 2.0 ** -24)


def near_bf16(out, ref, err):
    bad = ~((out.double() - ref).abs() <= err + (ref.abs() + err) * 2.0 ** -8 + 1e-38)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


# rows around the tiles' heights, widths off the tiles and off the 16-byte
# stores, K off the blocks and steps
PRODUCTS = [(1, 1, 1), (1, 16, 32), (2, 17, 33), (3, 64, 128), (7, 100, 129), (16, 896, 896),
            (17, 1152, 896), (31, 900, 300), (32, 4864, 896), (33, 40, 4864), (48, 2050, 640),
            (64, 896, 4864), (65, 72, 257), (100, 1001, 1000), (127, 128, 128), (128, 130, 2048),
            (129, 257, 384), (200, 520, 4096), (255, 255, 255), (256, 256, 256), (257, 300, 512),
            (333, 896, 4864), (513, 1025, 130), (618, 2056, 1152), (1025, 640, 896),
            (2100, 1100, 300), (5000, 900, 160), (70, 5, 40), (66, 8, 33), (300, 9, 200),
            (130, 15, 100), (2000, 3, 64), (700, 1031, 96)]


# ... and those that reach every kernel and tiling; test_mx_tiling.py holds the
# rule to these names.
KERNELS = {
    (16, 1000, 384): "few rows 1/8", (17, 1000, 384): "few rows 1/8",
    (33, 1000, 1200): "few rows 1/8", (9, 4130, 200): "few rows 2/4",
    (32, 17001, 140): "few rows 2/4", (50, 32801, 700): "few rows 2/4",
    (20, 8010, 260): "64x32", (65, 101, 640): "64x32", (37, 70, 5000): "64x32",
    (600, 900, 700): "64x64", (130, 5204, 300): "64x64",
    (618, 2056, 1152): "128x64", (5463, 134, 1100): "128x64", (5515, 139, 200): "128x64",
    (999, 4010, 1100): "128x128", (1999, 2054, 900): "128x128 pair",
    (1430, 4014, 2000): "256x128", (4669, 1668, 2000): "256x256",
}
KERNELS_GATED = {
    (10, 160, 600): "few rows 2/4", (12, 8224, 140): "few rows 2/2",
    (32, 8224, 140): "few rows 2/2", (26, 96, 700): "few rows 2/2",
    (20, 96, 4200): "64x64", (53, 128, 900): "64x64", (71, 4352, 2000): "128x64",
    (80, 4416, 200): "128x64", (700, 2080, 500): "128x128",
    (1100, 2080, 300): "128x128 pair",
    (652, 4128, 2000): "256x128",
    (658, 5856, 2000): "256x256",
}


@pytest.mark.parametrize("epi", ["none", "bias", "residual", "both"])
@pytest.mark.parametrize("m,n,k", PRODUCTS + list(KERNELS))
def test_linear(pa, m, n, k, epi):
    g = gen(m, n, k, epi)
    x = pa.quantize_mx(hidden_states(g, m, k))
    w = weight(pa, g, n, k)
    bias = res = None
    if epi in ("bias", "both"):  # at an odd offset: the bias has no alignment of its own
        bias = torch.randn(n + 1, generator=g, device=DEV).to(torch.bfloat16)[1:]
    if epi in ("residual", "both"):
        res = hidden_states(g, m, n, torch.bfloat16)
    ref, err = product(plain.dequantize(x)[:, :k], plain.weight_values(w))
    for more in (bias, res):
        if more is not None:
            err = err + (ref.abs() + err + more.double().abs()) * 2.0 ** -24
            ref = ref + more.double()
    out = pa.linear_mx(x, w, bias=bias, residual=res)
    near_bf16(out, ref, err)
    assert torch.equal(out, pa.linear_mx(x, w, bias=bias, residual=res))
    if res is not None:  # the residual stream updated in place
        assert pa.linear_mx(x, w, bias=bias, residual=res, out=res) is res
        assert torch.equal(out, res)


GATED = [(1, 32, 1), (2, 32, 40), (3, 64, 128), (16, 96, 300), (17, 4864, 896), (32, 160, 896),
         (33, 128, 129), (64, 416, 1000), (65, 32, 64), (100, 224, 256), (130, 288, 896),
         (257, 1056, 384), (333, 4864, 896), (700, 352, 1100), (1100, 2080, 160),
         (4000, 192, 256)]


def gated_reference(x, w, n):
    gu, err = product(x, w)
    gate, up, eg, eu = gu[:, :n], gu[:, n:], err[:, :n], err[:, n:]
    silu = gate / (1 + torch.exp(-gate))
    y = silu * up
    # |silu'| < 1.1; the exponential, the sum, the division and two products
    return y, 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + y.abs() * 16 * 2.0 ** -24


@pytest.mark.parametrize("m,n,k", GATED + list(KERNELS_GATED))
def test_linear_swiglu(pa, m, n, k):
    g = gen(m, n, k)
    x = pa.quantize_mx(hidden_states(g, m, k))
    w = weight(pa, g, 2 * n, k)
    y, err = gated_reference(plain.dequantize(x)[:, :k], plain.weight_values(w), n)
    out = pa.linear_mx(x, w, act=pa.ops.ACT_SILU_MUL)
    near_bf16(out, y, err)
    mx = pa.linear_mx(x, w, act=pa.ops.ACT_SILU_MUL, mx_out=True)
    plain.assert_rounds(mx, y, err)
    again = pa.linear_mx(x, w, act=pa.ops.ACT_SILU_MUL, mx_out=True)
    assert torch.equal(mx.codes, again.codes)
    assert torch.equal(plain.row_scales(mx), plain.row_scales(again))


@pytest.mark.parametrize("m", [5, 70, 300])
def test_linear_outputs_stay_in_their_rows(pa, m):
    """What follows an output, and the scales of the rows behind the last, stay."""
    g = gen(m)
    n, k = 96, 200
    x = pa.quantize_mx(hidden_states(g, m, k))
    w = weight(pa, g, 2 * n, k)
    r = plain.up(m, 16)
    codes = torch.full((m + 2, 128), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((r * 4 + 64,), 0xCD, dtype=torch.uint8, device=DEV)
    out = pa.MxRows(codes[:m], scales[:r * 4].view(1, r, 4), m, n)
    pa.linear_mx(x, w, act=pa.ops.ACT_SILU_MUL, out=out, mx_out=True)
    assert (codes[m:] == 0xAB).all() and (scales[r * 4:] == 0xCD).all()
    assert (out.scales[:, m:] == 0xCD).all()
    assert not out.codes[:, n:].any() and not out.scales[0, :m, 3].any()
    for n in (96, 90):
        buf = torch.full((m + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
        pa.linear_mx(x, weight(pa, g, n, k), out=buf[:m])
        assert (buf[m:] == 7).all()


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_non_finite(pa, m):
    """A NaN in a row of x reaches that row of the output alone, one in a row
    of the weight that column; products beyond f32 are infinite."""
    g = gen(m)
    n, k = 80, 300
    xf = hidden_states(g, m, k)
    xf[1, 299] = float("nan")
    wf = torch.randn(n, k, generator=g, device=DEV)
    wf[70, 0] = float("inf")
    out = pa.linear_mx(pa.quantize_mx(xf), pa.MxWeight(wf))
    nan = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    nan[1] = True
    nan[:, 70] = True
    assert torch.equal(torch.isnan(out), nan) and torch.isfinite(out[~nan]).all()
    big = torch.full((m, 128), 2.0 ** 70, device=DEV)
    assert (pa.linear_mx(pa.quantize_mx(big), pa.MxWeight(big)) == float("inf")).all()
    small = torch.full((m, 128), 2.0 ** -90, device=DEV)
    assert (pa.linear_mx(pa.quantize_mx(small), pa.MxWeight(small)) == 0).all()


def test_linear_scale_range(pa):
    """Scales from both ends of their range cancel in a product."""
    x = pa.quantize_mx(torch.full((3, 160), 2.0 ** 100, device=DEV))
    w = pa.MxWeight(torch.full((20, 160), 2.0 ** -101, device=DEV))
    assert (pa.linear_mx(x, w) == 80).all()


@pytest.mark.parametrize("m", [5, 40, 300])
def test_swiglu_non_finite(pa, m):
    """NaN and infinite gates and ups in bf16 and as codes: NaN codes in their
    columns alone, and no part in their block's scale; gates far below zero
    give zeros."""
    n, k = 96, 128
    x = torch.zeros(m, k, device=DEV)
    x[:, 0] = 1
    x[1, 1] = 1
    w = torch.zeros(2 * n, k, device=DEV)
    w[:n, 0], w[n:, 0] = 2, 3
    big = 2.0 ** 127
    w[4, 1], w[n + 9, 1] = float("nan"), float("inf")  # both NaN codes
    w[40, 1] = -600
    w[70, 0], w[n + 70, 0] = big, big  # inf in every row
    xq, wq = pa.quantize_mx(x), pa.MxWeight(w)
    out = pa.linear_mx(xq, wq, act=pa.ops.ACT_SILU_MUL)
    y = 2 / (1 + torch.exp(torch.tensor(-2., dtype=torch.float64))).item() * 3
    plainly = torch.ones(m, n, dtype=torch.bool, device=DEV)
    plainly[1, 40] = False
    plainly[:, [4, 9, 70]] = False  # 0 * NaN is NaN: in the rows whose x is 0 too
    # the constants' own codes (2, 3, 1 are exact), the result's rounding, and
    # the exponential and reciprocal
    assert ((out[plainly].double() / y - 1).abs() <= 2.0 ** -8 + 2.0 ** -20).all()
    assert torch.isnan(out[:, [4, 9]]).all() and (out[1, 40].abs() < 1e-30).all()
    assert (out[:, 70] == float("inf")).all()
    mx = pa.linear_mx(xq, wq, act=pa.ops.ACT_SILU_MUL, mx_out=True)
    v = plain.dequantize(mx)
    nan = torch.zeros(m, 128, dtype=torch.bool, device=DEV)
    nan[:, [4, 9, 70]] = True
    assert torch.equal(torch.isnan(v), nan)
    assert ((v[:, :n][plainly] / y - 1).abs() <= 2.0 ** -4 + 2.0 ** -20).all()
    assert v[1, 40].abs() < 1e-2 and not v[:, n:].any()


def integers(g, rows, cols, low=-2, high=3):
    """Small integers: their codes, products and (below 2^24) sums are exact."""
    return torch.randint(low, high, (rows, cols), generator=g, device=DEV, dtype=torch.int8)


def exact_product(x, w):
    """Of integer matrices, in f64 by columns."""
    out = torch.zeros(len(x), len(w), dtype=torch.float64, device=DEV)
    for i in range(0, x.shape[1], 1 << 20):
        out += x[:, i:i + (1 << 20)].double() @ w[:, i:i + (1 << 20)].double().t()
    return out


@pytest.mark.parametrize("m,n", [(1, 20), (17, 40), (70, 24), (257, 32)])
def test_longest_rows(pa, m, n):
    """2^22 columns, the most: quantised, normed and multiplied."""
    k, g = 1 << 22, gen(m, n)
    xi, wi = integers(g, m, k), integers(g, n, k)
    xb = xi.to(torch.bfloat16)
    x = pa.quantize_mx(xb)
    ref = exact_product(xi, wi)
    assert ref.abs().max() < 2 ** 24
    w = pa.MxWeight(wi.to(torch.bfloat16))
    assert torch.equal(pa.linear_mx(x, w), ref.to(torch.bfloat16))
    if m <= 17:
        one = torch.ones(k, dtype=torch.bfloat16, device=DEV)
        s = xb.double()
        same_as_definition(pa.rms_norm_mx(xb, one, EPS),
                           s / (s.pow(2).mean(-1, keepdim=True) + EPS).sqrt())


def test_past_32_bits(pa):
    """Arrays of more than 2^32 bytes and 2^31 elements: the last rows as in a
    call of their own."""
    rows, cols, last = 540_001, 4096, slice(540_001 - 70, 540_001)
    g = gen(0)
    x = integers(g, rows, cols, -100, 100).to(torch.bfloat16)
    q = pa.quantize_mx(x)
    few = pa.quantize_mx(x[last])
    assert torch.equal(q.codes[last], few.codes)
    assert torch.equal(q.scales[:, last], few.scales[:, :70])
    wt = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
    add = x[last].clone()
    few = pa.rms_norm_mx(x[last].contiguous(), wt, EPS)
    q = pa.rms_norm_mx(x, wt, EPS, out=q)
    assert torch.equal(q.codes[last], few.codes)
    assert torch.equal(q.scales[:, last], few.scales[:, :70])
    assert torch.equal(x[last], add)
    del q
    k = 128
    xi, wi = integers(g, rows, k), integers(g, cols, k)
    xq, w = pa.quantize_mx(xi.to(torch.bfloat16)), pa.MxWeight(wi.to(torch.bfloat16))
    out = pa.linear_mx(xq, w, residual=x, out=x)
    want = exact_product(xi[last], wi) + add.double()
    assert torch.equal(out[last], want.to(torch.bfloat16))
    del out, x
    gu = pa.MxWeight(torch.cat([wi, wi]).to(torch.bfloat16))
    act = pa.linear_mx(xq, gu, act=pa.ops.ACT_SILU_MUL, mx_out=True)
    y = exact_product(xi[last], wi)
    y = y * y / (1 + torch.exp(-y))
    part = pa.MxRows.empty(70, cols, DEV)
    part.codes.copy_(act.codes[last])
    part.scales[:, :70] = act.scales[:, last]
    plain.assert_rounds(part, y, y.abs() * 16 * 2.0 ** -24)


def test_no_rows(pa):
    x = torch.empty(0, 896, dtype=torch.bfloat16, device=DEV)
    w = pa.MxWeight(torch.ones(64, 896, device=DEV))
    one = torch.ones(896, dtype=torch.bfloat16, device=DEV)
    for rows in (pa.quantize_mx(x), pa.rms_norm_mx(x, one, EPS, add=x.clone())):
        assert rows.codes.shape == (0, 896) and rows.scales.shape == (7, 0, 4)
        assert pa.linear_mx(rows, w).shape == (0, 64)
        assert pa.linear_mx(rows, w, act=pa.ops.ACT_SILU_MUL, mx_out=True).codes.shape == (0, 128)


def test_refused_outputs(pa):
    """Views that the kernels' wide accesses cannot take, and tensors that do
    not fit."""
    x = pa.quantize_mx(torch.ones(4, 128, device=DEV))
    w = pa.MxWeight(torch.ones(64, 128, device=DEV))
    buf = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    for bad in (buf[1:].view(4, 64), torch.zeros(4, 65, device=DEV, dtype=torch.bfloat16)[:, :64],
                torch.zeros(4, 64, device=DEV),
                torch.zeros(3, 64, device=DEV, dtype=torch.bfloat16)):
        with pytest.raises((ValueError, RuntimeError)):
            pa.linear_mx(x, w, out=bad)
        with pytest.raises((ValueError, RuntimeError)):
            pa.linear_mx(x, w, residual=bad)
    with pytest.raises(ValueError):
        pa.quantize_mx(torch.ones(4, 256, device=DEV), out=x)
    with pytest.raises(ValueError):
        pa.quantize_mx(torch.ones(1, 128, device=DEV).expand(4, 128))
    row = torch.ones(4, 128, device=DEV)
    with pytest.raises((ValueError, RuntimeError)):  # the sum onto add
        pa.rms_norm_mx(row, torch.ones(128, device=DEV), EPS, add=row)
