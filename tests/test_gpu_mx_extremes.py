"""rms_norm_mx at both ends of the floats' range: the codes of the formula."""
import pytest
import torch

import mx_plain as plain
from test_gpu_mx import DEV, gen, same_as_definition

pytestmark = pytest.mark.gpu

def either_side(mx, y, rel):
    """The codes of y, which is known to within rel: of one end or the other.
    Small integers times a power of two (bf16 below the normal floats) have
    roots that make y a tie between two codes exactly, and which side 64 bits
    put it on is then their rounding.  rel, for n columns: the squares are
    exact, their sum has less than n roundings of 2^-53, halved by the root, in
    the reference and again in the kernel: n 2^-53 for both; and the mean, eps,
    the root, the division and the product of each with less than 8 2^-53."""
    lo, hi = y * (1 - rel), y * (1 + rel)
    got, _ = plain.row_values(mx)
    scales = plain.row_scales(mx)
    fits = torch.zeros_like(got, dtype=torch.bool)
    for end in (lo, hi):
        v, s = plain.quantize(end)
        fits |= (got == v) & (scales == s).repeat_interleave(32, 1)
    assert fits.all(), int((~fits).sum())


# name: (scale of even columns, of odd columns, weight of even columns, of odd, eps)
CASES = {
    "rows as small as floats go, no eps": (1e-39, 3e-44, 1., 1., 0.),
    "squares below f32, no eps": (1e-25, 1e-30, 1., 1., 0.),
    "small rows under eps": (1e-38, 1e-38, 1e10, 1., 1e-6),
    "large rows, a reciprocal below the normal floats": (3e37, 1e37, 1., 1., 1e-6),
    "small values, large weights": (1e-36, 1e5, 1e36, 1., 1e-6),
    "values below the normal floats, large weights": (1e-39, 1e4, 1e37, 1., 1e-6),
    "results below the normal floats": (1., 1., 1e-39, 1e-41, 1e-6),
    "blocks of small results": (1., 1e-3, 1e-19, 1e-23, 1e-6),
    "a large eps": (1e-30, 1e-33, 1e30, 1e33, 1e10),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(64, 1024), (3, 4500), (2, 17000), (4096, 500)])
@pytest.mark.parametrize("name", list(CASES))
def test_rms_norm_range(pa, name, rows, cols, dtype):
    even, odd, w_even, w_odd, eps = CASES[name]
    g = gen(name, rows, cols)
    x = torch.randn(rows, cols, generator=g, device=DEV).clamp(-5, 5).double()
    x[:, ::2] *= even
    x[:, 1::2] *= odd
    # blocks of zeros between them
    x[:, 64:96] = 0
    x = x.to(dtype)
    w = 1 + 0.2 * torch.randn(cols, generator=g, device=DEV).clamp(-4, 4).double()
    w[::2] *= w_even
    w[1::2] *= w_odd
    w = w.to(dtype)
    s = x.double()
    eps = float(torch.tensor(eps, dtype=torch.float32))
    y = s / (s.pow(2).mean(1, keepdim=True) + eps).sqrt() * w.double()
    assert y.abs().max() < 3e38
    either_side(pa.rms_norm_mx(x, w, eps), y, (cols + 16) * 2.0 ** -53)


def test_signalling_nans(pa):
    """NaNs that no arithmetic has quieted take no part in their block's scale."""
    for dtype, whole, bits in ((torch.float32, torch.int32, 0x7F810000),
                               (torch.bfloat16, torch.int16, 0x7F81)):
        x = torch.randn(8, 256, generator=gen(dtype), device=DEV).to(dtype)
        x[:, 3] = 100
        x.view(whole)[2, 5] = bits
        x.view(whole)[3, 31] = bits
        assert torch.isnan(x).sum() == 2
        same_as_definition(pa.quantize_mx(x), x.double())
        w = x[0].clone()
        w.view(whole)[40] = bits
        one = torch.ones(8, 256, dtype=dtype, device=DEV)
        same_as_definition(pa.rms_norm_mx(one, w, 0.), one.double() * w.double())
