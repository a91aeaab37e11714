"""Calls of more rows than one launch takes (its threads are counted in 32
bits): every row as in a call of its own.  The rows repeat with a period."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PERIOD = 4096
# a workgroup of 256 threads per row: 2^24 rows pass 2^32 threads
ROWS = (1 << 24) + 3 * PERIOD


def rows_of(cols, rows=ROWS):
    g = torch.Generator(device=DEV).manual_seed(cols)
    base = torch.randn(PERIOD, cols, generator=g, device=DEV).to(torch.bfloat16)
    return base, base.repeat(rows // PERIOD, 1)


def repeats(big, base):
    big = big.view(-1, *base.shape)
    return all(bool((big[i:i + 256] == base).all()) for i in range(0, len(big), 256))


def same_rows(big, base):
    """MxRows of every row equal those of one period."""
    scales = big.scales[:, :big.rows].reshape(big.scales.shape[0], -1, PERIOD, 4)
    return repeats(big.codes, base.codes) and bool((scales == base.scales[:, None]).all())


def test_quantize_mx(pa):
    base, x = rows_of(1032)
    assert same_rows(pa.quantize_mx(x), pa.quantize_mx(base))


def test_pack_mx(pa):
    base, x = rows_of(1032)
    big, few = pa.MxWeight(x), pa.MxWeight(base)
    assert repeats(big.codes, few.codes) and repeats(big.scales, few.scales)


@pytest.mark.parametrize("with_add", [False, True])
def test_rms_norm_mx(pa, with_add):
    base, x = rows_of(1032)
    w = torch.linspace(0.5, 2, 1032, device=DEV).to(torch.bfloat16)
    add = x.flip(1) if with_add else None
    few = pa.rms_norm_mx(base, w, 1e-6, add=add[:PERIOD].clone() if with_add else None)
    assert same_rows(pa.rms_norm_mx(x, w, 1e-6, add=add), few)
    assert repeats(x, base)  # with add the sum, in place


@pytest.mark.parametrize("cols", [1032, 1001])  # rows in registers, and read again
@pytest.mark.parametrize("name", ["rms_norm", "layer_norm"])
def test_norms(pa, name, cols):
    base, x = rows_of(cols)
    w = torch.linspace(0.5, 2, cols, device=DEV).to(torch.bfloat16)
    norm = getattr(pa, name)
    add = x.flip(1)
    few = norm(base, w, 1e-6, add=add[:PERIOD].clone())
    assert repeats(norm(x, w, 1e-6, add=add), few)
    assert repeats(x, base)


def test_norm_of_wide_rows(pa):
    """A workgroup per row held in registers."""
    base, x = rows_of(2056)
    w = torch.linspace(0.5, 2, 2056, device=DEV).to(torch.bfloat16)
    few = pa.rms_norm(base, w, 1e-6)
    assert repeats(pa.rms_norm(x, w, 1e-6, out=x), few)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [24, 17])
def test_argmax(pa, cols, dtype):
    """1024 threads per row."""
    base, x = rows_of(cols, (1 << 22) + 3 * PERIOD)
    base, x = base.to(dtype), x.to(dtype)
    assert bool((pa.argmax(x).view(-1, PERIOD) == pa.argmax(base)).all())
