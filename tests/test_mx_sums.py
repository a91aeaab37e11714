"""That the operands of mx_sums.py show mistakes in a product's sums: planted
here, in the oracle, on the CPU."""
import pytest
import torch

from mx_sums import STEP, cancel, gate_scale, integers, silu_ends, totals


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def bf16(t):
    return t.to(torch.bfloat16).double()


def drop_last_column(x, w):
    return x[:, :-1].double() @ w[:, :-1].double().t()


def drop_one_group(x, w):
    w = w.clone()
    w[:, 16:32] = 0
    return x.double() @ w.double().t()


def parts(x, w, split):
    """The K steps' sums of two groups, joined in bf16."""
    step = torch.arange(x.shape[1]) // STEP
    n = int(step[-1]) + 1
    mine = step % 2 == 0 if split == "in turn" else step < n // 2
    return sum(bf16(x.double()[:, s] @ w.double()[:, s].t()) for s in (mine, ~mine))


def groups(x, w):
    """The sums of 16 columns, each rounded to bf16."""
    return sum(bf16(x[:, c:c + 16].double() @ w[:, c:c + 16].double().t())
               for c in range(0, x.shape[1], 16))


def last_scale(x, w):
    """The last block of 32 columns times two."""
    w = w.clone()
    w[:, -32:] *= 2
    return x.double() @ w.double().t()


MISTAKES = {"last column": drop_last_column, "16 columns": drop_one_group,
            "halves in bf16": lambda x, w: parts(x, w, "halves"),
            "every other step in bf16": lambda x, w: parts(x, w, "in turn"),
            "16 columns in bf16": groups, "last scale": last_scale}


@pytest.mark.parametrize("k", [384, 896, 2000, 4865])
@pytest.mark.parametrize("mistake", list(MISTAKES))
def test_mistakes_show(mistake, k):
    m, n = 20, 48
    x, w = integers(gen(k), m, n, k, "cpu")
    t, wrong = totals(x, w), MISTAKES[mistake](x, w)
    res = cancel(t)
    # with a residual most outputs, and without one still many
    assert ((wrong + res.double()).to(torch.bfloat16) != (t + res.double()).to(
        torch.bfloat16)).float().mean() > 0.5
    assert (wrong.to(torch.bfloat16) != t.to(torch.bfloat16)).float().mean() > 0.01
    # in gates
    scale = gate_scale(k)
    half = n // 2
    lo, hi = silu_ends(t[:, :half] * scale, t[:, half:] * scale)
    y = wrong * scale
    y = (y[:, :half] / (1 + torch.exp(-y[:, :half])) * y[:, half:]).to(torch.bfloat16)
    bad = (y < lo.to(torch.bfloat16)) | (y > hi.to(torch.bfloat16))
    assert bad.float().mean() > 0.02


def test_ranges():
    """The sums of every shape stay exact, and gates within the exponential."""
    for k in (128, 1000, 4864, 16384):
        x, w = integers(gen(k), 8, 64, k, "cpu")
        t = totals(x, w)
        assert (t * gate_scale(k)).abs().max() < 80
