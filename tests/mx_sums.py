"""Operands of pa_linear_mx whose sums over K are exact, whatever their order,
so that outputs can be held to the last bit: small integers, whose products of
16 columns need no more than 7 binary places and whose sums stay below 2^24.
The sign of a weight changes with every step of 128 columns, so the parts that
share K are large and partly cancel."""
import torch

STEP = 128


def integers(g, m, n, k, device, same_rows=False):
    """x [m, k] of 1 to 8, w [n, k] of magnitudes 1 to 8, signs by step."""
    def small(rows):
        return torch.randint(1, 9, (rows, k), generator=g, device=device).float()

    x, w = small(1).expand(m, k).contiguous() if same_rows else small(m), small(n)
    sign = torch.randint(0, 2, (n, -(-k // STEP)), generator=g, device=device).float() * 2 - 1
    return x, w * sign.repeat_interleave(STEP, 1)[:, :k]


def totals(x, w):
    t = x.double() @ w.double().t()
    assert t.abs().max() < 2 ** 24
    return t


def cancel(t):
    """A residual (or bias) that leaves what bf16 cannot hold of t."""
    return -t.to(torch.bfloat16)


def gate_scale(k):
    """The power of two that makes gates of integers() about 4."""
    size = 20.25 * STEP * (k / STEP) ** 0.5
    return 2.0 ** -round(torch.tensor(size / 4).log2().item())


def silu_ends(gate, up):
    """silu(gate) up of exact gates and ups at both ends of what the kernel may
    return, before its rounding to the output's type: e^-g is exp2 of g log2(e)
    rounded (log2(e) is off by less than 2^-25 of itself, the product by 2^-24:
    1.5 |g| 2^-24 of e^-g) within a step of 2^-23; the sum 2^-24, the reciprocal
    a step of 2^-23, two products 2^-24 each: 7 2^-24 and second-order terms."""
    y = gate / (1 + torch.exp(-gate)) * up
    off = y.abs() * (1.5 * gate.abs() + 8) * 2.0 ** -24
    return y - off, y + off
