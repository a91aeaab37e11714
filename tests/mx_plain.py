"""MXFP8 in 64 bits, from its definition: blocks of 32 columns, the smallest
power of two (at least 2^-127) that keeps the block's largest finite value
within 448 of it, E4M3 values rounded to nearest even."""
import torch


def up(n, m):
    return -(-n // m) * m


def decode_table():
    v = torch.zeros(256, dtype=torch.float64)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[b] = float("nan") if b & 127 == 127 else (-x if b & 128 else x)
    return v


def quantize(y):
    """f64 rows -> (E4M3 values [rows, Kp], scale bytes [rows, Kp / 32])."""
    rows, cols = y.shape
    wide = torch.zeros(rows, up(cols, 128), dtype=torch.float64, device=y.device)
    wide[:, :cols] = y
    t = wide.view(rows, -1, 32)
    mag = torch.where(torch.isfinite(t), t.abs(), 0.0)
    m, x = torch.frexp(mag.amax(-1))  # m 2^x, 0.5 <= m < 1; 448 = 0.875 2^9
    e = torch.where(m == 0, -127, (x - 9 + (m > 0.875))).clamp(min=-127)
    t = t * torch.exp2(-e.double())[..., None]
    t = torch.where(torch.isfinite(t), t, float("nan"))
    _, x = torch.frexp(t)
    step = torch.exp2((x - 4).clamp(min=-9).double())  # 8 steps a power of two
    v = torch.where(torch.isnan(t), t, (t / step).round() * step)
    return v.view(rows, -1), (e + 127).to(torch.uint8)


def row_scales(mx):
    """The scale bytes of MxRows as [rows, Kp / 32]."""
    return mx.scales[:, :mx.rows].permute(1, 0, 2).reshape(mx.rows, -1)


def row_values(mx):
    """The E4M3 values and the scales (f64) of MxRows, per column."""
    v = decode_table().to(mx.codes.device)[mx.codes.long()]
    s = torch.exp2(row_scales(mx).double() - 127).repeat_interleave(32, 1)
    return v, s


def dequantize(mx):
    v, s = row_values(mx)
    return v * s


def weight_values(w):
    """An MxWeight's values [N, K] in 64 bits."""
    n, k = w.shape
    np_, steps = up(n, 16), up(k, 128) // 128
    codes = w.codes.view(np_ // 16, steps, 8, 16, 16).permute(0, 3, 1, 2, 4).reshape(np_, -1)
    s = w.scales.view(np_ // 16, steps, 16, 4).permute(0, 2, 1, 3).reshape(np_, -1)
    v = decode_table().to(codes.device)[codes.long()]
    return (v * torch.exp2(s.double() - 127).repeat_interleave(32, 1))[:n, :k]


def assert_rounds(mx, y, err):
    """mx holds f64 rows y, themselves off by at most err: every value within
    half an E4M3 step (2^-4 of the value, 2^-10 of the scale at the bottom) of
    one within err of y, and every scale the definition's for a largest value
    within err; columns behind the last are zero."""
    v, s = row_values(mx)
    cols = y.shape[1]
    assert not v[:, cols:].any()
    half = torch.maximum((y.abs() + err) * 2.0 ** -4, s[:, :cols] * 2.0 ** -10)
    off = (v * s)[:, :cols] - y
    bad = ~(off.abs() <= half + err)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float(off.abs().max()))
    pad = up(cols, 128) - cols
    top = torch.nn.functional.pad(y.abs(), (0, pad)).view(len(y), -1, 32).amax(-1)
    e = torch.nn.functional.pad(err, (0, pad)).view(len(y), -1, 32).amax(-1)
    s = s.view(len(y), -1, 32)[..., 0]
    assert (top - e <= 448 * s).all()
    assert ((top + e >= 224 * s) | (s == 2.0 ** -127)).all()
