"""The MXFP8 entry points' sizes and refusals: checked on the host before any
launch, so without a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib(pa):
    return pa._lib.load()


P = C.c_void_p(64)
ODD = C.c_void_p(65)
FAR, NEAR = C.c_void_p(1 << 40), C.c_void_p((1 << 40) + 48)


def test_sizes(lib):
    assert [lib.pa_mx_row_bytes(c) for c in (1, 128, 129, 896, 4864, 0, -1)] == \
        [128, 128, 256, 896, 4864, 0, 0]
    assert lib.pa_mx_scale_bytes(1, 1) == 16 * 4
    assert lib.pa_mx_scale_bytes(17, 896) == 32 * 7 * 4
    assert lib.pa_mx_scale_bytes(0, 896) == 0
    assert lib.pa_mx_weight_bytes(33, 130) == 48 * 256
    # beyond 32 bits
    assert lib.pa_mx_weight_bytes(1 << 20, 1 << 14) == 1 << 34


def quantize(lib, codes=P, scales=P, x=P, rows=4, cols=100, stride=0, dtype=1):
    return lib.pa_quantize_mx(codes, scales, x, rows, cols, stride, dtype, None)


def test_quantize_refusals(lib):
    assert quantize(lib, rows=0, codes=None, scales=None, x=None) == 0
    assert quantize(lib, rows=-1) == -1
    assert quantize(lib, cols=0) == -1
    assert quantize(lib, dtype=2) == -1 and b"dtype" in lib.pa_last_error()
    assert quantize(lib, stride=99) == -1 and b"overlap" in lib.pa_last_error()
    assert quantize(lib, stride=-100) == -1
    assert quantize(lib, stride=1 << 61) == -1 and b"stride" in lib.pa_last_error()
    assert quantize(lib, cols=(1 << 22) + 1) == -3
    for name in ("codes", "scales", "x"):
        assert quantize(lib, **{name: None}) == -1 and b"null" in lib.pa_last_error()
        assert quantize(lib, **{name: ODD}) == -1 and b"aligned" in lib.pa_last_error()
    assert quantize(lib) == -1 and b"overlap" in lib.pa_last_error()
    assert quantize(lib, codes=FAR, x=NEAR) == -1 and b"overlap" in lib.pa_last_error()
    assert quantize(lib, scales=FAR, x=NEAR) == -1 and b"overlap" in lib.pa_last_error()
    assert quantize(lib, codes=FAR, scales=NEAR) == -1 and b"overlap" in lib.pa_last_error()


def norm(lib, codes=None, scales=None, sum=None, residual=None, add=None, weight=None, rows=4,
         hidden=100, dtype=1, **given):
    """Arrays far apart, but for those given (0: none)."""
    at = {n: C.c_void_p((i + 1) << 30) for i, n in enumerate(
        ("codes", "scales", "sum", "residual", "add", "weight"))}
    for n, v in (("codes", codes), ("scales", scales), ("sum", sum), ("residual", residual),
                 ("add", add), ("weight", weight)):
        if v is not None:
            at[n] = C.c_void_p(v) if v else None
    return lib.pa_rms_norm_mx(at["codes"], at["scales"], at["sum"], at["residual"], at["add"],
                              at["weight"], rows, hidden, 1e-6, dtype, None)


def test_norm_refusals(lib):
    assert norm(lib, rows=0, codes=0) == 0
    assert norm(lib, rows=-1) == -1
    assert norm(lib, hidden=0) == -1
    assert norm(lib, dtype=7) == -1
    assert norm(lib, hidden=(1 << 22) + 1) == -3
    assert norm(lib, sum=0) == -1 and b"needs sum" in lib.pa_last_error()
    names = ("codes", "scales", "sum", "residual", "add", "weight")
    for i, name in enumerate(names):
        if name not in ("sum", "add"):
            assert norm(lib, **{name: 0}) == -1 and b"null" in lib.pa_last_error()
        assert norm(lib, **{name: (1 << 40) + 1}) == -1 and b"aligned" in lib.pa_last_error()
    # outputs that reach into another array: 4 rows of 100 bf16 are 800 bytes,
    # of 128 codes 512
    for out, other in (("codes", "scales"), ("codes", "sum"), ("codes", "residual"),
                       ("codes", "add"), ("codes", "weight"), ("scales", "sum"),
                       ("scales", "residual"), ("scales", "add"), ("scales", "weight"),
                       ("sum", "add"), ("sum", "weight")):
        assert norm(lib, **{out: 1 << 40, other: (1 << 40) + 48}) == -1, (out, other)
        assert b"overlap" in lib.pa_last_error()
    # the sum in place is allowed, a shifted one is not
    assert norm(lib, sum=1 << 40, residual=(1 << 40) + 16) == -1
    assert b"overlap" in lib.pa_last_error()


def pack(lib, codes=P, scales=P, weight=P, rows=4, cols=100, dtype=1):
    return lib.pa_linear_mx_pack(codes, scales, weight, rows, cols, dtype, None)


def test_pack_refusals(lib):
    assert pack(lib, rows=0) == -1
    assert pack(lib, cols=0) == -1
    assert pack(lib, dtype=2) == -1
    assert pack(lib, cols=(1 << 22) + 1) == -3
    for name in ("codes", "scales", "weight"):
        assert pack(lib, **{name: None}) == -1
        assert pack(lib, **{name: ODD}) == -1
    assert pack(lib) == -1 and b"overlap" in lib.pa_last_error()


def linear(lib, out=P, out_scales=None, x=P, xs=P, w=P, ws=P, bias=None, residual=None, rows=4,
           n=96, k=100, act=0):
    return lib.pa_linear_mx(out, out_scales, x, xs, w, ws, bias, residual, rows, n, k, act, None)


def test_linear_refusals(lib):
    assert linear(lib, rows=0, out=None, x=None) == 0
    assert linear(lib, rows=-1) == -1
    assert linear(lib, n=0) == -1
    assert linear(lib, k=0) == -1
    assert linear(lib, act=2) == -1 and b"activation" in lib.pa_last_error()
    assert linear(lib, act=1, bias=P) == -1
    assert linear(lib, act=1, residual=P) == -1
    assert linear(lib, out_scales=P) == -1 and b"SwiGLU" in lib.pa_last_error()
    assert linear(lib, act=1, n=48) == -3 and b"multiple of 32" in lib.pa_last_error()
    assert linear(lib, k=(1 << 22) + 1) == -3
    assert linear(lib, n=1 << 24, k=1 << 22) == -3
    for name in ("out", "x", "xs", "w", "ws"):
        assert linear(lib, **{name: None}) == -1 and b"null" in lib.pa_last_error()
    for name in ("out", "x", "xs", "w", "ws", "bias", "residual"):
        assert linear(lib, **{name: ODD}) == -1 and b"aligned" in lib.pa_last_error()
    assert linear(lib, act=1, out_scales=ODD) == -1
    # 4 rows of 96 bf16: 768 bytes
    for name in ("x", "xs", "w", "ws", "bias", "residual"):
        assert linear(lib, out=FAR, **{name: NEAR}) == -1, name
        assert b"overlap" in lib.pa_last_error()
    for name in ("x", "xs", "w", "ws", "out"):
        assert linear(lib, act=1, out_scales=FAR, **{**{"out": C.c_void_p(1 << 41)},
                                                     name: NEAR}) == -1, name
        assert b"overlap" in lib.pa_last_error()


def test_wrappers_refuse_host_tensors(pa):
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        pa.quantize_mx(x)
    with pytest.raises(ValueError):
        pa.rms_norm_mx(x, torch.ones(64), 1e-6)
    with pytest.raises(ValueError):
        pa.MxWeight(x)
    with pytest.raises(ValueError):
        pa.linear_mx(x, x)
    with pytest.raises(ValueError):
        pa.MxRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 16, 4, dtype=torch.uint8),
                  4, 64)


@pytest.mark.parametrize("rows,cols", [(-1, 64), (1 << 31, 64), (4, 0), (4, (1 << 22) + 1),
                                       (4, (1 << 32) + 64)])
def test_wrappers_refuse_sizes(pa, rows, cols):
    """Before anything is allocated, or cut to 32 bits on its way to the library."""
    some = torch.zeros(1, dtype=torch.uint8)
    for make in (lambda: pa.MxRows.empty(rows, cols), lambda: pa.MxRows(some, some, rows, cols),
                 lambda: pa.MxWeight.from_packed(some, some, rows, cols)):
        with pytest.raises(ValueError, match=f"{rows} x {cols}"):
            make()
