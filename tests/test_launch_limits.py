"""Calls whose launch would pass 2^32 threads are refused on the host (the
runtime would start a part of them and report success)."""
import ctypes as C

UNSUPPORTED = -3
MOST = 2 ** 31 - 1
FAR = [C.c_void_p(i << 50) for i in range(1, 8)]  # never read


def test_linear_mx(pa):
    lib = pa._lib.load()
    out, x, xs, w, ws = FAR[:5]
    assert lib.pa_linear_mx(out, None, x, xs, w, ws, None, None, MOST, 1, 1, 0,
                            None) == UNSUPPORTED
    assert b"outputs" in lib.pa_last_error()


def test_linear(pa):
    lib = pa._lib.load()
    out, x, w = FAR[:3]
    assert lib.pa_linear(out, x, w, None, MOST, 16, 64, 0, 0, 0, 0., None, 0, 1,
                         None) == UNSUPPORTED
    assert b"outputs" in lib.pa_last_error()
