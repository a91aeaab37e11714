"""Calls whose launch would pass 2^32 threads are refused on the host (the
runtime would start a part of them and report success)."""
import ctypes as C

import pytest

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


def test_cache_calls(pa):
    """A workgroup per token, block, id or sequence."""
    lib = pa._lib.load()
    a, b, c, d, e, f, g = FAR
    n = 1 << 24  # with 256 threads each

    def refused(rc):
        return rc == UNSUPPORTED and b"2^32" in lib.pa_last_error()

    odd = C.c_void_p((1 << 50) + 4)  # off the 16-byte paths
    for dtype in (0, 1):
        assert refused(lib.pa_reshape_and_cache(odd, b, c, d, e, n, 1, 8, 1 << 20, 0, 0, dtype,
                                                None))
        assert refused(lib.pa_reshape_and_cache(a, b, c, d, e, 16 * n, 1, 8, 1 << 20, 0, 0, dtype,
                                                None))
        assert refused(lib.pa_reshape_and_cache_fp8(odd, b, c, d, e, n, 1, 8, 1 << 20, 0, 0,
                                                    dtype, None))
        assert refused(lib.pa_reshape_and_cache_fp8(a, b, c, d, e, 16 * n, 1, 8, 1 << 20, 0, 0,
                                                    dtype, None))
        assert refused(lib.pa_rope_reshape_and_cache(odd, 0, b, 0, c, 0, d, e, f, g, a, n, 1, 1,
                                                     16, 1 << 20, dtype, None))
        assert refused(lib.pa_rope_reshape_and_cache(a, 0, b, 0, c, 0, d, e, f, g, a, 2 ** 31 - 1,
                                                     1, 1, 16, 1 << 20, dtype, None))
        # by token and by block
        assert lib.pa_read_kv(a, b, c, n, n, 1, 1 << 14, 1 << 20, d, e, dtype, None) == UNSUPPORTED
        assert lib.pa_read_kv(a, b, c, n, 16 * n, 1, 8, 1 << 20, d, e, dtype, None) == UNSUPPORTED
    assert refused(lib.pa_read_kv(a, b, c, n, n, 1, 8, 1 << 20, d, e, 2, None))
    assert refused(lib.pa_block_hash(a, b, n, 1, 8, 1 << 20, c, None))
    assert refused(lib.pa_slot_mapping(a, 1, b, c, n, 2 * n, d, None))


@pytest.mark.parametrize("dtype,seqs,heads", [(0, 1 << 24, 1), (0, 1 << 20, 16), (1, 1 << 20, 16)])
def test_decode(pa, dtype, seqs, heads):
    """Contexts in partitions: a workgroup per row joins them."""
    lib = pa._lib.load()
    out, q, k, v, tables, lens, ws = FAR
    assert lib.pa_decode(out, q, k, v, tables, 1 << 12, lens, 1 << 16, seqs, heads, 1, 64, 1 << 20,
                         1., ws, 1 << 62, dtype, None) == UNSUPPORTED
    assert b"in partitions" in lib.pa_last_error()


@pytest.mark.parametrize("dtype,head_dim,max_q", [(0, 64, 1 << 26), (0, 24, 1 << 26),
                                                  (1, 256, 1 << 26), (1, 40, 2 ** 31 - 1),
                                                  (2, 40, 1 << 26), (1, 64, 2 ** 31 - 1),
                                                  (1, 128, 2 ** 31 - 1)])
def test_prefill(pa, dtype, head_dim, max_q):
    """A bound on the rows of a sequence that no launch holds (the tiled kernels:
    over enough sequences and heads)."""
    lib = pa._lib.load()
    out, q, k, v, tables, cu, past = FAR
    assert lib.pa_prefill(out, q, k, v, tables, 16, cu, past, 64, 1000, max_q, 8, 8, head_dim,
                          1 << 20, 1., dtype, None) == UNSUPPORTED
    assert b"too large" in lib.pa_last_error()
