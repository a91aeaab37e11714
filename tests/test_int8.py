"""The int8 cache without a GPU: refusals of its entry points, and the definition's
plain form against itself."""
import ctypes as C

import numpy as np
import pytest
import torch

import int8_plain

P = C.c_void_p(256)


@pytest.fixture(scope="module")
def lib(pa):
    return pa._lib.load()


def append(lib, **kw):
    a = dict(k=P, v=P, ks=P, vs=P, key=P, kst=0, value=P, vst=0, q=None, qst=0, inv=None, tab=P,
             mbs=4, cu=P, ctx=P, b=2, t=4, most=2, hq=4, hkv=2, d=64, nb=16, dtype=1, stream=None)
    a.update(kw)
    return lib.pa_append_int8(*a.values())


def decode(lib, **kw):
    a = dict(out=P, q=P, k=P, v=P, ks=P, vs=P, tab=P, mbs=4, ctx=P, most=64, b=2, hq=4, hkv=2,
             d=64, nb=16, scale=1.0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return lib.pa_decode_int8(*a.values())


def prefill(lib, **kw):
    a = dict(out=P, q=P, k=P, v=P, ks=P, vs=P, tab=P, mbs=4, cu=P, past=P, b=2, t=4, most=2, hq=4,
             hkv=2, d=64, nb=16, scale=1.0, stream=None)
    a.update(kw)
    return lib.pa_prefill_int8(*a.values())


@pytest.mark.parametrize("call,kw,rc", [
    (append, dict(dtype=2), -1), (append, dict(b=-1), -1), (append, dict(t=-1), -1),
    (append, dict(most=-1), -1), (append, dict(hkv=0), -1), (append, dict(nb=0), -1),
    (append, dict(mbs=0), -1), (append, dict(d=80), -3), (append, dict(d=512), -3),
    (append, dict(q=P), -1), (append, dict(inv=P), -1), (append, dict(q=P, inv=P, hq=0), -1),
    (append, dict(k=None), -1), (append, dict(vs=None), -1), (append, dict(value=None), -1),
    (append, dict(tab=None), -1), (append, dict(cu=None), -1), (append, dict(ctx=None), -1),
    (append, dict(k=C.c_void_p(264)), -1), (append, dict(kst=127), -1), (append, dict(vst=-1), -1),
    (append, dict(q=P, inv=P, qst=255), -1), (append, dict(hkv=40000), -3),
    (append, dict(b=1 << 30), -3),
    (append, dict(b=0), 0), (append, dict(t=0), 0), (append, dict(most=0), 0),
    (decode, dict(b=-1), -1), (decode, dict(hq=5), -1), (decode, dict(hkv=0, hq=0), -1),
    (decode, dict(most=-1), -1), (decode, dict(most=65), -2), (decode, dict(d=80), -3),
    (decode, dict(q=None), -1), (decode, dict(ks=None), -1), (decode, dict(ctx=None), -1),
    (decode, dict(v=C.c_void_p(264)), -1), (decode, dict(q=C.c_void_p(258)), -1),
    (decode, dict(mbs=1 << 20, most=100000), -4),
    (decode, dict(mbs=1 << 20, most=100000, ws=P, wsb=1000), -4),
    (decode, dict(mbs=1 << 28), -2), (decode, dict(b=70000), -3),
    (decode, dict(b=0), 0), (decode, dict(most=0), 0),
    (prefill, dict(b=-1), -1), (prefill, dict(hq=5), -1), (prefill, dict(most=-1), -1),
    (prefill, dict(d=16), -3), (prefill, dict(out=None), -1), (prefill, dict(past=None), -1),
    (prefill, dict(k=C.c_void_p(264)), -1), (prefill, dict(out=C.c_void_p(260)), -1),
    (prefill, dict(b=1 << 30), -3), (prefill, dict(mbs=1 << 28), -3),
    (prefill, dict(b=0), 0), (prefill, dict(t=0), 0), (prefill, dict(most=0), 0),
])
def test_refusals(lib, call, kw, rc):
    assert call(lib, **kw) == rc
    assert (lib.pa_last_error() != b"") == (rc != 0)


def test_read_refusals(lib):
    def read(k=P, ids=1, n=16, h=2, d=64, nb=4):
        return lib.pa_read_kv_int8(k, P, P, P, P, ids, n, h, d, nb, P, P, None)

    assert read(n=17) == -2 and read(n=-1) == -1 and read(k=None) == -1 and read(nb=0) == -1
    assert read(h=70000) == -3 and read(n=0) == 0


def test_workspace_size(lib):
    size = lib.pa_decode_int8_workspace_size
    assert size(2, 4, 2, 64, 64) == 0
    assert size(0, 4, 2, 64, 64) == 0 and size(2, 5, 2, 64, 64) == 0
    parts = size(1, 32, 8, 128, 100000)
    assert parts > 0 and parts % (32 * 130 * 4) == 0


def test_kv_cache_create_rejects_bad_sizes(lib):
    h = C.c_void_p()
    assert lib.pa_kv_cache_create_int8(0, 2, 64, 4, C.byref(h)) == -1
    assert lib.pa_kv_cache_create_int8(1, 2, 64, -4, C.byref(h)) == -1
    assert lib.pa_kv_cache_create_int8(1, 2, 64, 4, None) == -1
    assert lib.pa_kv_cache_create(1, 2, 64, 4, 3, C.byref(h)) == -1  # not by its dtype
    assert not h.value
    assert lib.pa_kv_cache_key_scales_ptr(None, 0) is None


def test_wrappers_refuse(pa):
    cpu = [torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, 64, 16, dtype=torch.int8),
           torch.zeros(4, 2, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)]
    with pytest.raises(ValueError):
        pa.Int8Cache(*cpu)
    with pytest.raises(ValueError):
        pa.Int8Cache(cpu[0][:, :, :8], *cpu[1:])


def test_plain_quantisation_error():
    """A block written at once: every value within half a step, and the step at most
    2^-6 of the block's largest (127 * 2^e >= the largest > 63.5 * 2^e)."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, 3, 64)) * np.exp2(rng.uniform(-20, 20, (1, 3, 1)))
    cache = int8_plain.random_cache(rng, 2, 3, 64)
    k, v, ks, vs = int8_plain.append(cache, x, -x, [[1]], [0, 16], [16], 16)
    for got, want in ((int8_plain.values(k, ks)[1], x.transpose(1, 0, 2)),
                      (int8_plain.values(v, vs)[1], -x.transpose(1, 2, 0))):
        step = np.exp2(ks[1].astype(float) - 127)[:, None, None]
        assert np.all(np.abs(got - want) <= 0.5 * step)
        assert np.all(step <= 2.0 ** -5.98 * np.abs(want).max((1, 2), keepdims=True))
    for other, was in ((k, cache[0]), (v, cache[1]), (ks, cache[2])):
        assert np.array_equal(other[0], was[0])
