"""pa_sample without a GPU: its refusals, and the plain form of its definition."""
import ctypes as C

import numpy as np
import pytest
import torch

import sample_plain

P = C.c_void_p(256)


@pytest.fixture(scope="module")
def lib(pa):
    return pa._lib.load()


def call(lib, **kw):
    a = dict(out=P, x=P, u=P, t=None, k=None, p=None, m=None, rows=2, cols=100, stride=0, ws=P,
             wsb=1 << 30, dtype=1, stream=None)
    a.update(kw)
    return lib.pa_sample(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=2), -1), (dict(rows=-1), -1), (dict(cols=0), -1), (dict(cols=-4), -1),
    (dict(stride=99), -1), (dict(stride=-100), -1), (dict(cols=(1 << 22) + 1), -3),
    (dict(rows=65536), -3), (dict(out=None), -1), (dict(x=None), -1), (dict(u=None), -1),
    (dict(x=C.c_void_p(257)), -1), (dict(dtype=0, x=C.c_void_p(258)), -1), (dict(ws=None), -4),
    (dict(wsb=100), -4), (dict(ws=C.c_void_p(264)), -4), (dict(rows=0), 0),
])
def test_refusals(lib, kw, rc):
    assert call(lib, **kw) == rc
    assert (lib.pa_last_error() != b"") == (rc != 0)


def test_workspace_size(lib):
    size = lib.pa_sample_workspace_size
    assert size(0) == 0 and size(-3) == 0 and size(1) > 0 and size(7) == 7 * size(1)
    assert call(lib, rows=3, wsb=size(3) - 1) == -4
    # many rows take a workgroup each
    assert size(511) > 0 and size(512) == size(65535) == 0


def test_wrapper_refuses_host_tensors(pa):
    with pytest.raises(ValueError):
        pa.sample(torch.zeros(2, 10), torch.zeros(2))


def test_plain_definition():
    x = np.log([0.4, 0.1, 0.3, 0.1, 0.1])
    assert list(sample_plain.kept(x, 1, 3, 1.0, 0)[0]) == [0, 1, 2]  # the first of three equal
    assert list(sample_plain.kept(x, 1, 0, 0.75, 0)[0]) == [0, 1, 2]
    assert list(sample_plain.kept(x, 1, 0, 0.65, 0)[0]) == [0, 2]
    assert list(sample_plain.kept(x, 1, 2, 0.5, 0)[0]) == [0]  # 0.4 of 0.7
    assert list(sample_plain.kept(x, 1, 0, 1.0, 0.5)[0]) == [0, 2]
    assert [sample_plain.draw(x, u) for u in (0, 0.39, 0.41, 0.51, 0.79, 0.81, 0.999)] == \
        [0, 0, 1, 2, 2, 3, 4]
    assert sample_plain.draw(x, 0.9, t=0.0) == 0
    assert sample_plain.draw([-np.inf, np.nan], 0.9) == 0
