"""pa_decode_int8's workspace without a GPU: a size does for its own launch and for
whatever is smaller."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADS = [(32, 8, 128), (14, 2, 64), (24, 4, 96), (16, 8, 256), (34, 2, 192), (1, 1, 32),
         (600, 300, 64), (20, 1, 32), (8, 8, 256), (130, 130, 64)]
SEQS = [1, 2, 3, 4, 5, 7, 8, 9, 11, 16, 19, 20, 21, 33, 64, 80, 100, 159, 160, 161, 300, 1000]
CTX = sorted({n + d for n in (64, 768, 1344, 2688, 4032, 4096, 4704, 5000, 8192, 20000, 100000)
              for d in (-1, 0, 1, 64, 100)} | set(range(700, 6200, 37)))


@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_sizes_grow_with_both(pa, hq, hkv, d):
    size = pa._lib.load().pa_decode_int8_workspace_size
    fewer = None  # of fewer sequences, by context
    for b in SEQS:
        of = [size(b, hq, hkv, d, n) for n in CTX]
        assert of == sorted(of)
        assert fewer is None or all(x >= y for x, y in zip(of, fewer))
        fewer = of


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("decode") / "int8_plan")
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "vllm-lite_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "int8_plan.cpp"), "-o", exe], check=True)

    def run(rows):
        r = subprocess.run([exe], input="\n".join(" ".join(map(str, x)) for x in rows), check=True,
                           capture_output=True, text=True)
        return [tuple(map(int, x.split())) for x in r.stdout.splitlines()]
    return run


@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_a_size_does_for_its_launch(pa, plans, hq, hkv, d):
    size = pa._lib.load().pa_decode_int8_workspace_size
    rows = [(b, hq, hkv, d, n) for b in SEQS for n in CTX]
    several = 0
    for x, (_, length, parts, most) in zip(rows, plans(rows)):
        b, n = x[0], x[4]
        assert length % 64 == 0 and (parts - 1) * length < n <= parts * length
        assert parts == 1 or b * parts <= most, x
        assert size(*x) == most * hq * (d + 2) * 4
        several += parts > 1
    assert several > 0
