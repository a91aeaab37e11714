"""The rule that picks pa_linear_mx's kernel and tiling, on the CPU: the shapes
with which the GPU tests reach each of them do so."""
import os
import shutil
import subprocess

import pytest
from test_gpu_mx import KERNELS, KERNELS_GATED

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TILED = {"64x64", "128x64", "128x128", "128x128 pair", "256x128", "256x256"}


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("mx") / "mx_tiling")
    subprocess.run([gxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "vllm-lite_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "mx_tiling.cpp"), "-o", exe],
                   check=True)

    def run(m, n, k, silu):
        r = subprocess.run([exe], input=f"{m} {n} {k} {int(silu)}", check=True,
                           capture_output=True, text=True)
        return r.stdout.strip()
    return run


def test_kernels_of_the_gpu_tests(choose):
    for (m, n, k), name in KERNELS.items():
        assert choose(m, n, k, False) == name, (m, n, k)
    for (m, n, k), name in KERNELS_GATED.items():
        assert choose(m, n, k, True) == name, (m, n, k)
    assert set(KERNELS.values()) == TILED | {"64x32", "few rows 1/8", "few rows 2/4"}
    assert set(KERNELS_GATED.values()) == TILED | {"few rows 2/4", "few rows 2/2"}
    # one, two and four tiles of X rows (SwiGLU: one and two)
    assert {(v, (m > 16) + (m > 32)) for (m, _, _), v in KERNELS.items() if "few" in v} == {
        (f"few rows {k}", t) for k in ("1/8", "2/4") for t in (0, 1, 2)}
    assert {(v, int(m > 16)) for (m, _, _), v in KERNELS_GATED.items() if "few" in v} == {
        ("few rows 2/4", 0), ("few rows 2/2", 0), ("few rows 2/2", 1)}


def test_largest_sizes(choose):
    """Sizes whose products pass 32 bits."""
    assert choose(2 ** 31 - 1, 2 ** 24, 4096, False) in TILED | {"64x32"}
    assert choose(2 ** 31 - 1, 2 ** 24, 2 ** 22, True) in TILED
