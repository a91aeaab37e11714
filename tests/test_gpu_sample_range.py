"""pa_sample over logits whose differences leave f32's range."""
import numpy as np
import pytest
import torch

from test_gpu_sample import DEV, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 600])
@pytest.mark.parametrize("cols", [5, 9001])
def test_values_further_apart_than_the_largest_float(pa, rows, cols):
    """Logits of both signs near the ends of f32 at temperatures to match: what lies
    between them passes f32's range, their weights do not vanish."""
    rng = np.random.default_rng(rows + cols)
    x = (3.4e38 * (2 * rng.random((rows, cols)) - 1)).astype(np.float32)
    x[:, 0], x[:, -1] = 3.4e38, -3.4e38
    x[0, 1:] = -np.abs(x[0, 1:])
    x[1, :] = -3.3e38
    x[1, 0], x[1, 2], x[1, 3] = 3.3e38, -1e38, -2e38
    u = rng.random(rows).astype(np.float32)
    t = rng.choice([1e38, 5e37, 3e38, 1e37, 2e36, np.inf], rows)
    k = rng.choice([0, 2, 3, 4, cols // 2], rows)
    p = rng.choice([1.0, 0.9, 0.5], rows)
    t[1], k[1], p[1], u[1] = 3e38, 2, 1.0, 0.999
    check(pa, torch.from_numpy(x).to(DEV), u, t, k, p)
    check(pa, torch.from_numpy(x).to(DEV), u, t, k)
    check(pa, torch.from_numpy(x).to(DEV), u, t, p=p)
