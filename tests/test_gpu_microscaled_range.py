"""Microscaled operators at the ends of the value range, against float64. Tolerances are test_gpu_microscaled.py's."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ancha_b200 import microscaled as mx  # noqa: E402
from oracle import microscaled as O  # noqa: E402
from test_gpu_microscaled import FORMATS, check_near, f64, poisoned_memory, rows_of  # noqa: E402,F401


# ---------------------------------------------------------------------------------------- norm

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [1, 320, 600, 1500, 4000, 8192, 20001])
def test_norm_of_zero_and_extreme_rows_with_any_eps(fmt, dim):
    """Rows of zeros are zeros whatever eps is; rows of subnormal numbers and of numbers next to f32's largest have
    the norm of any other row."""
    x = rows_of(6, dim, torch.float32, seed=dim, spread=0)
    x[0] = 0
    x[1] *= 1e-44
    x[2] *= 1e-40
    x[3] *= 1e-30
    x[4] = torch.clamp(x[4], -3, 3) * 1e38
    for eps in (1e-30, 1e-76, 1e-78, 1e-100, 1e-300, 5e-324):
        y = O.rms_norm(f64(x), 1.0, eps)
        q, _ = mx.add_rms_norm(x, None, None, eps, fmt)
        assert not f64(mx.dequantize(q))[0].any()
        check_near(q, y, 4 * 2.0 ** -24 * np.abs(y))
