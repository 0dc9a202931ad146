"""The microscaled operators on values at the edges of their formats."""
import numpy as np
import pytest

import _mx as X
from qw3_amd import ds3
from test_gpu_mx import FP4, I8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 2048, 8224])
def test_the_sum_without_delta_is_x(hip_ready, n):
    """Bit for bit, zeros with their signs and subnormal values too; y keeps the signs."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((3, n)).astype(np.float32)
    x[:, ::5], x[:, 1::5] = -0.0, 0.0
    x[1, 2::5] = -1e-42
    s, y, m = ds3.Buffer.alloc(x.nbytes), ds3.Buffer.alloc(x.nbytes), ds3.MxMatrix.alloc(I8, 3, n)
    ds3.add_rms_norm_mx(ds3.Buffer.from_array(x), ds3.Buffer.from_array(np.ones(n, np.float32)), 1e-6, m, sum_out=s, x_norm=y)
    assert np.array_equal(s.read(np.int32, x.shape), x.view(np.int32))
    assert np.array_equal(np.signbit(y.read(np.float32, x.shape)), np.signbit(x))
