"""The microscaled operators at the ends of their sizes: rows, columns and
groups near 2^31, where 32-bit sums and a launch's grid reach their limits."""
import numpy as np
import pytest

import _mx as X
from qw3_amd import ds3
from test_gpu_mx import FP4, I8, check

pytestmark = pytest.mark.gpu

SOME = 20


def rows_at(w, places, part):
    """SOME rows of `part` at each of `places` of the zeroed matrix w."""
    for i, at in enumerate(places):
        r = slice(i * SOME, (i + 1) * SOME)
        w.codes.view(at * part.codes.shape[1], part.codes[r].nbytes).write(part.codes[r])
        w.scales.view(at * part.scales.shape[1], part.scales[r].nbytes).write(part.scales[r])


@pytest.mark.parametrize("m,n", [(9, 2 ** 31 - 60), (1, 2 ** 31 - 1)])
def test_most_columns(hip_ready, m, n):
    """N up to 2^31 - 1 (118 GB with nine rows): zero weights but for the first, some middle and the last rows."""
    k = 32
    rng = np.random.default_rng(m)
    places = [0, 2 ** 30 - 7, n - SOME]
    x, part = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, SOME * len(places), k)
    w, c = ds3.MxMatrix.alloc(FP4, n, k), ds3.Buffer.alloc(4 * m * n)
    rows_at(w, places, part)
    print(f"  matmul_mx {m}x{n}x{k}", flush=True)
    ds3.matmul_mx(x.dev, w, c)
    want, mag = X.product(x.values, part.values)
    for row in range(m):
        for i, at in enumerate(places):
            got = c.view(4 * (row * n + at), 4 * SOME).read(np.float32, SOME)
            cols = slice(i * SOME, (i + 1) * SOME)
            check(got, want[row, cols], mag[row, cols], k)
