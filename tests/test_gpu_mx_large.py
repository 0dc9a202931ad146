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


@pytest.mark.parametrize("rows,n", [(2 ** 26 + 5, 32), (2 ** 24 + 3, 1056)])
def test_norm_of_most_rows(hip_ready, rows, n):
    """More rows than one dimension of a launch has threads for (89 GB): zero rows but for the first, some middle and
    the last ones, whose results are those of a call of their own."""
    rng = np.random.default_rng(n)
    some, eps = 7, 1e-6
    places = [0, 2 ** 20 - 3, 2 ** 22 - 3, 2 ** 23, rows - some]
    part = rng.standard_normal((some * len(places), n)).astype(np.float32)
    g = ds3.Buffer.from_array((1 + 0.2 * rng.standard_normal(n)).astype(np.float32))
    x, m = ds3.Buffer.alloc(4 * rows * n), ds3.MxMatrix.alloc(I8, rows, n)
    for i, at in enumerate(places):
        x.view(4 * at * n, 4 * some * n).write(part[i * some:(i + 1) * some])
    print(f"  norm {rows}x{n}", flush=True)
    ds3.add_rms_norm_mx(x, g, eps, m)
    own = ds3.MxMatrix.alloc(I8, len(part), n)
    ds3.add_rms_norm_mx(ds3.Buffer.from_array(part), g, eps, own)
    codes, scales = own.codes.read(np.uint8, part.shape), own.scales.read(np.uint8, (len(part), n // 32))
    assert scales.any(1).all()
    for i, at in enumerate(places):
        r = slice(i * some, (i + 1) * some)
        assert np.array_equal(m.codes.view(at * n, some * n).read(np.uint8, (some, n)), codes[r]), at
        assert np.array_equal(m.scales.view(at * (n // 32), some * (n // 32)).read(np.uint8, (some, n // 32)), scales[r]), at


def test_largest_group(hip_ready):
    """A group of nearly 2^31 rows (17 GB with their ids), and one behind it."""
    rng = np.random.default_rng(6)
    rows, n, k, n_x = 2 ** 31 - 1, 1, 32, 9
    offsets = np.array([0, rows - 5, rows], np.int32)
    x, w = X.random_matrix(rng, I8, n_x, k), X.random_matrix(rng, FP4, 2 * n, k)
    ids, c = ds3.Buffer.alloc(4 * rows), ds3.Buffer.alloc(4 * rows)      # zeroed: x's first row
    places = [0, 2 ** 29 - 3, 2 ** 30 + 77, rows - 2 ** 20, rows - 1000]
    own = rng.integers(0, n_x, (len(places), 1000)).astype(np.int32)
    for at, v in zip(places, own):
        ids.write(v, 4 * at)
    print(f"  matmul_mx_grouped {rows}x{n}x{k}", flush=True)
    ds3.matmul_mx_grouped(x.dev, w.dev, ds3.Buffer.from_array(offsets), c, rows, 2, ids=ids)
    want, mag = X.product(x.values, w.values)
    for at, v in zip(places, own):
        group = (np.arange(at, at + 1000) >= offsets[1]).astype(int)
        check(c.read(np.float32, 1000, 4 * at), want[v, group], mag[v, group], k)
    for at in (5000, 2 ** 30 - 99, rows - 2 ** 21):
        check(c.read(np.float32, 99, 4 * at), want[0, 0], mag[0, 0], k)
