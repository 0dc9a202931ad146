"""The microscaled products at sizes on both sides of every line of their
launcher: the number of 16 x 64 blocks of products, rows a group, the columns
that fit the shared memory, and few or many row tiles."""
import numpy as np
import pytest

import _mx as X
from qw3_amd import ds3
from test_gpu_mx import FP4, I8, SENTINEL, check, group_offsets, grouped_reference, h_of, read_mx

pytestmark = pytest.mark.gpu

DENSE = [(20, 4000, 128), (33, 2700, 256), (70, 4100, 1024), (70, 4100, 1056), (200, 2600, 96), (200, 2600, 3584),
         (200, 2600, 3616), (500, 1040, 7680), (500, 1040, 7712), (1000, 2100, 544), (500, 4200, 64), (1000, 2100, 3584),
         (1000, 2100, 3616), (1, 33000, 1056), (1, 33000, 1024),
         (4, 33000, 288), (5, 33000, 288), (4, 300, 1600), (5, 300, 1600), (2, 70, 96),
         (8, 33000, 288), (9, 33000, 288), (8, 300, 1600), (9, 300, 1600), (6, 2000, 2080),
         (512, 4096, 288), (3001, 1197, 96), (1500, 2200, 2560), (1500, 2200, 2592)]


@pytest.mark.parametrize("m,n,k", DENSE)
def test_matmul(hip_ready, m, n, k):
    rng = np.random.default_rng(m + 13 * n + k)
    x, w = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, n, k)
    c = ds3.Buffer.from_array(np.full((m, n), SENTINEL))
    print(f"  matmul_mx {m}x{n}x{k}", flush=True)
    ds3.matmul_mx(x.dev, w.dev, c)
    check(c.read(np.float32, (m, n)), *X.product(x.values, w.values), k)


def sizes_of(rng, groups, rows):
    """`rows` rows in `groups` groups of all sizes, some empty."""
    return np.bincount(np.minimum(rng.exponential(groups / 3, rows).astype(int), groups - 1), minlength=groups)


# groups, rows, n, k
GROUPED = [(260, 200, 224, 1056), (260, 200, 224, 1024), (300, 1000, 160, 512), (300, 1000, 160, 3616), (40, 640, 608, 1536),
           (40, 640, 608, 1568), (40, 639, 608, 320), (1024, 1024, 64, 96), (24, 900, 480, 3616), (24, 900, 480, 7712),
           (9, 3000, 320, 96), (9, 6000, 608, 96), (9, 3000, 608, 2080), (9, 2000, 608, 1056)]


@pytest.mark.parametrize("groups,rows,n,k", GROUPED)
def test_matmul_grouped(hip_ready, groups, rows, n, k):
    rng = np.random.default_rng(groups + 13 * rows + k)
    offsets = group_offsets(sizes_of(rng, groups, rows - 1), 1)
    n = n - 3
    ids = rng.integers(0, 50, rows).astype(np.int32)
    ids[rng.integers(0, rows, 4)] = [-1, 50, -2 ** 31, 2 ** 31 - 1]
    x, w = X.random_matrix(rng, I8, 50, k), X.random_matrix(rng, FP4, groups * n, k)
    c = ds3.Buffer.from_array(np.full((rows, n), SENTINEL))
    print(f"  matmul_mx_grouped {groups} groups {rows}x{n}x{k}", flush=True)
    ds3.matmul_mx_grouped(x.dev, w.dev, ds3.Buffer.from_array(offsets), c, rows, groups, ids=ds3.Buffer.from_array(ids))
    got = c.read(np.float32, (rows, n))
    want, mag, written = grouped_reference(x.values, w.values, offsets, ids, rows, n)
    check(got[written], want[written], mag[written], k)
    assert (got[~written] == SENTINEL).all(), "rows of no group stay as they were"


@pytest.mark.parametrize("groups,rows,n,k", GROUPED)
def test_gate_up(hip_ready, groups, rows, n, k):
    rng = np.random.default_rng(groups + 17 * rows + k)
    n = n // 64 * 32                        # the gate and the up rows together
    offsets = group_offsets(sizes_of(rng, groups, rows))
    x = X.random_matrix(rng, I8, rows, k, spread=2)
    g, u = (X.random_matrix(rng, FP4, groups * n, k, spread=2, centre=121) for _ in range(2))
    h = ds3.MxMatrix.alloc(I8, rows, n)
    print(f"  moe_gate_up_mx {groups} groups {rows}x{n}x{k}", flush=True)
    ds3.moe_gate_up_mx(x.dev, g.dev, u.dev, ds3.Buffer.from_array(offsets), h, groups)
    gv, gm, _ = grouped_reference(x.values, g.values, offsets, None, rows, n)
    uv, um, _ = grouped_reference(x.values, u.values, offsets, None, rows, n)
    # as in the small sizes' test
    h64 = X.silu_mul(gv, uv)
    dg, du = X.sum_bound(gm, k), X.sum_bound(um, k)
    rel = 1.1 * dg * (np.abs(uv) + du) + np.abs(gv) * du + (16 + np.abs(gv)) * 2.0 ** -23 * np.abs(h64) + 1e-44
    h_of(*read_mx(h), h64, rel)


@pytest.mark.parametrize("m,n,k", [(260, 2600, 96), (1100, 2100, 64)])
def test_scales(hip_ready, m, n, k):
    """The ends of the scales' range where the digits of x are kept in shared memory."""
    rng = np.random.default_rng(m)
    x, w = X.random_matrix(rng, I8, m, k, spread=10, centre=5), X.random_matrix(rng, FP4, n, k, spread=8, centre=244)
    x.scales[5:9, 1] = 255
    x = X.Mat(I8, x.codes, x.scales)
    c = ds3.Buffer.alloc(4 * m * n)
    ds3.matmul_mx(x.dev, w.dev, c)
    got = c.read(np.float32, (m, n))
    assert np.isnan(got[5:9]).all()
    rows = np.r_[0:5, 9:m]
    want, mag = X.product(x.values[rows], w.values)
    # scale bytes below 5 round x to multiples of 2^-128: half of one for each term
    slack = np.abs(w.values).sum(1)[None] * 2.0 ** -129
    assert (np.abs(got[rows] - want) <= X.sum_bound(mag, k) + slack).all()


def test_outputs_beyond_32_bits(hip_ready):
    """C of more than 2^32 bytes: its first, middle and last rows."""
    rng = np.random.default_rng(4)
    m, n, k = 33000, 33000, 32
    x, w = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, n, k)
    c = ds3.Buffer.alloc(4 * m * n)
    print(f"  matmul_mx {m}x{n}x{k}", flush=True)
    ds3.matmul_mx(x.dev, w.dev, c)
    for row in (0, 1, 2 ** 30 // n, 2 ** 30 // n + 1, 2 ** 31 // n, m - 2, m - 1):
        row = min(row, m - 1)
        got = c.view(4 * row * n, 4 * n).read(np.float32, (1, n))
        check(got, *X.product(x.values[row:row + 1], w.values), k)


@pytest.mark.parametrize("rows,groups", [(1, 1), (40, 1), (6, 2)])
def test_weights_beyond_32_bits(hip_ready, rows, groups):
    """More than 2^32 bytes of weights, zeros but for the first and the last rows."""
    rng = np.random.default_rng(rows)
    n, k, some = 70016 // groups, 131072, 20
    x, part = X.random_matrix(rng, I8, rows, k), X.random_matrix(rng, FP4, 2 * some, k)
    w = ds3.MxMatrix.alloc(FP4, n * groups, k)          # zeroed
    last = n * groups - some
    for at, r in ((0, slice(0, some)), (last, slice(some, None))):
        w.codes.view(at * k // 2, some * k // 2).write(part.codes[r])
        w.scales.view(at * k // 32, some * k // 32).write(part.scales[r])
    c = ds3.Buffer.alloc(4 * rows * n)
    print(f"  {rows} rows, {n * groups} x {k} weights in {groups} groups", flush=True)
    want, mag = X.product(x.values, part.values)
    if groups == 1:
        ds3.matmul_mx(x.dev, w, c)
        got = c.read(np.float32, (rows, n))
        check(got[:, :some], want[:, :some], mag[:, :some], k)
        check(got[:, -some:], want[:, some:], mag[:, some:], k)
        assert not got[:, some:-some].any()
    else:
        half = rows // 2
        ds3.matmul_mx_grouped(x.dev, w, ds3.Buffer.from_array(np.array([0, half, rows], np.int32)), c, rows, 2)
        got = c.read(np.float32, (rows, n))
        check(got[:half, :some], want[:half, :some], mag[:half, :some], k)
        check(got[half:, -some:], want[half:, some:], mag[half:, some:], k)
        assert not got[:half, some:].any() and not got[half:, :-some].any()
