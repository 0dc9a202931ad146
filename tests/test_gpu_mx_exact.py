"""That products are exact: with all scales of a matrix equal every term is a
whole number of units, at most 128 x 12 of them by one digit of x, so up to 8192
columns every partial sum fits 24 bits and the fp32 result has to equal the
whole-number one, in every kernel and variant (the sizes of _mx_plan); up to 544
columns with scales of three neighbouring powers in either matrix, too.  A sum
that dropped bits below its largest terms, or a misplaced block, shows."""
import numpy as np
import pytest

import _mx as X
import _mx_plan as M
from qw3_amd import ds3
from qw3_amd._native import hip
from test_gpu_mx import FP4, I8, SENTINEL, group_offsets, h_of, read_mx
from test_gpu_mx_block import Block
from test_gpu_mx_sizes import sizes_of

pytestmark = pytest.mark.gpu

NIBBLES = np.float32([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12])       # twice the values
PAIRS = np.stack((np.tile(NIBBLES, 16), np.repeat(NIBBLES, 16)), 1)


def random_codes(rng, rows, nbytes):
    return np.frombuffer(rng.bytes(rows * nbytes), np.uint8).reshape(rows, nbytes).copy()


def rows_of_x(rng, rows, k):
    """MXINT8 codes; the first rows' neighbours are the largest and the smallest magnitudes."""
    q = random_codes(rng, rows, k).view(np.int8)
    edge = np.resize(np.int8([-128, 1, 127, -1, 5, -128, 3, -5]), k)
    q[0] = edge
    if rows > 2:
        q[rows // 2], q[-1] = np.roll(edge, 1), np.where(np.arange(k) % 32 == 7, -128, 1)
    return q


def weights(rng, rows, k):
    c = random_codes(rng, rows, k // 2)
    c[0], c[-1] = 0x17, 0xF1                              # 6 and .5, .5 and -6
    return c


def powers(rng, rows, k):
    """What each block's scale byte has above the lowest one."""
    assert 544 * 128 * 12 * 2 ** 4 < 2 ** 24 and 8192 * 128 * 12 < 2 ** 24
    return rng.integers(0, 3 if k <= 544 else 1, (rows, k // 32)).astype(np.uint8)


def whole(codes, p):
    """A matrix's values in halves (nibbles) or 64ths (bytes) of its lowest scale, float32."""
    v = PAIRS[codes].reshape(len(codes), -1) if codes.dtype == np.uint8 else codes.astype(np.float32)
    return v * np.repeat(np.exp2(p.astype(np.float32)), 32, axis=1)


def matrix(type_, codes, p, scale):
    return ds3.MxMatrix(ds3.Buffer.from_array(codes.view(np.uint8)), ds3.Buffer.from_array(p + np.uint8(scale)), type_,
                        len(codes), 32 * p.shape[1])


def unit(sx, sw):
    return np.float32(2.0) ** (sx + sw - 254 - 7)


def takes(kind, size):
    """The kernel that the size is meant for."""
    assert M.brief(M.plan(hip(), kind, *size)) == M.KINDS[kind][size]
    print(f"  {kind} {size}: {M.KINDS[kind][size]}", flush=True)


@pytest.mark.parametrize("size", M.DENSE)
def test_matmul(hip_ready, size):
    takes("dense", size)
    m, _, n, k = size
    rng = np.random.default_rng(m + n + k)
    x, w = (rows_of_x(rng, m, k), powers(rng, m, k)), (weights(rng, n, k), powers(rng, n, k))
    c = ds3.Buffer.from_array(np.full((m, n), SENTINEL))
    ds3.matmul_mx(matrix(I8, *x, 130), matrix(FP4, *w, 121), c)
    want = whole(*x) @ whole(*w).T
    assert np.abs(want).max() < 2 ** 24
    assert np.array_equal(c.read(np.float32, (m, n)), want * unit(130, 121))


def grouped_case(rng, size):
    """(offsets, four groups' weights that repeat)."""
    rows, groups, n, k = size
    sizes = sizes_of(rng, groups, rows)
    return group_offsets(sizes), [(weights(rng, n, k), powers(rng, n, k)) for _ in range(min(4, groups))]


def of_groups(base, groups, scale):
    return matrix(FP4, *(np.concatenate([base[g % len(base)][i] for g in range(groups)]) for i in (0, 1)), scale)


def group_products(x, base, offsets, rows, n):
    """Row r's whole-number products with its group's weights (x: the rows' own)."""
    out = np.empty((rows, n), np.float32)
    for b, w in enumerate(base):
        r = np.concatenate([np.arange(offsets[g], offsets[g + 1]) for g in range(b, len(offsets) - 1, len(base))])
        out[r] = x[r] @ whole(*w).T
    return out


@pytest.mark.parametrize("size", M.GROUPED)
def test_matmul_grouped(hip_ready, size):
    takes("grouped", size)
    rows, groups, n, k = size
    rng = np.random.default_rng(rows + n + k)
    offsets, base = grouped_case(rng, size)
    n_x = min(rows, 77)
    x, ids = (rows_of_x(rng, n_x, k), powers(rng, n_x, k)), rng.integers(0, n_x, rows).astype(np.int32)
    ids[rng.integers(0, rows, 3)] = [-1, n_x, 2 ** 31 - 1]
    ok = (ids >= 0) & (ids < n_x)
    c = ds3.Buffer.from_array(np.full((rows, n), SENTINEL))
    ds3.matmul_mx_grouped(matrix(I8, *x, 125), of_groups(base, groups, 128), ds3.Buffer.from_array(offsets), c, rows, groups,
                          ids=ds3.Buffer.from_array(ids))
    got = c.read(np.float32, (rows, n))
    want = group_products(whole(*x)[np.where(ok, ids, 0)], base, offsets, rows, n) * unit(125, 128)
    assert np.array_equal(got[ok], want[ok])
    assert (got[~ok] == SENTINEL).all()


@pytest.mark.parametrize("size", M.GATE_UP)
def test_gate_up(hip_ready, size):
    """h from exact sums: off by the roundings of silu and the product, then of the block."""
    takes("gate_up", size)
    rows, groups, n, k = size
    rng = np.random.default_rng(rows + n + k)
    offsets, gates = grouped_case(rng, size)
    ups = [(weights(rng, n, k), powers(rng, n, k)) for _ in gates]
    x = random_codes(rng, rows, k).view(np.int8), powers(rng, rows, k)
    h = ds3.MxMatrix.alloc(I8, rows, n)
    ds3.moe_gate_up_mx(matrix(I8, *x, 126), of_groups(gates, groups, 120), of_groups(ups, groups, 120),
                       ds3.Buffer.from_array(offsets), h, groups)
    g, u = (group_products(whole(*x), b, offsets, rows, n).astype(np.float64) * unit(126, 120) for b in (gates, ups))
    h64 = X.silu_mul(g, u)
    # exp, the sum, the division and the product round within 2 ulp each, and exp
    # carries the rounding of its argument: |g| 2^-23 more
    h_of(*read_mx(h), h64, (16 + np.abs(g)) * 2.0 ** -23 * np.abs(h64) + 1e-44)


def test_block_whose_waves_walk(hip_ready):
    """A block whose waves walk three tiles in both products, against its steps and 64 bits."""
    T, embd, E, k, ff = 1000, 2048, 16, 4, 1056
    assert M.brief(M.plan(hip(), "gate_up", T * k, E, ff, embd)) == (1, 8, 48, 1, 3)
    assert M.brief(M.plan(hip(), "grouped", T * k, E, embd, ff)) == (1, 4, 32, 1, 3)
    m = Block(T, embd, E, k, ff)
    one, two = m.hidden(), m.hidden()
    m.steps(one, m.buffers())
    m.block(two)
    a, b = one.read(np.float32, (T, embd)), two.read(np.float32, (T, embd))
    assert np.array_equal(a, b)
    want, err = m.reference(m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k)))
    assert (np.abs(b - want) <= err).all()
