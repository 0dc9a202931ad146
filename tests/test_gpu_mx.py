"""The microscaled operators on the GPU against 64-bit numpy: rounding bit for
bit, products within the bound of an fp32 sum, rows that no group owns, graphs,
and the operators one after the other as an FFN block uses them."""
import ctypes as C

import numpy as np
import pytest

import _mx as X
import _oracle as O
from qw3_amd import ds3
from qw3_amd._native import hip

pytestmark = pytest.mark.gpu

FP4, I8 = X.FP4, X.I8
SENTINEL = np.float32(-12345.5)


def read_mx(m):
    codes = m.codes.read(np.uint8, (m.rows, m.cols // 2 if m.type == FP4 else m.cols))
    return codes, m.scales.read(np.uint8, (m.rows, m.cols // 32))


def shifted(a, off):
    """A view of a's bytes that starts `off` bytes into a buffer (kept alive by the view's `parent`)."""
    a = np.ascontiguousarray(a)
    raw = np.zeros(off + a.nbytes, np.uint8)
    raw[off:] = a.reshape(-1).view(np.uint8)
    parent = ds3.Buffer.from_array(raw)
    v = parent.view(off, a.nbytes)
    v.parent = parent
    return v


def hard_rows(rng, rows, cols):
    """Normal rows of many sizes with blocks where rounding can go wrong."""
    v = rng.standard_normal((rows, cols)).astype(np.float32) * np.exp2(rng.integers(-30, 30, (rows, 1))).astype(np.float32)
    b = v.reshape(-1, 32)
    special = [np.zeros(32), np.full(32, -0.0), np.full(32, 1e-42), np.arange(32) * 2.0 ** -149,
               np.full(32, 3.4028235e38), np.r_[np.inf, np.ones(31)], np.r_[np.ones(31), np.nan], np.r_[-np.inf, np.nan, np.zeros(30)],
               np.r_[7.0, np.arange(31) / 4], np.r_[np.nextafter(np.float32(7), np.float32(8)), np.arange(31) / 4],
               np.r_[6.0, 5.0, 3.5, 2.5, 1.75, 1.25, .75, .25, -5, -3.5, -2.5, -1.75, -1.25, -.75, -.25, np.zeros(17)],
               np.r_[1.0, np.arange(1, 32) / 128], np.r_[np.float32(2) - np.float32(2) ** -23, np.arange(31) / 64 + 1 / 128],
               np.r_[2.0 ** -126, np.zeros(31)], np.r_[2.0 ** -127, 2.0 ** -130 * np.ones(31)], np.r_[2.0 ** 127, 1.0, np.zeros(30)]]
    for i, s in enumerate(special):
        if 2 * i < len(b):
            b[2 * i] = s
    return v


@pytest.mark.parametrize("to", [FP4, I8])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (40, 2048), (7, 4128)])
def test_quantize_f32(hip_ready, to, rows, cols):
    v = hard_rows(np.random.default_rng(rows), rows, cols)
    m = ds3.MxMatrix.alloc(to, rows, cols)
    print(f"  quantize f32 {rows}x{cols} to {to}", flush=True)
    ds3.mx_quantize(ds3.Buffer.from_array(v), ds3.TYPE_F32, m)
    codes, scales = read_mx(m)
    want_c, want_s = X.encode(to, v)
    assert np.array_equal(scales, want_s)
    assert np.array_equal(codes, want_c)


@pytest.mark.parametrize("to", [FP4, I8])
@pytest.mark.parametrize("t,size", [(ds3.TYPE_F32, 4), (ds3.TYPE_F16, 2)])
def test_quantize_strided_rows(hip_ready, to, t, size):
    """Rows with gaps, from addresses that take no vector loads; what lies between and behind the rows does not count."""
    rng = np.random.default_rng(5)
    rows, cols = 9, 160
    for pad, off in ((0, size), (size, 0), (16 * size, 0), (3 * size, 7 * size)):
        v = rng.standard_normal((rows, cols + pad // size)).astype(np.float32 if size == 4 else np.float16)
        v[:, cols:] = 1e4
        m = ds3.MxMatrix.alloc(to, rows, cols)
        ds3.mx_quantize(shifted(v, off), t, m, src_row_stride=(cols * size + pad))
        codes, scales = read_mx(m)
        want_c, want_s = X.encode(to, v[:, :cols].astype(np.float32))
        assert np.array_equal(scales, want_s) and np.array_equal(codes, want_c), (pad, off)


@pytest.mark.parametrize("to", [FP4, I8])
@pytest.mark.parametrize("t", [ds3.TYPE_Q8_0, ds3.TYPE_Q4_K, ds3.TYPE_Q6_K])
@pytest.mark.parametrize("rows,blocks", [(1, 8), (5, 24), (33, 64)])
def test_quantize_gguf_rows(hip_ready, to, t, rows, blocks):
    """The blocks' values as the CPU dequantiser gives them, rounded: bit for bit."""
    rng = np.random.default_rng(t + rows)
    cols, rb = 32 * blocks, ds3.row_bytes(t, 32 * blocks)
    raw = rng.integers(0, 256, (rows, rb), dtype=np.uint8)
    per, nb = ds3.BLOCK[t]
    half = rng.uniform(1e-4, 2e-3, (rows, rb // nb, 2)).astype(np.float16)
    blk = raw.reshape(rows, -1, nb)
    for i, at in enumerate({ds3.TYPE_Q8_0: (0,), ds3.TYPE_Q4_K: (0, 2), ds3.TYPE_Q6_K: (208,)}[t]):
        blk[:, :, at:at + 2] = half[:, :, i:i + 1].view(np.uint8).reshape(rows, -1, 2)
    stride = rb + (32 if t == ds3.TYPE_Q4_K else 6)
    gap = np.full((rows, stride), 0xAA, np.uint8)
    gap[:, :rb] = raw
    want = X.encode(to, O.dequantize(t, raw.reshape(-1), rows * cols).reshape(rows, cols))
    for src, st in ((raw, rb), (gap, stride)):
        m = ds3.MxMatrix.alloc(to, rows, cols)
        ds3.mx_quantize(ds3.Buffer.from_array(src), t, m, src_row_stride=st)
        codes, scales = read_mx(m)
        assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0]), st


@pytest.mark.parametrize("to", [FP4, I8])
@pytest.mark.parametrize("t", [ds3.TYPE_Q8_0, ds3.TYPE_Q4_K, ds3.TYPE_Q6_K])
def test_quantize_gguf_scales_that_are_not_finite(hip_ready, to, t):
    """Infinite and NaN block scales, also times sub-block scales of zero: the MX blocks they reach get 255."""
    rng = np.random.default_rng(t)
    rows, cols = 9, 1024
    per, nb = ds3.BLOCK[t]
    blk = rng.integers(0, 256, (rows, cols // per, nb), dtype=np.uint8)
    at = {ds3.TYPE_Q8_0: (0,), ds3.TYPE_Q4_K: (0, 2), ds3.TYPE_Q6_K: (208,)}[t]
    for i in at:
        blk[:, :, i:i + 2] = rng.uniform(1e-4, 2e-3, blk.shape[:2] + (1,)).astype(np.float16).view(np.uint8)
    if t != ds3.TYPE_Q8_0:                              # some sub-block scales of zero
        sub = slice(4, 16) if t == ds3.TYPE_Q4_K else slice(192, 208)
        blk[:, :, sub] *= rng.integers(0, 2, blk[:, :, sub].shape, dtype=np.uint8)
    for r, v in ((1, np.inf), (3, np.nan), (5, -np.inf), (7, np.inf)):
        i = at[-1] if r > 4 else at[0]
        blk[r, r % 3, i:i + 2] = np.array([v], np.float16).view(np.uint8)
    raw = blk.reshape(rows, -1)
    with np.errstate(invalid="ignore"):
        v = O.dequantize(t, raw.reshape(-1), rows * cols).reshape(rows, cols)
        want = X.encode(to, v)
    m = ds3.MxMatrix.alloc(to, rows, cols)
    ds3.mx_quantize(ds3.Buffer.from_array(raw), t, m)
    codes, scales = read_mx(m)
    bad = ~np.isfinite(v).reshape(rows, -1, 32).all(2)
    assert bad.any() and np.array_equal(scales == 255, bad)
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])


@pytest.mark.parametrize("t", [FP4, I8])
@pytest.mark.parametrize("dst,size", [(ds3.TYPE_F32, 4), (ds3.TYPE_F16, 2)])
def test_dequantize(hip_ready, t, dst, size):
    """Every code with every scale, to aligned and unaligned places."""
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], (512 if t == FP4 else 256) // 32, axis=1)
    m = X.Mat(t, codes, scales)
    dtype = np.float32 if size == 4 else np.float16
    with np.errstate(over="ignore"):
        want = m.values.astype(np.float32).astype(dtype)
    for off in (0, size):
        out = shifted(np.zeros(m.rows * m.cols, dtype), off)
        ds3.mx_dequantize(m.dev, out, dst)
        got = out.read(dtype, (m.rows, m.cols))
        assert np.array_equal(got, want, equal_nan=True), off


@pytest.mark.parametrize("n", [32, 96, 256, 288, 1024, 1056, 2048, 2080, 4096, 5120, 8192, 8224])
@pytest.mark.parametrize("rows", [1, 5])
def test_add_rms_norm(hip_ready, n, rows):
    rng = np.random.default_rng(n + rows)
    x = rng.standard_normal((rows, n)).astype(np.float32) * np.exp(rng.standard_normal((1, n))).astype(np.float32)
    d = (0.5 * rng.standard_normal((rows, n))).astype(np.float32)
    g = (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    eps = 1e-6
    print(f"  norm {rows}x{n}", flush=True)
    first = None
    for delta, keep, off, alias in ((d, True, 0, None), (d, False, 0, "x"), (d, True, 4, None), (None, True, 0, None),
                                    (d, True, 0, "delta"), (None, False, 12, None)):
        s = x + delta if delta is not None else x
        xb, gb = shifted(x, off), shifted(g, off)
        db = shifted(delta, off) if delta is not None else None
        sb = {"x": xb, "delta": db, None: ds3.Buffer.alloc(x.nbytes)}[alias] if delta is not None else None
        yb = shifted(np.zeros_like(x), off) if keep else None
        m = ds3.MxMatrix.alloc(I8, rows, n)
        ds3.add_rms_norm_mx(xb, gb, eps, m, delta=db, sum_out=sb, x_norm=yb)
        got = read_mx(m)
        if sb is not None:
            assert np.array_equal(sb.read(np.float32, x.shape), s), "the sum is one fp32 addition"
        y64 = s.astype(np.float64) / np.sqrt((s.astype(np.float64) ** 2).mean(1, keepdims=True) + eps) * g
        # A sum of n squares in any order is within n u of itself, so the root and
        # its reciprocal within n u / 2; square, mean, + eps, root, reciprocal and the
        # two products add eight roundings at most (u = 2^-24).
        bound = (n / 2 + 8) * 2.0 ** -24
        if keep:
            y = yb.read(np.float32, x.shape)
            assert (np.abs(y - y64) <= bound * np.abs(y64)).all()
            want = X.encode(I8, y)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), "the rounding of the rows written"
        if delta is not None:
            first = first or got
            assert np.array_equal(got[0], first[0]) and np.array_equal(got[1], first[1]), (off, alias)
        # half a step, a whole one where 127.5 and more saturates, and the rows' own error
        step = np.repeat(X.powers(got[1]) / 64, 32, axis=1)
        err = np.abs(X.values(I8, *got) - y64)
        top = np.abs(X.elements(I8, got[0])) * 64 == 127
        assert (err <= step * np.where(top, 1.0, 0.5) + bound * np.abs(y64)).all()


@pytest.mark.parametrize("n", [64, 1024, 2048, 8192, 8224])
def test_add_rms_norm_range(hip_ready, n):
    """Rows whose squares leave the range of 32 bits, and y within one rounding."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((6, n)) * np.r_[1e30, 3e18, 1.0, 1e-18, 1e-25, 1e-30][:, None]).astype(np.float32)
    d = (x * rng.standard_normal(x.shape)).astype(np.float32)
    g = (1 + 0.2 * rng.standard_normal(n)).astype(np.float32)
    for eps, delta in ((0.0, None), (1e-6, None), (0.0, d), (1e-6, d)):
        m, y = ds3.MxMatrix.alloc(I8, 6, n), ds3.Buffer.alloc(x.nbytes)
        ds3.add_rms_norm_mx(ds3.Buffer.from_array(x), ds3.Buffer.from_array(g), eps, m, x_norm=y,
                            delta=None if delta is None else ds3.Buffer.from_array(delta))
        x64 = x.astype(np.float64) + (0 if delta is None else delta)      # not rounded in between
        want = x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + np.float32(eps)) * g
        got = y.read(np.float32, x.shape)
        # half a step of the result, and what n additions in 64 bits may lose
        assert (np.abs(got - want) <= (2.0 ** -24 + n * 2.0 ** -52) * np.abs(want) + 2.0 ** -150).all()
        codes = X.encode(I8, got)
        assert all(np.array_equal(a, b) for a, b in zip(read_mx(m), codes))


def test_add_rms_norm_rows_of_nothing(hip_ready):
    """Rows of zeros, of infinities and of NaN: only their own outputs show them."""
    n = 512
    x = np.ones((6, n), np.float32)
    x[1] = 0
    x[2, 7] = np.inf
    x[3, 100] = np.nan
    x[4] = 1e-30
    m, y = ds3.MxMatrix.alloc(I8, 6, n), ds3.Buffer.alloc(x.nbytes)
    ds3.add_rms_norm_mx(ds3.Buffer.from_array(x), ds3.Buffer.from_array(np.ones(n, np.float32)), 0.0, m, x_norm=y)
    codes, scales = read_mx(m)
    y = y.read(np.float32, x.shape)
    want = X.encode(I8, y)
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])
    assert np.array_equal(y[0], np.ones(n)) and np.array_equal(y[5], np.ones(n))
    assert np.isnan(y[1]).all(), "0 / sqrt(0 + 0)"
    assert np.isnan(y[2, 7]) and (y[2, :7] == 0).all() and np.isnan(y[3]).all()


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 16, 128), (1, 33, 2048), (2, 17, 96), (3, 256, 512), (5, 100, 736), (15, 31, 160), (16, 64, 256),
          (17, 32, 2048), (31, 48, 1024), (33, 130, 96), (48, 257, 288), (64, 512, 512), (65, 96, 3616), (100, 255, 640),
          (128, 256, 2048), (130, 300, 1056), (257, 513, 384), (1, 5000, 4096), (700, 128, 128)]


def check(got, want, mag, k):
    bad = np.abs(got - want) > X.sum_bound(mag, k)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.max(np.abs(got - want) / (mag + 1e-300)):.3g} of the magnitudes"


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(hip_ready, m, n, k):
    rng = np.random.default_rng(m * 7919 + n)
    x, w = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, n, k)
    c = ds3.Buffer.from_array(np.full((m, n), SENTINEL))
    print(f"  matmul_mx {m}x{n}x{k}", flush=True)
    ds3.matmul_mx(x.dev, w.dev, c)
    got = c.read(np.float32, (m, n))
    check(got, *X.product(x.values, w.values), k)
    ds3.matmul_mx(x.dev, w.dev, c)
    assert np.array_equal(c.read(np.float32, (m, n)), got), "the same sums on every call"


@pytest.mark.parametrize("m,n,k", [(1, 64, 512), (40, 96, 320), (300, 256, 1024)])
def test_matmul_scales(hip_ready, m, n, k):
    """Scales far apart within a row, the lowest ones, and NaN blocks, which show in their rows and columns alone."""
    rng = np.random.default_rng(11)
    x, w = X.random_matrix(rng, I8, m, k, spread=60), X.random_matrix(rng, FP4, n, k, spread=60)
    c = ds3.Buffer.alloc(4 * m * n)
    ds3.matmul_mx(x.dev, w.dev, c)
    check(c.read(np.float32, (m, n)), *X.product(x.values, w.values), k)

    x, w = X.random_matrix(rng, I8, m, k, spread=10, centre=5), X.random_matrix(rng, FP4, n, k, spread=10, centre=250)
    w.scales = np.minimum(w.scales, 249)
    w = X.Mat(FP4, w.codes, w.scales)
    ds3.matmul_mx(x.dev, w.dev, c)
    want, mag = X.product(x.values, w.values)
    # scale bytes below 5 round x to multiples of 2^-128: half of one for each term
    slack = np.abs(w.values).sum(1)[None] * 2.0 ** -129
    got = c.read(np.float32, (m, n))
    assert (np.abs(got - want) <= X.sum_bound(mag, k) + slack).all()

    x, w = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, n, k)
    x.scales[m // 2, 1] = 255
    w.scales[n // 3, 0] = 255
    x, w = X.Mat(I8, x.codes, x.scales), X.Mat(FP4, w.codes, w.scales)
    ds3.matmul_mx(x.dev, w.dev, c)
    got = c.read(np.float32, (m, n))
    nan = np.zeros((m, n), bool)
    nan[m // 2] = nan[:, n // 3] = True
    assert np.array_equal(np.isnan(got), nan)


def test_matmul_unaligned_places(hip_ready):
    """Scales and C from any address that their elements allow."""
    rng = np.random.default_rng(3)
    for m, n, k in ((3, 40, 544), (70, 132, 512)):
        x, w = X.random_matrix(rng, I8, m, k), X.random_matrix(rng, FP4, n, k)
        for off in (1, 2, 3):
            x.dev.scales, w.dev.scales = shifted(x.scales, off), shifted(w.scales, 4 - off)
            c = shifted(np.zeros((m, n), np.float32), 4 * off)
            ds3.matmul_mx(x.dev, w.dev, c)
            check(c.read(np.float32, (m, n)), *X.product(x.values, w.values), k)


def group_offsets(sizes, first=0):
    return (first + np.r_[0, np.cumsum(sizes)]).astype(np.int32)


GROUPS = [
    # sizes, first row, rows behind the last group, n, k
    ([1], 0, 0, 48, 96),
    ([1, 0, 0, 1, 1], 0, 0, 32, 256),
    ([0, 0, 5, 0, 16, 17, 1, 0], 2, 3, 100, 160),
    ([0, 0, 0], 0, 7, 64, 128),
    ([3] * 130, 0, 1, 32, 64),
    ([40, 0, 33, 64, 65, 2], 0, 0, 96, 512),
    ([300, 1, 128, 129], 1, 2, 256, 384),
    ([2, 1] * 40 + [0] * 50 + [70], 0, 0, 64, 2048),
]


def grouped_reference(x, w, offsets, ids, n_rows, n):
    """(values, magnitudes, rows written) of a grouped product."""
    out, mag = np.zeros((n_rows, n)), np.zeros((n_rows, n))
    written = np.zeros(n_rows, bool)
    for g in range(len(offsets) - 1):
        r = np.arange(offsets[g], offsets[g + 1])
        src = ids[r] if ids is not None else r
        keep = (src >= 0) & (src < len(x))
        r, src = r[keep], src[keep]
        out[r], mag[r] = X.product(x[src], w[g * n:(g + 1) * n])
        written[r] = True
    return out, mag, written


@pytest.mark.parametrize("sizes,first,behind,n,k", GROUPS)
@pytest.mark.parametrize("gather", [False, True])
def test_matmul_grouped(hip_ready, sizes, first, behind, n, k, gather):
    rng = np.random.default_rng(len(sizes) * 31 + n)
    offsets = group_offsets(sizes, first)
    n_rows = int(offsets[-1]) + behind
    n_x = 7 if gather else n_rows
    ids = rng.integers(0, n_x, n_rows).astype(np.int32) if gather else None
    if gather and n_rows > 4:
        ids[rng.integers(0, n_rows, 3)] = [-1, n_x, 2 ** 31 - 1]
    x, w = X.random_matrix(rng, I8, n_x, k), X.random_matrix(rng, FP4, len(sizes) * n, k)
    c = ds3.Buffer.from_array(np.full((n_rows, n), SENTINEL))
    print(f"  matmul_mx_grouped {sizes[:8]} n={n} k={k}", flush=True)
    ds3.matmul_mx_grouped(x.dev, w.dev, ds3.Buffer.from_array(offsets), c, n_rows, len(sizes),
                          ids=ds3.Buffer.from_array(ids) if gather else None)
    got = c.read(np.float32, (n_rows, n))
    want, mag, written = grouped_reference(x.values, w.values, offsets, ids, n_rows, n)
    check(got[written], want[written], mag[written], k)
    assert (got[~written] == SENTINEL).all(), "rows of no group stay as they were"


def h_of(got_c, got_s, h64, rel):
    """h against the 64-bit value: half a step, a whole one at the saturated code, and the fp32 error of h."""
    step = np.repeat(X.powers(got_s) / 64, 32, axis=1)
    top = np.abs(X.elements(I8, got_c)) * 64 == 127
    err = np.abs(X.values(I8, got_c, got_s) - h64)
    assert (err <= step * np.where(top, 1.0, 0.5) + rel).all()
    amax = np.abs(h64).reshape(len(h64), h64.shape[1] // 32, 32).max(2)
    slack = rel.reshape(len(h64), h64.shape[1] // 32, 32).max(2)
    assert (X.powers(got_s) <= amax + slack).all() and (2 * X.powers(got_s) > amax - slack).all()


@pytest.mark.parametrize("sizes,first,behind,n,k", GROUPS)
def test_gate_up(hip_ready, sizes, first, behind, n, k):
    rng = np.random.default_rng(len(sizes) * 17 + n)
    n = n // 32 * 32
    offsets = group_offsets(sizes, first)
    n_rows, n_x = int(offsets[-1]) + behind, 9
    ids = rng.integers(0, n_x, n_rows).astype(np.int32)
    if n_rows > 4:
        ids[rng.integers(0, n_rows, 2)] = [-5, n_x]
    x = X.random_matrix(rng, I8, n_x, k, spread=2)
    g, u = (X.random_matrix(rng, FP4, len(sizes) * n, k, spread=2, centre=121) for _ in range(2))
    h = ds3.MxMatrix.alloc(I8, n_rows, n)
    h.codes.write(np.full((n_rows, n), 0x5A, np.uint8))
    h.scales.write(np.full((n_rows, n // 32), 0x5B, np.uint8))
    print(f"  moe_gate_up_mx {sizes[:8]} n={n} k={k}", flush=True)
    ds3.moe_gate_up_mx(x.dev, g.dev, u.dev, ds3.Buffer.from_array(offsets), h, len(sizes), ids=ds3.Buffer.from_array(ids))
    codes, scales = read_mx(h)
    gv, gm, written = grouped_reference(x.values, g.values, offsets, ids, n_rows, n)
    uv, um, _ = grouped_reference(x.values, u.values, offsets, ids, n_rows, n)
    # silu' is at most 1.1; exp, the sum, the division and the product round within
    # 2 ulp each, and exp carries the rounding of its argument: |g| 2^-23 more
    h64 = X.silu_mul(gv, uv)
    dg, du = X.sum_bound(gm, k), X.sum_bound(um, k)
    rel = 1.1 * dg * (np.abs(uv) + du) + np.abs(gv) * du + (16 + np.abs(gv)) * 2.0 ** -23 * np.abs(h64) + 1e-44
    h_of(codes[written], scales[written], h64[written], rel[written])
    assert (codes[~written] == 0x5A).all() and (scales[~written] == 0x5B).all()


def test_offsets_that_make_no_sense(hip_ready):
    """Offsets out of range or decreasing: nothing outside C and no hang (values unspecified)."""
    rng = np.random.default_rng(2)
    n, k, rows = 32, 128, 20
    x, w = X.random_matrix(rng, I8, rows, k), X.random_matrix(rng, FP4, 3 * n, k)
    for off in ([0, 2 ** 31 - 1, 5, 20], [-7, -1, 3, 90], [20, 10, 5, 0]):
        parent = ds3.Buffer.from_array(np.full((rows + 40, n), SENTINEL))
        ds3.matmul_mx_grouped(x.dev, w.dev, ds3.Buffer.from_array(np.array(off, np.int32)),
                              parent.view(20 * n * 4, rows * n * 4), rows, 3)
        got = parent.read(np.float32, (rows + 40, n))
        assert (got[:20] == SENTINEL).all() and (got[-20:] == SENTINEL).all(), off


def test_empty_calls(hip_ready):
    """No rows: nothing to do, and nothing written."""
    rng = np.random.default_rng(1)
    w = X.random_matrix(rng, FP4, 64, 64)
    x0 = ds3.MxMatrix(ds3.Buffer.alloc(16), ds3.Buffer.alloc(16), I8, 0, 64)
    c = ds3.Buffer.from_array(np.full(64, SENTINEL))
    ds3.matmul_mx(x0, w.dev, c)
    ds3.matmul_mx_grouped(x0, w.dev, ds3.Buffer.from_array(np.zeros(3, np.int32)), c, 0, 2)
    ds3.moe_gate_up_mx(x0, w.dev, w.dev, ds3.Buffer.from_array(np.zeros(3, np.int32)),
                       ds3.MxMatrix(c, c, I8, 0, 32), 2)
    ds3.mx_quantize(c, ds3.TYPE_F32, x0)
    ds3.mx_dequantize(x0, c)
    ds3.add_rms_norm_mx(c, c, 1e-6, x0)
    assert (c.read(np.float32, 64) == SENTINEL).all()
