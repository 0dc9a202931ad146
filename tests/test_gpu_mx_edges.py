"""The microscaled operators on values, places and sizes at the edges of what they take."""
import numpy as np
import pytest

from qw3_amd import ds3
from test_gpu_mx import I8, shifted
from test_gpu_mx_block import Block

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


@pytest.mark.parametrize("T", [5, 40])
def test_block_rows_that_are_not_finite(hip_ready, T):
    """A token with an infinity or a NaN gets NaN; every other token's result is the same bit for bit."""
    m = Block(T, 512, 16, 3, 96)
    clean, hard = m.hidden(), m.x.copy()
    m.block(clean)
    hard[1, 7], hard[3, 500] = np.nan, -np.inf
    h = ds3.Buffer.from_array(hard)
    m.block(h)
    idx = m.idx.read(np.int32, (T, 3))
    assert ((idx >= 0) & (idx < 16)).all()
    got, want = h.read(np.float32, m.x.shape), clean.read(np.float32, m.x.shape)
    assert np.isnan(got[[1, 3]]).all()
    rest = np.setdiff1d(np.arange(T), [1, 3])
    assert np.array_equal(got[rest], want[rest])


@pytest.mark.parametrize("T", [1, 6, 40])
def test_block_from_any_address(hip_ready, T):
    """Buffers that start on four bytes, scales on any: as from aligned ones."""
    m = Block(T, 512, 16, 3, 96)
    one = m.hidden()
    m.block(one)
    want, idx = one.read(np.float32, m.x.shape), m.idx.read(np.int32, (T, 3))
    two = shifted(m.x, 4)
    m.dev["delta"], m.dev["weight"] = shifted(m.delta, 8), shifted(m.weight, 12)
    m.idx, m.scores = shifted(np.zeros((T, 3), np.int32), 4), shifted(np.zeros((T, 3), np.float32), 4)
    for i, mat in enumerate((m.gate, m.up, m.down)):
        mat.dev.scales = shifted(mat.scales, i + 1)
    m.block(two)
    assert np.array_equal(m.idx.read(np.int32, (T, 3)), idx)
    assert np.array_equal(two.read(np.float32, m.x.shape), want)


@pytest.mark.parametrize("T,embd,E,k,ff", [(3, 256, 1, 1, 32), (1, 32, 2, 2, 32), (5, 64, 256, 16, 32), (20, 256, 2, 2, 64),
                                           (1300, 64, 256, 16, 32)])
def test_block_of_few_and_many_experts(hip_ready, T, embd, E, k, ff):
    m = Block(T, embd, E, k, ff)
    hidden = m.hidden()
    m.block(hidden)
    want, err = m.reference(m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k)))
    assert (np.abs(hidden.read(np.float32, (T, embd)) - want) <= err).all()


def test_block_with_a_read_only_router(hip_ready):
    """An imported router of another type is expanded once; a capture after that replays."""
    m = Block(24, 256, 8, 2, 64, router_type=ds3.TYPE_F16)
    one, two = m.hidden(), m.hidden()
    m.block(one)
    want = one.read(np.float32, m.x.shape)
    m.dev["router"] = ds3.Buffer.from_mmap_array(m.router.astype(np.float16))
    m.block(two)
    assert np.array_equal(two.read(np.float32, m.x.shape), want)
    with ds3.Graph() as g:
        m.block(two)
    for _ in range(3):
        two.write(m.x)
        g.launch()
        assert np.array_equal(two.read(np.float32, m.x.shape), want)
        other = m.hidden()
        m.block(other)
        assert np.array_equal(other.read(np.float32, m.x.shape), want)


def test_combine_replayed(hip_ready):
    """Captured without a call before, replayed with eager calls between."""
    rng = np.random.default_rng(3)
    y, pos = rng.standard_normal((30, 96)).astype(np.float32), rng.integers(-1, 31, (9, 4)).astype(np.int32)
    w = rng.standard_normal((9, 4)).astype(np.float32)
    old = rng.standard_normal((9, 96)).astype(np.float32)
    b = [ds3.Buffer.from_array(a) for a in (y, pos, w)]
    one, two = ds3.Buffer.from_array(old), ds3.Buffer.from_array(old)
    with ds3.Graph() as g:
        ds3.moe_combine(*b, one, 9, 4, 30, 96, True)
    ds3.moe_combine(*b, two, 9, 4, 30, 96, True)
    want = two.read(np.float32, old.shape)
    for _ in range(3):
        one.write(old)
        g.launch()
        assert np.array_equal(one.read(np.float32, old.shape), want)
        two.write(old)
        ds3.moe_combine(*b, two, 9, 4, 30, 96, True)
        assert np.array_equal(two.read(np.float32, old.shape), want)
