"""Attention of new tokens over a paged cache against its 64-bit form."""
import numpy as np
import pytest

import _decode as D
from _decode import F16, F32
from qw3_amd import ds3

pytestmark = pytest.mark.gpu


def run(q, pages, new, lens, type_, window=0, scale=None, rows=None, pad=0, fill=3.0):
    """The operator's rows [rows][heads][dim], with `pad` values behind each row."""
    n, heads, dim = q.shape
    rows = rows or n
    wide = heads * dim + pad
    host = np.full((rows, wide), 0.5, D.NP[type_])
    host[:n, :heads * dim] = q.reshape(n, heads * dim)
    out = ds3.Buffer.from_array(np.full((rows, wide), fill, D.NP[type_]))
    offsets = np.concatenate(([0], np.cumsum(new)))
    step = wide * host.itemsize
    ds3.attention_paged(ds3.Buffer.from_array(host), pages.device(), D.ints(pages.table), D.ints(offsets), D.ints(lens), out,
                        rows, len(new), heads, pages.max_blocks, dim ** -0.5 if scale is None else scale, type_, window,
                        row_stride=step, out_row_stride=step)
    got = out.read(D.NP[type_], (rows, wide))
    assert np.all(got[:, heads * dim:] == fill) and np.all(got[n:] == fill)      # behind the rows, behind the last request
    return got[:n, :heads * dim].reshape(q.shape)


def check(seed, new, lens, heads, kv, dim, block, type_, window=0, scale=None, change=None, **more):
    rng = np.random.default_rng(seed)
    pages = D.Pages(rng, lens, block, kv, dim)
    q = (1.5 * rng.standard_normal((sum(new), heads, dim))).astype(D.NP[type_])
    if change:
        change(pages, q)
    got = run(q, pages, new, lens, type_, window, scale, **more)
    want, tol = D.attention(q, pages, new, lens, dim ** -0.5 if scale is None else scale, window, type_)
    tol = D.rounded_to(tol, want, type_)
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - want)[bad])), np.argwhere(bad)[:3].tolist())
    return got


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,block", [(32, 4, 128, 16), (4, 4, 64, 8), (7, 1, 80, 32), (6, 2, 256, 1),
                                                (16, 1, 192, 128), (3, 3, 8, 4), (20, 4, 112, 2)])
def test_one_token(hip_ready, type_, heads, kv, dim, block):
    lens = [1, 2, 31, 64, 65, 200, 7]
    check(dim, [1] * 7, lens, heads, kv, dim, block, type_)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,block", [(8, 1, 128, 16), (2, 2, 64, 64), (5, 1, 96, 8), (4, 2, 256, 32),
                                                (6, 2, 40, 1)])
def test_chunks(hip_ready, type_, heads, kv, dim, block):
    """Chunks behind cached tokens, whole prompts, single tokens and requests without tokens."""
    new = [17, 1, 0, 40, 130, 1, 0]
    lens = [60, 90, 33, 40, 131, 1, 0]
    check(dim + 1, new, lens, heads, kv, dim, block, type_)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_window(hip_ready, type_, window):
    check(window, [1, 70, 3, 1], [300, 150, 3, 64], 4, 2, 64, 16, type_, window)


@pytest.mark.parametrize("type_", [F32, F16])
def test_long_contexts(hip_ready, type_):
    """Keys split over workgroups: one stream, few streams, one of them short."""
    check(1, [1], [5000], 8, 1, 128, 16, type_)
    check(2, [1, 1, 2], [3000, 9, 4100], 4, 2, 64, 32, type_)
    check(3, [20], [2500], 2, 1, 128, 64, type_, window=2000)


@pytest.mark.parametrize("type_", [F32, F16])
def test_rows_that_see_nothing(hip_ready, type_):
    """More new tokens than length (positions below 0), and a request whose blocks all lie outside the cache."""
    def change(pages, q):
        pages.table[1] = [-1, 99, -2 ** 31, 2 ** 31 - 1][:pages.max_blocks]
    got = check(4, [6, 2, 3], [4, 20, 30], 4, 2, 64, 8, type_, change=change)
    assert not got[:2].any() and not got[6:8].any() and got[2:6].any()


@pytest.mark.parametrize("type_", [F32, F16])
def test_single_blocks_outside_the_cache(hip_ready, type_):
    def change(pages, q):
        pages.table[0, 1] = -1
        pages.table[0, 3] = pages.n_blocks
    check(5, [3, 1], [70, 90], 4, 1, 128, 16, type_, change=change)


@pytest.mark.parametrize("type_", [F32, F16])
def test_values_that_are_not_finite_where_nothing_looks(hip_ready, type_):
    """Rows behind the last position of a block and blocks of others: infinite and NaN."""
    def change(pages, q):
        n = 37
        used = pages.table[0, :3]
        junk = np.ones((pages.n_blocks, pages.block), bool)
        pos = np.arange(n)
        junk[used[pos // 16], pos % 16] = False
        for a, bad in ((pages.k, np.nan), (pages.v, np.inf)):
            a.transpose(0, 2, 1, 3)[junk] = bad
            a.transpose(0, 2, 1, 3)[junk & (np.arange(pages.block) % 2 == 0)] = -bad
    check(6, [1], [37], 4, 2, 64, 16, type_, change=change)
    check(7, [20], [37], 4, 2, 64, 16, type_, change=change)


def test_first_tokens_see_no_later_ones(hip_ready):
    """Infinities and NaN at positions that a causal row does not see leave it as it is."""
    for type_ in (F32, F16):
        rng = np.random.default_rng(8)
        pages = D.Pages(rng, [50], 16, 2, 64)
        q = rng.standard_normal((50, 4, 64)).astype(D.NP[type_])
        clean = run(q, pages, [50], [50], type_)
        for a, bad in ((pages.k, np.nan), (pages.v, np.inf)):
            a[pages.table[0, 30 // 16], :, 30 % 16] = bad
        got = run(q, pages, [50], [50], type_)
        assert np.array_equal(got[:30], clean[:30]) and not np.isfinite(got[30:]).any()


@pytest.mark.parametrize("type_", [F32, F16])
def test_extreme_scores(hip_ready, type_):
    """Large and tiny q (F32: beyond F16's range), a zero and a negative scale."""
    def large(pages, q):
        q[:, ::2] *= 1000
        if type_ == F32:
            q[:, 1] *= 1e6
            q[:, 3] *= 1e-9
    check(9, [1, 18], [60, 40], 4, 2, 64, 8, type_, change=large, scale=0.01)
    check(10, [1, 18], [60, 40], 4, 2, 64, 8, type_, scale=0.0)
    check(11, [1, 18], [60, 40], 4, 2, 64, 8, type_, scale=-0.1)


@pytest.mark.parametrize("type_", [F32, F16])
def test_padded_batch_and_strides(hip_ready, type_):
    check(12, [1, 1, 0], [30, 50, 10], 4, 2, 64, 16, type_, rows=9, pad=16)
    check(13, [30, 1], [30, 50], 4, 2, 64, 16, type_, rows=64, pad=8)


def test_offsets_that_end_before_the_rows(hip_ready):
    """A plan that was not carried out: nothing is written."""
    pages = D.Pages(np.random.default_rng(0), [20, 20], 16, 2, 64)
    for type_ in (F32, F16):
        run(np.zeros((0, 4, 64), D.NP[type_]), pages, [0, 0], [20, 20], type_, rows=5)


def test_same_result_again_and_in_a_graph(hip_ready):
    rng = np.random.default_rng(14)
    new, lens = [1, 40, 1], [700, 900, 5]
    pages = D.Pages(rng, lens, 16, 2, 128)
    cache, table, offsets, n = pages.device(), D.ints(pages.table), D.ints([0, 1, 41, 42]), D.ints(lens)
    q = rng.standard_normal((42, 8, 128)).astype(np.float32)
    qb, out = ds3.Buffer.from_array(q), ds3.Buffer.alloc(q.nbytes)

    def call():
        ds3.attention_paged(qb, cache, table, offsets, n, out, 42, 3, 8, pages.max_blocks, 0.1)
    call()
    want = out.read(np.float32, q.shape)
    call()
    assert np.array_equal(out.read(np.float32, q.shape), want)
    with ds3.Graph() as graph:
        call()
    for shift in range(3):                            # new lengths, the same graph
        lens2 = [x - 3 * shift for x in lens]
        lens2[2] = 5
        n.write(np.asarray(lens2, np.int32))
        out.zero()
        graph.launch()
        got = out.read(np.float32, q.shape)
        out.zero()
        call()
        assert np.array_equal(out.read(np.float32, q.shape), got)
    n.write(np.asarray(lens, np.int32))
    graph.launch()
    assert np.array_equal(out.read(np.float32, q.shape), want)


@pytest.mark.parametrize("type_", [F32, F16])
def test_queries_that_are_not_finite(hip_ready, type_):
    """NaN in one head's q makes that head NaN and nothing else."""
    rng = np.random.default_rng(15)
    for new, lens in (([1, 1], [40, 2000]), ([18, 2], [40, 700])):
        pages = D.Pages(rng, lens, 16, 2, 64)
        q = rng.standard_normal((sum(new), 4, 64)).astype(D.NP[type_])
        clean = run(q, pages, new, lens, type_)
        q[1, 2, 5] = np.nan
        got = run(q, pages, new, lens, type_)
        assert np.isnan(got[1, 2]).all()
        got[1, 2] = clean[1, 2]
        assert np.array_equal(got, clean)


def test_groups_that_do_not_divide_tiles(hip_ready):
    """20 heads a kv head: tiles begin inside a token; an infinity that only the later token sees."""
    for type_ in (F32, F16):
        rng = np.random.default_rng(16)
        pages = D.Pages(rng, [33, 12], 4, 1, 64)
        q = rng.standard_normal((5, 20, 64)).astype(D.NP[type_])
        clean = run(q, pages, [3, 2], [33, 12], type_)
        pages.v[pages.table[0, 8], :, 0, 7] = np.inf  # position 32, the third token's own
        got = run(q, pages, [3, 2], [33, 12], type_)
        assert np.array_equal(got[:2], clean[:2]) and not np.isfinite(got[2, :, 7]).any()
        got[2, :, 7] = clean[2, :, 7]
        assert np.array_equal(got, clean)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("n_seq", [64, 65, 300, 700])
def test_many_requests(hip_ready, type_, n_seq):
    """Requests beyond a wave's and a workgroup's, of few and many rows, some without tokens."""
    rng = np.random.default_rng(n_seq)
    new = rng.choice([0, 1, 1, 1, 2], n_seq)
    new[[3, n_seq // 2, n_seq - 1]] = 33, 70, 40
    lens = new + rng.integers(0, 40, n_seq)
    lens[n_seq // 2] = 1200
    check(n_seq, new.tolist(), lens.tolist(), 4, 1, 64, 16, type_)
    one = np.ones(n_seq, int)
    check(n_seq + 1, one.tolist(), (one + rng.integers(0, 300, n_seq) * (np.arange(n_seq) % 50 == 7)).tolist(), 2, 2, 64, 8, type_)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,block", [(2, 1, 128, 2), (2, 1, 64, 4), (2, 2, 256, 1), (1, 1, 24, 2), (3, 1, 128, 1),
                                                (2, 1, 136, 4), (1, 1, 104, 8)])
def test_chunks_of_small_blocks(hip_ready, type_, heads, kv, dim, block):
    """Blocks of fewer keys than are read at once, and the head sizes that fill no whole tile, over several steps."""
    check(dim + block, [90, 150], [90, 230], heads, kv, dim, block, type_)
    check(dim + block + 1, [100], [700], heads, kv, dim, block, type_, window=150)


@pytest.mark.parametrize("type_", [F32, F16])
def test_chunks_split_over_their_keys(hip_ready, type_):
    """Tiles of many rows whose keys are split, with blocks that lie outside the cache and rows that see nothing."""
    def change(pages, q):
        pages.table[0, 10:50] = -1
        pages.table[1, :200] = pages.n_blocks
    check(20, [40, 35], [1700, 3000], 4, 2, 64, 8, type_, change=change)
    got = check(21, [80], [60], 2, 1, 128, 16, type_)
    assert not got[:20].any() and got[20:].any()


def test_requests_that_pass_the_rows(hip_ready):
    """A request whose rows end behind n_tokens, or whose offsets fall, is left out; others are not."""
    rng = np.random.default_rng(22)
    for type_ in (F32, F16):
        pages = D.Pages(rng, [30, 40, 9, 12], 16, 2, 64)
        q = rng.standard_normal((12, 4, 64)).astype(D.NP[type_])
        want = run(q[:3], pages, [3], [30], type_)
        out = ds3.Buffer.from_array(np.full(q.shape, 7, D.NP[type_]))
        ds3.attention_paged(ds3.Buffer.from_array(q), pages.device(), D.ints(pages.table), D.ints([0, 3, 13, 2, -1]),
                            D.ints([30, 40, 9, 12]), out, 12, 4, 4, pages.max_blocks, 64 ** -0.5, type_)
        got = out.read(D.NP[type_], q.shape)
        assert np.array_equal(got[:3], want) and np.all(got[3:] == 7)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,new,lens,window", [
    (4, 2, 64, [100], [130], 40), (8, 1, 128, [90], [1500], 700), (4, 1, 256, [70], [300], 33),       # tiles of many rows
    (4, 2, 64, [7], [60], 5), (16, 1, 128, [2], [1300], 600), (6, 2, 80, [9, 20], [40, 900], 16)])    # of few
def test_window_over_values_that_are_not_finite(hip_ready, type_, heads, kv, dim, new, lens, window):
    """Rows whose window does not reach a NaN key and an infinite value are what they are without them."""
    rng = np.random.default_rng(dim + window)
    pages = D.Pages(rng, lens, 8, kv, dim)
    q = rng.standard_normal((sum(new), heads, dim)).astype(D.NP[type_])
    want, tol = D.attention(q, pages, new, lens, dim ** -0.5, window, type_)
    tol = D.rounded_to(tol, want, type_)
    at = [n - m + m // 2 - window // 2 for m, n in zip(new, lens)]               # half of the rows see it
    for i, p in enumerate(at):
        pages.k[pages.table[i, p // 8], :, p % 8, 1] = np.nan
        pages.v[pages.table[i, p // 8], :, p % 8] = np.inf
    got = run(q, pages, new, lens, type_, window)
    pos = np.concatenate([np.arange(n - m, n) for m, n in zip(new, lens)])
    bad = np.repeat(at, new)
    sees = (bad <= pos) & (bad > pos - window)
    assert sees.any() and not np.isfinite(got[sees]).any()
    assert (np.abs(got[~sees].astype(np.float64) - want[~sees]) <= tol[~sees]).all()


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("heads,kv,dim,block", [(2, 2, 64, 16), (4, 1, 128, 16), (16, 1, 64, 2), (32, 2, 256, 1), (6, 1, 40, 8)])
@pytest.mark.parametrize("new,lens,window", [([1], [1000], 100), ([1], [3000], 2050), ([1] * 3, [40, 70, 500], 33),
                                             ([1] * 70, [90] * 70, 5), ([2], [75], 1), ([3], [400], 70)])
def test_values_just_before_a_window(hip_ready, type_, heads, kv, dim, block, new, lens, window):
    """NaN and infinities at the keys before each request's first one that is seen leave every row as it is."""
    rng = np.random.default_rng(dim + window)
    pages = D.Pages(rng, lens, block, kv, dim)
    q = rng.standard_normal((sum(new), heads, dim)).astype(D.NP[type_])
    want, tol = D.attention(q, pages, new, lens, dim ** -0.5, window, type_)
    for i, (m, n) in enumerate(zip(new, lens)):
        first = n - m - window + 1                    # of the first new token; later ones see less
        for p in {first - 1, first & ~31, max(first - 17, 0)}:
            if 0 <= p < first:
                at = pages.table[i, p // block], slice(None), p % block
                pages.k[at], pages.v[at] = np.nan, [np.inf, -np.inf, np.nan][i % 3]
    got = run(q, pages, new, lens, type_, window)
    assert np.isfinite(got).all()
    assert (np.abs(got.astype(np.float64) - want) <= D.rounded_to(tol, want, type_)).all()


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("short,n", [(0, 2 ** 31 - 2 ** 16), (0, 2 ** 30 + 5), (1, 2 ** 31 - 2 ** 16 - 3), (70, 2 ** 31 - 2 ** 22 + 7)])
def test_lengths_near_2_31(hip_ready, type_, short, n):
    """One request of nearly 2^31 keys, its blocks shared, beside short ones.  k is 0, so every key has the same weight, a
    power of two; v is 1 in one block and 3 in the other.  Sums of a run are whole multiples of that weight below 2^24,
    so only those over at most 512 runs round, and the quotient: 520 half steps of 2^-24."""
    block, dim = 1 << 16, 8
    rng = np.random.default_rng(short)
    lens = [n] + [5] * short
    of = rng.integers(0, 2, 0x7fff).astype(np.int32)
    pages = D.Pages(rng, [1], 1, 1, dim)
    pages.block, pages.n_blocks, pages.max_blocks = block, 2, 0x7fff
    pages.k, pages.v = np.zeros((2, 1, block, dim), np.float16), np.ones((2, 1, block, dim), np.float16)
    pages.v[1] = 3
    pages.table = np.zeros((len(lens), 0x7fff), np.int32)
    pages.table[0], pages.table[1:, 0] = of, 1
    q = rng.standard_normal((len(lens), 1, dim)).astype(D.NP[type_])
    got = run(q, pages, [1] * len(lens), lens, type_)
    keys = np.minimum(np.maximum(n - block * np.arange(0x7fff), 0), block)      # of each block
    want = float((keys * (1 + 2 * of.astype(np.int64))).sum()) / n
    assert np.abs(got[0].astype(np.float64) - want).max() <= want * (520 * 2.0 ** -24 + D.HALF_STEP[type_])
    assert np.all(got[1:] == 3)


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("new,lens,window", [([1, 1], [60, 700], 0), ([1], [50], 20), ([20, 40], [33, 300], 0), ([70], [100], 30)])
def test_scales_and_queries_at_the_ends_of_their_range(hip_ready, type_, new, lens, window):
    """Scales that are no normal numbers, q next to them, and products of a tiny q with a large scale: masked keys stay
    masked, and scores of 0 stay 0."""
    def times(f):
        def change(pages, q):
            q[...] = q.astype(np.float64) * f
        return change

    def zero(pages, q):
        pages.k[...] = 0
        if type_ == F32:
            q *= 1e30
    cases = [(1e-42, None), (-1e-45, None), (2.0 ** 127, zero), (-1e30, zero)]
    if type_ == F32:
        cases += [(1e-4, times(2e-38)), (1e-4, times(1e-40)), (1e-42, times(1e-40)), (1e-44, times(1e30)), (0.1, times(0)),
                  (1e38, times(1e-38)), (1e37, times(1e-37)), (1e38, times(0))]
    for i, (scale, change) in enumerate(cases):
        check(100 + i, new, lens, 4, 2, 64, 8, type_, window, scale=scale, change=change)
