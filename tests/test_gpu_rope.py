"""Rotary positions and the writing of new tokens' k and v against 64-bit forms."""
import numpy as np
import pytest

import _decode as D
from _decode import F16, F32
from qw3_amd import ds3

pytestmark = pytest.mark.gpu

TABLES = {
    "plain": (1e6, ds3.ROPE_PLAIN),
    "linear": (1e4, ds3.ROPE_LINEAR, 4.0),
    "wavelength": (5e5, ds3.ROPE_WAVELENGTH, 8.0, 1.0, 4.0, 8192),
    "yarn": (1e6, ds3.ROPE_YARN, 4.0, 1.0, 32.0, 32768),
}


def check(got, want, tol, type_):
    tol = D.rounded_to(tol, want, type_)
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want)[bad].max()))


@pytest.mark.parametrize("tokens,heads,dim,rotary,types,inter,norm,name", [
    (1, 32, 128, 128, (F32, F32), False, True, "plain"),
    (3, 4, 128, 128, (F32, F16), True, False, "linear"),
    (7, 5, 64, 32, (F16, F16), False, True, "yarn"),
    (130, 3, 96, 24, (F16, F32), True, True, "wavelength"),
    (33, 1, 80, 20, (F32, F32), False, True, "yarn"),
    (33, 2, 80, 20, (F16, F16), True, False, "plain"),
    (5, 2, 256, 254, (F32, F32), False, True, "plain"),
    (5, 2, 512, 510, (F32, F16), True, True, "linear"),
    (9, 3, 512, 512, (F16, F16), False, False, "plain"),
    (2, 7, 8, 2, (F32, F32), False, True, "plain"),
    (2, 7, 8, 8, (F16, F32), True, True, "plain"),
    (2, 3, 24, 6, (F32, F32), True, False, "yarn"),
    (2500, 16, 64, 64, (F32, F32), False, True, "yarn"),          # several heads a group of lanes
    (900, 20, 192, 96, (F16, F16), True, True, "plain"),
])
def test_rope(hip_ready, tokens, heads, dim, rotary, types, inter, norm, name):
    rng = np.random.default_rng(tokens * 1000 + dim)
    x = (rng.standard_normal((tokens, heads, dim)) * np.exp(rng.standard_normal(dim))).astype(D.NP[types[0]])
    pos = np.exp(rng.uniform(0, np.log(1 << 20), tokens)).astype(np.int32)
    pos[0], pos[-1] = 0, -5
    if tokens > 2:
        pos[1] = 2 ** 31 - 1
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None
    table = ds3.rope_table(rotary, *TABLES[name])
    theta, m = D.frequencies(rotary, *TABLES[name])
    held = table.read(np.float64, rotary // 2 + 1)
    assert np.allclose(held[:-1] * 2 * np.pi, theta, rtol=1e-14, atol=0) and held[-1] == pytest.approx(m, rel=1e-15)
    out = ds3.Buffer.alloc(tokens * heads * dim * 4)
    ds3.rope(ds3.Buffer.from_array(x), D.ints(pos), table, out, tokens, heads, dim, rotary, types[0], types[1],
             norm=None if w is None else D.floats(w), interleaved=inter)
    got = out.read(D.NP[types[1]], x.shape)
    want, tol = D.rope(x, pos, theta, m, w, interleaved=inter)
    check(got, want, tol, types[1])


def test_rope_strided_and_in_place(hip_ready):
    rng = np.random.default_rng(3)
    tokens, heads, dim, wide = 11, 3, 64, 5 * 64
    packed = rng.standard_normal((tokens, wide)).astype(np.float32)
    pos = rng.integers(0, 5000, tokens).astype(np.int32)
    table, (theta, m) = ds3.rope_table(64, 1e4), D.frequencies(64, 1e4)
    buf = ds3.Buffer.from_array(packed)
    part = buf.view(64 * 4, packed.nbytes - 64 * 4)
    span = (tokens - 1) * wide * 4 + heads * dim * 4
    out = ds3.Buffer.from_array(np.full((tokens, heads * dim + 16), 7, np.float32))
    ds3.rope(part.view(0, span), D.ints(pos), table, out, tokens, heads, dim, row_stride=wide * 4,
             out_row_stride=(heads * dim + 16) * 4)
    want, tol = D.rope(packed[:, 64:256].reshape(tokens, heads, dim), pos, theta, m)
    got = out.read(np.float32, (tokens, heads * dim + 16))
    check(got[:, :heads * dim].reshape(want.shape), want, tol, F32)
    assert np.all(got[:, heads * dim:] == 7)
    ds3.rope(part, D.ints(pos), table, part, tokens, heads, dim, row_stride=wide * 4, out_row_stride=wide * 4)
    after = buf.read(np.float32, packed.shape)
    assert np.array_equal(after[:, 64:256], got[:, :heads * dim])
    assert np.array_equal(after[:, :64], packed[:, :64]) and np.array_equal(after[:, 256:], packed[:, 256:])


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,types,inter,norm,block", [
    (1, 32, 4, 128, 128, (F32, F32), False, True, 16),
    (8, 32, 4, 128, 128, (F32, F16), False, True, 16),
    (37, 6, 2, 80, 40, (F16, F16), True, True, 1),
    (37, 6, 6, 64, 20, (F16, F32), False, False, 8),
    (700, 4, 1, 256, 256, (F32, F32), True, True, 128),
    (1500, 32, 4, 128, 64, (F32, F16), False, True, 64),
    (5, 1, 1, 24, 6, (F32, F32), False, True, 2),
])
def test_append(hip_ready, tokens, heads, kv, dim, rotary, types, inter, norm, block):
    rng = np.random.default_rng(tokens + dim)
    n_blocks = tokens // block + 5
    t_in = D.NP[types[0]]
    wide = (heads + 2 * kv) * dim + 8
    packed = rng.standard_normal((tokens, wide)).astype(t_in)
    cut = np.cumsum([0, heads * dim, kv * dim, kv * dim])
    q, k, v = (packed[:, cut[i]:cut[i + 1]].reshape(tokens, -1, dim) for i in range(3))
    pos = rng.integers(0, 100000, tokens).astype(np.int32)
    slots = rng.permutation(n_blocks * block)[:tokens].astype(np.int32)
    slots[tokens // 2::5] = -1
    if tokens > 3:
        slots[3] = n_blocks * block                   # past the cache
    wq, wk = ((1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in range(2))
    theta, m = D.frequencies(rotary, *TABLES["yarn"])
    shape = (n_blocks, kv, block, dim)
    old_k, old_v = rng.standard_normal(shape).astype(np.float16), rng.standard_normal(shape).astype(np.float16)
    cache = ds3.KvCache(ds3.Buffer.from_array(old_k), ds3.Buffer.from_array(old_v), n_blocks, block, kv, dim)
    buf, size, step = ds3.Buffer.from_array(packed), packed.itemsize, packed.itemsize * wide
    views = [buf.view(int(cut[i]) * size, (tokens - 1) * step + int(cut[i + 1] - cut[i]) * size) for i in range(3)]
    out = ds3.Buffer.alloc(tokens * heads * dim * 4)
    some = lambda w: None if w is None else D.floats(w)                          # noqa: E731
    ds3.rope_append(*views, D.ints(pos), D.ints(slots), cache, out, tokens, heads, types[0], types[1],
                    table=ds3.rope_table(rotary, *TABLES["yarn"]), rotary_dim=rotary, q_norm=some(wq), k_norm=some(wk),
                    interleaved=inter, strides=(step,) * 3)
    want, tol = D.rope(q, pos, theta, m, wq, interleaved=inter)
    check(out.read(D.NP[types[1]], want.shape), want, tol, types[1])
    live = (slots >= 0) & (slots < n_blocks * block)
    b, r = slots[live] // block, slots[live] % block
    got_k, got_v = cache.k.read(np.float16, shape), cache.v.read(np.float16, shape)
    want, tol = D.rope(k, pos, theta, m, wk, interleaved=inter)
    check(got_k[b, :, r], want[live], tol[live], F16)
    assert np.array_equal(got_v[b, :, r], v[live].astype(np.float16))
    rest = np.ones((n_blocks, block), bool)
    rest[b, r] = False
    keep = np.broadcast_to(rest[:, None], (n_blocks, kv, block))
    assert np.array_equal(got_k[keep], old_k[keep]) and np.array_equal(got_v[keep], old_v[keep])


def test_append_without_q_or_table(hip_ready):
    rng = np.random.default_rng(9)
    k, v = rng.standard_normal((2, 6, 2, 64)).astype(np.float32)
    k[0, 0, 0], v[1, 1, 1], v[2, 0, 5] = 1e6, -1e6, np.nan                       # beyond float16, and NaN
    cache = ds3.KvCache.alloc(3, 4, 2, 64)
    slots = np.array([11, 0, 5, 6, 7, 2], np.int32)
    ds3.rope_append(None, ds3.Buffer.from_array(k), ds3.Buffer.from_array(v), None, D.ints(slots), cache, None, 6, 0)
    with np.errstate(over="ignore"):
        for buf, x in ((cache.k, k), (cache.v, v)):
            got = buf.read(np.float16, (3, 2, 4, 64))
            assert np.array_equal(got[slots // 4, :, slots % 4], x.astype(np.float16), equal_nan=True)
            got[slots // 4, :, slots % 4] = 0
            assert not got.any()


def test_no_tokens(hip_ready):
    table, b = ds3.rope_table(8, 1e4), ds3.Buffer.alloc(64)
    ds3.rope(b, D.ints([0]), table, ds3.Buffer.alloc(64), 0, 1, 8)
    ds3.rope_append(None, b, b, None, D.ints([0]), ds3.KvCache.alloc(1, 1, 1, 8), None, 0, 0)


@pytest.mark.parametrize("tokens,heads,dim,rotary", [(301, 1, 8, 8), (301, 1, 8, 6), (1025, 2, 16, 2), (77, 1, 512, 510),
                                                     (77, 3, 512, 508), (40, 20, 264, 264), (600, 1, 40, 20), (3, 130, 64, 60)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_of_tokens_that_share_a_workgroup(hip_ready, tokens, heads, dim, rotary, inter):
    """Many tokens of few lanes, few of many, more groups of lanes than a workgroup's a token."""
    rng = np.random.default_rng(tokens + dim + rotary)
    x = rng.standard_normal((tokens, heads, dim)).astype(np.float32)
    pos = rng.integers(0, 1 << 17, tokens).astype(np.int32)
    theta, m = D.frequencies(rotary, *TABLES["linear"])
    out = ds3.Buffer.alloc(x.nbytes)
    ds3.rope(ds3.Buffer.from_array(x), D.ints(pos), ds3.rope_table(rotary, *TABLES["linear"]), out, tokens, heads, dim, rotary,
             interleaved=inter)
    want, tol = D.rope(x, pos, theta, m, interleaved=inter)
    check(out.read(np.float32, x.shape), want, tol, F32)


def test_append_in_place(hip_ready):
    """q_out may be q itself."""
    rng = np.random.default_rng(10)
    for tokens in (1, 70):
        q, k = rng.standard_normal((tokens, 6, 64)).astype(np.float32), rng.standard_normal((tokens, 2, 64)).astype(np.float32)
        cache, table = ds3.KvCache.alloc(20, 4, 2, 64), ds3.rope_table(48, 1e4)
        pos, slots, kb = D.ints(rng.integers(0, 9999, tokens)), D.ints(rng.permutation(80)[:tokens]), ds3.Buffer.from_array(k)
        same, out = ds3.Buffer.from_array(q), ds3.Buffer.alloc(q.nbytes)
        for b in (out, same):
            ds3.rope_append(ds3.Buffer.from_array(q) if b is out else b, kb, kb, pos, slots, cache, b, tokens, 6, table=table,
                            rotary_dim=48, q_norm=D.floats(np.linspace(0.5, 1.5, 64)))
        assert np.array_equal(same.read(np.float32, q.shape), out.read(np.float32, q.shape))
