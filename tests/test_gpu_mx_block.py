"""The microscaled operators one after the other, as an FFN block uses them:
against 64-bit numpy step by step, the whole block in one call against the
same steps, in batch mode and in graphs that are replayed."""
import numpy as np
import pytest

import _mx as X
from qw3_amd import ds3
from test_gpu_mx import FP4, I8, read_mx

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.mark.parametrize("n_tokens,k,n_rows,n", [(1, 1, 1, 1), (3, 8, 24, 64), (5, 2, 7, 33), (40, 16, 90, 2048), (70, 9, 300, 100),
                                                 (70000, 2, 50, 4), (65536, 1, 9, 3)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_combine(hip_ready, n_tokens, k, n_rows, n, accumulate):
    rng = np.random.default_rng(n_tokens + k)
    y = rng.standard_normal((n_rows, n)).astype(np.float32)
    slots = rng.integers(0, n_rows, (n_tokens, k)).astype(np.int32)
    out = [-1, n_rows, -2 ** 31, 2 ** 31 - 1]
    slots.reshape(-1)[rng.integers(0, slots.size, 4)] = out if slots.size > 4 else slots.reshape(-1)[0]
    scores = rng.standard_normal((n_tokens, k)).astype(np.float32)
    old = rng.standard_normal((n_tokens, n)).astype(np.float32)
    c = ds3.Buffer.from_array(old)
    ds3.moe_combine(ds3.Buffer.from_array(y), ds3.Buffer.from_array(slots), ds3.Buffer.from_array(scores), c, n_tokens, k,
                    n_rows, n, accumulate)
    got = c.read(np.float32, old.shape)
    want, mag = old * np.float64(accumulate), np.abs(old) * np.float64(accumulate)
    for j in range(k):
        ok = (slots[:, j] >= 0) & (slots[:, j] < n_rows)
        t = np.where(ok[:, None], scores[:, j, None].astype(np.float64) * y[np.where(ok, slots[:, j], 0)], 0)
        want, mag = want + t, mag + np.abs(t)
    # a product and a sum a slot, each rounded once
    assert (np.abs(got - want) <= (2 * k + 1) * 2.0 ** -24 * mag).all()


class Block:
    def __init__(self, T, embd, E, k, ff, router_type=ds3.TYPE_F32, seed=0):
        rng = np.random.default_rng(seed + T + embd)
        self.T, self.embd, self.E, self.k, self.ff, self.router_type = T, embd, E, k, ff, router_type
        self.x, self.delta = (rng.standard_normal((T, embd)).astype(np.float32) for _ in range(2))
        self.weight = (1 + rng.standard_normal(embd) / 8).astype(np.float32)
        self.router = (rng.standard_normal((E, embd)) / np.sqrt(embd)).astype(np.float32)
        centre = 127 - int(np.log2(embd) / 2) - 1
        self.gate, self.up = (X.random_matrix(rng, FP4, E * ff, embd, spread=2, centre=centre) for _ in range(2))
        self.down = X.random_matrix(rng, FP4, E * embd, ff, spread=2, centre=127 - int(np.log2(ff) / 2) - 1)
        self.dev = {n: ds3.Buffer.from_array(getattr(self, n)) for n in ("delta", "weight", "router")}
        if router_type == ds3.TYPE_F16:
            self.dev["router"] = ds3.Buffer.from_array(self.router.astype(np.float16))
        self.idx, self.scores = ds3.Buffer.alloc(4 * T * k), ds3.Buffer.alloc(4 * T * k)

    def hidden(self):
        return ds3.Buffer.from_array(self.x)

    def block(self, hidden, delta=True):
        ds3.moe_block_mx(hidden, self.dev["weight"], EPS, self.dev["router"], self.router_type, self.gate.dev, self.up.dev,
                         self.down.dev, self.T, self.E, self.k, delta=self.dev["delta"] if delta else None,
                         indices=self.idx, scores=self.scores)

    def buffers(self):
        T, k, S = self.T, self.k, self.T * self.k
        b = {n: ds3.Buffer.alloc(4 * size) for n, size in
             (("xn", T * self.embd), ("counts", self.E), ("offsets", self.E + 1), ("ids", S), ("wts", S), ("pos", S),
              ("y", S * self.embd), ("logits", T * self.E))}
        b["xq"], b["h"] = ds3.MxMatrix.alloc(I8, T, self.embd), ds3.MxMatrix.alloc(I8, S, self.ff)
        return b

    def steps(self, hidden, b):
        """The same with the separate calls (up to 2048 tokens)."""
        T, E, k = self.T, self.E, self.k
        ds3.add_rms_norm_mx(hidden, self.dev["weight"], EPS, b["xq"], delta=self.dev["delta"], sum_out=hidden, x_norm=b["xn"])
        rb = ds3.row_bytes(self.router_type, self.embd)
        L = ds3.hip()
        assert L.ds3_hip_moe_route(b["xn"], self.dev["router"], b["logits"], self.idx, self.scores, T, self.embd, E, k, rb,
                                   self.router_type, True) == 0
        assert L.ds3_hip_moe_bucket(self.idx, self.scores, T, k, E, b["counts"], b["offsets"], b["ids"], b["wts"],
                                    b["pos"]) == 0
        ds3.moe_gate_up_mx(b["xq"], self.gate.dev, self.up.dev, b["offsets"], b["h"], E, ids=b["ids"])
        ds3.matmul_mx_grouped(b["h"], self.down.dev, b["offsets"], b["y"], T * k, E)
        ds3.moe_combine(b["y"], b["pos"], self.scores, hidden, T, k, T * k, self.embd, accumulate=True)

    def reference(self, idx, scores):
        """hidden in 64 bits with this routing, and how far the roundings may take it."""
        s = self.x.astype(np.float64) + self.delta
        y = s / np.sqrt((s ** 2).mean(1, keepdims=True) + EPS) * self.weight
        # fp32 norm: the sum and its square's, the mean's, the root's and the products'
        # roundings, under 16 in all on the way to a value; then half a step of at
        # most amax / 64, or a whole one at the saturated code
        amax = np.repeat(np.abs(y).reshape(len(y), -1, 32).max(2), 32, axis=1)
        dy = 16 * 2.0 ** -24 * np.abs(y) + amax * (2.0 ** -6 + 2.0 ** -20)
        out, err = s.copy(), 2.0 ** -23 * np.abs(s)
        for e in range(self.E):
            t, j = np.nonzero(idx == e)
            if len(t) == 0:
                continue
            g, u = (m.values[e * self.ff:(e + 1) * self.ff] for m in (self.gate, self.up))
            d = self.down.values[e * self.embd:(e + 1) * self.embd]
            gv, uv = y[t] @ g.T, y[t] @ u.T
            dg, du = ((dy[t] @ np.abs(m).T) + X.sum_bound((np.abs(y) + dy)[t] @ np.abs(m).T, self.embd) for m in (g, u))
            h = X.silu_mul(gv, uv)
            dh = 1.1 * dg * (np.abs(uv) + du) + np.abs(gv) * du + (16 + np.abs(gv)) * 2.0 ** -23 * np.abs(h)
            top = np.repeat((np.abs(h) + dh).reshape(len(h), -1, 32).max(2), 32, axis=1)
            dh = dh + top * 2.0 ** -6
            w = scores[t, j, None].astype(np.float64)
            mag = (np.abs(h) + dh) @ np.abs(d).T
            out[t] += w * (h @ d.T)
            err[t] += np.abs(w) * (dh @ np.abs(d).T + X.sum_bound(mag, self.ff) + 2 * (self.k + 1) * 2.0 ** -24 * mag)
        return out, err


SHAPES = [(1, 64, 4, 1, 32), (3, 256, 8, 3, 96), (17, 512, 16, 8, 128), (100, 1024, 32, 4, 160), (300, 288, 128, 8, 64)]


@pytest.mark.parametrize("T,embd,E,k,ff", SHAPES)
def test_steps(hip_ready, T, embd, E, k, ff):
    m = Block(T, embd, E, k, ff)
    hidden = m.hidden()
    m.steps(hidden, m.buffers())
    idx, scores = m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k))
    got = hidden.read(np.float32, (T, embd))
    want, err = m.reference(idx, scores)
    assert (np.abs(got - want) <= err).all(), f"worst {np.max(np.abs(got - want) / err):.3g} of the bound"


@pytest.mark.parametrize("router_type", [ds3.TYPE_F32, ds3.TYPE_F16])
@pytest.mark.parametrize("T,embd,E,k,ff", SHAPES + [(16, 256, 16, 4, 64)])
def test_block_is_its_steps(hip_ready, T, embd, E, k, ff, router_type):
    m = Block(T, embd, E, k, ff, router_type)
    one, two, bufs = m.hidden(), m.hidden(), m.buffers()
    m.steps(one, bufs)
    idx, scores = m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k))
    m.block(two)
    assert np.array_equal(m.idx.read(np.int32, (T, k)), idx)
    a, b = one.read(np.float32, (T, embd)), two.read(np.float32, (T, embd))
    if T > 16:
        assert np.array_equal(m.scores.read(np.float32, (T, k)), scores) and np.array_equal(a, b)
    else:
        # few tokens are routed by another order of sums: a logit is off by at most embd
        # roundings of its terms' magnitudes in either, a score by twice two logits' errors
        xn = bufs["xn"].read(np.float32, (T, embd)).astype(np.float64)
        tol = 4 * embd * 2.0 ** -24 * 1.01 * (np.abs(xn) @ np.abs(m.router).T).max() + 16 * 2.0 ** -24
        assert np.allclose(m.scores.read(np.float32, (T, k)), scores, rtol=tol, atol=0)
        y = np.abs(bufs["y"].read(np.float32, (T * k, embd))).max()
        assert (np.abs(a - b) <= tol * y + (2 * k + 2) * 2.0 ** -24 * (y + np.abs(m.x + m.delta))).all()


@pytest.mark.parametrize("mode", [1, 2])
def test_block_in_the_other_router_modes(hip_ready, mode):
    """The sequential router for one token, the certified one for many."""
    T, k = (1, 3) if mode == 1 else (40, 3)
    m = Block(T, 256, 8, k, 64)
    old = ds3.hip().ds3_hip_set_router_mode(mode)
    try:
        hidden = m.hidden()
        m.block(hidden)
        got, idx, scores = hidden.read(np.float32, m.x.shape), m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k))
    finally:
        ds3.hip().ds3_hip_set_router_mode(old)
    want, err = m.reference(idx, scores)
    assert (np.abs(got - want) <= err).all()
    assert np.allclose(scores.sum(1), 1, atol=1e-5) and all(len(set(r)) == k for r in idx)


def test_block_of_more_than_a_chunk(hip_ready):
    """More tokens than are bucketed at once: as in two calls."""
    T, embd, E, k, ff = 2500, 128, 16, 3, 64
    m = Block(T, embd, E, k, ff)
    whole = m.hidden()
    m.block(whole)
    got, idx, scores = whole.read(np.float32, (T, embd)), m.idx.read(np.int32, (T, k)), m.scores.read(np.float32, (T, k))
    want, err = m.reference(idx, scores)
    assert (np.abs(got - want) <= err).all()


def test_block_without_delta(hip_ready):
    m = Block(20, 256, 8, 2, 64)
    m.delta[:] = 0
    m.dev["delta"] = ds3.Buffer.from_array(m.delta)
    one, two = m.hidden(), m.hidden()
    m.block(one)
    m.block(two, delta=False)
    assert np.array_equal(one.read(np.float32, m.x.shape), two.read(np.float32, m.x.shape))


@pytest.mark.parametrize("T", [1, 40])
def test_batch_and_graphs(hip_ready, T):
    """Two graphs that share the workspace, replayed in turn with eager calls between."""
    m, other = Block(T, 512, 32, 4, 96), Block(T + 30, 256, 16, 2, 64, seed=5)
    b = m.buffers()
    def eager(o):
        h = o.hidden()
        o.block(h)
        return h.read(np.float32, o.x.shape)
    want, want_other = eager(m), eager(other)
    h1, h2, h3 = m.hidden(), other.hidden(), m.hidden()
    ds3.hip().ds3_hip_begin_batch()
    m.block(h1)
    other.block(h2)
    ds3.hip().ds3_hip_end_batch()
    assert np.array_equal(h1.read(np.float32, m.x.shape), want)
    assert np.array_equal(h2.read(np.float32, other.x.shape), want_other)
    m.steps(h3, b)
    steps = h3.read(np.float32, m.x.shape)
    with ds3.Graph() as g1:
        m.block(h1)
    with ds3.Graph() as g2:
        other.block(h2)
    with ds3.Graph() as g3:
        m.steps(h3, b)
    for i in range(4):
        h1.write(m.x)
        h2.write(other.x)
        h3.write(m.x)
        g1.launch()
        g2.launch()
        g3.launch()
        assert np.array_equal(h2.read(np.float32, other.x.shape), want_other), i
        assert np.array_equal(h1.read(np.float32, m.x.shape), want), i
        assert np.array_equal(h3.read(np.float32, m.x.shape), steps), i
        assert np.array_equal(eager(other), want_other)


def test_first_use_in_a_capture(hip_ready):
    """The operators without a workspace are captured without a call before."""
    rng = np.random.default_rng(8)
    x, w = rng.standard_normal((600, 2048)).astype(np.float32), X.random_matrix(rng, FP4, 2100, 2048)
    src, q, c = ds3.Buffer.from_array(x), ds3.MxMatrix.alloc(I8, 600, 2048), ds3.Buffer.alloc(4 * 600 * 2100)
    with ds3.Graph() as g:
        ds3.mx_quantize(src, ds3.TYPE_F32, q)
        ds3.matmul_mx(q, w.dev, c)
    g.launch()
    got = c.read(np.float32, (600, 2100))
    ds3.matmul_mx(q, w.dev, c)
    assert np.array_equal(c.read(np.float32, (600, 2100)), got)
    xq = X.values(I8, *read_mx(q))
    want, mag = X.product(xq, w.values)
    assert (np.abs(got - want) <= X.sum_bound(mag, 2048)).all()
