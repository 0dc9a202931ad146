"""A small decoder's steps from the operators together: plan, projections, head norms with rotation and the paged cache,
attention, the FFN block, the output head, sampling -- prompts first, then tokens, eagerly and as one replayed graph.
Each attention, rotation and draw is checked against its 64-bit form on the device's own inputs to it; the graph's
results are the eager ones bit for bit."""
import numpy as np
import pytest

import _decode as D
from _decode import F16, F32
from qw3_amd import ds3
from qw3_amd import workload as W
from qw3_amd._native import hip

pytestmark = pytest.mark.gpu

Q8 = ds3.TYPE_Q8_0
K, HEADS, KV, DIM, VOCAB, EXPERTS, USED = 512, 8, 2, 64, 1000, 16, 4
BLOCK, BLOCKS, MAX_BLOCKS, ROWS, EPS = 8, 60, 20, 96, 1e-6
PROMPTS = [19, 1, 7, 57]


def weights(seed, rows, cols):
    return ds3.Buffer.from_array(W.quant_matrix(Q8, W.NORMAL, seed, 1, rows, cols, 0.0, 0.05))


def gain(seed, n):
    return 1 + 0.1 * np.random.default_rng(seed).standard_normal(n).astype(np.float32)


class Layer:
    def __init__(self, seed):
        self.q, self.k, self.v = (weights(seed + i, n * DIM, K) for i, n in enumerate((HEADS, KV, KV)))
        self.o = weights(seed + 4, K, HEADS * DIM)
        self.spec = W.LayerSpec(n_embd=K, n_ff=256, n_expert=EXPERTS)
        self.moe = W.make_layer(self.spec, seed).to_device()
        self.norm, self.ffn_norm = (ds3.Buffer.from_array(gain(seed + i, K)) for i in (5, 6))
        self.q_gain, self.k_gain = gain(seed + 7, DIM), gain(seed + 8, DIM)
        self.q_norm, self.k_norm = ds3.Buffer.from_array(self.q_gain), ds3.Buffer.from_array(self.k_gain)
        self.cache = ds3.KvCache.alloc(BLOCKS, BLOCK, KV, DIM)
        self.cache.k.zero()
        self.cache.v.zero()


class Snapshot(D.Pages):
    """A device cache as it is."""
    def __init__(self, cache, table):
        self.block, self.n_kv, self.dim, self.n_blocks, self.max_blocks = BLOCK, KV, DIM, BLOCKS, MAX_BLOCKS
        shape = (BLOCKS, KV, BLOCK, DIM)
        self.table, self.k, self.v = table, cache.k.read(np.float16, shape), cache.v.read(np.float16, shape)


class Decoder:
    def __init__(self, n_seq, type_):
        self.n, self.type = n_seq, type_
        self.layers = [Layer(100), Layer(200)]
        self.embd = ds3.Buffer.from_array(np.random.default_rng(1).standard_normal((VOCAB, K)).astype(np.float32))
        self.head, self.norm = weights(300, VOCAB, K), ds3.Buffer.from_array(gain(301, K))
        self.turns = ds3.rope_table(DIM, 1e6)
        self.new, self.lens = D.ints([0] * n_seq), D.ints([0] * n_seq)
        self.table, self.free = D.ints(np.full((n_seq, MAX_BLOCKS), -1)), D.ints(np.arange(BLOCKS)[::-1])
        self.n_free, self.offsets, self.status = D.ints([BLOCKS]), D.ints([0] * (n_seq + 1)), D.ints([0] * 4)
        self.ids, self.last, self.tokens = D.ints([0] * ROWS), D.ints([0] * n_seq), D.ints([0] * n_seq)
        self.positions, self.slots = D.ints([0] * ROWS), D.ints([0] * ROWS)
        f = lambda n: ds3.Buffer.alloc(ROWS * n * 4)                             # noqa: E731
        self.h, self.x, self.out = f(K), f(K), f(K)
        self.q, self.k, self.v, self.turned, self.att = f(HEADS * DIM), f(KV * DIM), f(KV * DIM), f(HEADS * DIM), f(HEADS * DIM)
        self.logits, self.probs, self.uniform = ds3.Buffer.alloc(n_seq * VOCAB * 4), D.floats([0] * n_seq), D.floats([0] * n_seq)
        self.temperature, self.top_k = D.floats(np.linspace(0.5, 1.2, n_seq)), D.ints([0, 20, 5, 400][:n_seq])
        self.top_p, self.min_p = D.floats([0.95, 0.9, 1.0, 0.99][:n_seq]), D.floats([0, 0, 0.02, 0][:n_seq])

    def product(self, a, w, c, rows, n, k):
        assert hip().ds3_hip_matmul_quantized_batch(a, w, c, rows, n, k, ds3.row_bytes(Q8, k), 0, Q8) == 0

    def step(self, rows, ids, watch=None):
        """One step of `rows` tokens; watch(layer, what) between its calls."""
        watch = watch or (lambda layer, what: None)
        ds3.kv_plan(self.new, self.lens, self.table, self.free, self.n_free, self.offsets, self.positions, self.slots,
                    self.status, self.n, MAX_BLOCKS, BLOCKS, BLOCK, rows)
        assert hip().ds3_hip_gather_rows_f32(self.embd, ids, self.h, K, rows, 0) == 0
        for layer in self.layers:
            ds3.rms_norm(self.h, layer.norm, self.x, K, rows, EPS)
            self.product(self.x, layer.q, self.q, rows, HEADS * DIM, K)
            self.product(self.x, layer.k, self.k, rows, KV * DIM, K)
            self.product(self.x, layer.v, self.v, rows, KV * DIM, K)
            ds3.rope_append(self.q, self.k, self.v, self.positions, self.slots, layer.cache, self.turned, rows, HEADS, F32,
                            self.type, table=self.turns, q_norm=layer.q_norm, k_norm=layer.k_norm, eps=EPS)
            watch(layer, "append")
            ds3.attention_paged(self.turned, layer.cache, self.table, self.offsets, self.lens, self.att, rows, self.n,
                                HEADS, MAX_BLOCKS, DIM ** -0.5, self.type)
            watch(layer, "attention")
            if self.type == F32:                      # (products take 32 bits; 16-bit attention ends the layer here)
                self.product(self.att, layer.o, self.out, rows, K, HEADS * DIM)
                assert hip().ds3_hip_vec_add_inplace(self.h, self.out, rows * K) == 0
            ds3.moe_block(self.h, layer.ffn_norm, EPS, layer.moe.router, layer.spec.router_type, layer.moe.experts, rows,
                          EXPERTS, USED)
        assert hip().ds3_hip_gather_rows_f32(self.h, self.last, self.out, K, self.n, 0) == 0
        ds3.rms_norm(self.out, self.norm, self.x, K, self.n, EPS)
        self.product(self.x, self.head, self.logits, self.n, VOCAB, K)
        ds3.sample(self.logits, self.uniform, self.tokens, self.n, VOCAB, self.temperature, self.top_k, self.top_p,
                   self.min_p, self.probs)
        watch(None, "sample")

    def prompts(self, rng, lens, watch=None):
        ids = rng.integers(0, VOCAB, sum(lens))
        self.ids.write(ids.astype(np.int32))
        self.new.write(np.asarray(lens, np.int32))
        at = np.cumsum(lens) - 1
        self.last.write(np.maximum(at, 0).astype(np.int32))
        self.uniform.write(rng.random(self.n).astype(np.float32))
        self.step(sum(lens) + 3, self.ids, watch)     # three rows of a padded batch
        assert self.status.read(np.int32, 4)[2:].tolist() == [0, 0]
        self.new.write(np.ones(self.n, np.int32))
        self.last.write(np.arange(self.n, dtype=np.int32))

    def state(self):
        caches = [b.read(np.uint8, b.nbytes) for layer in self.layers for b in (layer.cache.k, layer.cache.v)]
        return [self.tokens.read(np.int32, self.n), self.probs.read(np.float32, self.n), self.lens.read(np.int32, self.n),
                self.table.read(np.int32, (self.n, MAX_BLOCKS)), self.logits.read(np.float32, (self.n, VOCAB)), *caches]

    def check(self, layer, what):
        """The call that has just run, on what the device gave it."""
        lens, offsets = self.lens.read(np.int32, self.n), self.offsets.read(np.int32, self.n + 1)
        table, rows = self.table.read(np.int32, (self.n, MAX_BLOCKS)), int(offsets[-1])
        if what == "append":
            positions, slots = self.positions.read(np.int32, rows), self.slots.read(np.int32, rows)
            theta, m = D.frequencies(DIM, 1e6)
            q, tol = D.rope(self.q.read(np.float32, (rows, HEADS, DIM)), positions, theta, m, layer.q_gain, EPS)
            got = self.turned.read(D.NP[self.type], (rows, HEADS, DIM)).astype(np.float64)
            assert (np.abs(got - q) <= D.rounded_to(tol, q, self.type)).all()
            k, tol = D.rope(self.k.read(np.float32, (rows, KV, DIM)), positions, theta, m, layer.k_gain, EPS)
            pages = Snapshot(layer.cache, table)
            got = pages.k[slots // BLOCK, :, slots % BLOCK].astype(np.float64)
            assert (np.abs(got - k) <= D.rounded_to(tol, k, F16)).all()
            v = self.v.read(np.float32, (rows, KV, DIM)).astype(np.float16)
            assert np.array_equal(pages.v[slots // BLOCK, :, slots % BLOCK], v)
        elif what == "attention":
            q = self.turned.read(D.NP[self.type], (rows, HEADS, DIM))
            want, tol = D.attention(q, Snapshot(layer.cache, table), np.diff(offsets), lens, DIM ** -0.5, 0, self.type)
            got = self.att.read(D.NP[self.type], (rows, HEADS, DIM)).astype(np.float64)
            assert (np.abs(got - want) <= D.rounded_to(tol, want, self.type)).all()
        else:
            x, u = self.logits.read(np.float32, (self.n, VOCAB)), self.uniform.read(np.float32, self.n)
            t, k = self.temperature.read(np.float32, self.n), self.top_k.read(np.int32, self.n)
            p, m = self.top_p.read(np.float32, self.n), self.min_p.read(np.float32, self.n)
            got = self.tokens.read(np.int32, self.n)
            for r in range(self.n):
                assert got[r] == D.sample_row(x[r], float(u[r]), t[r], int(k[r]), float(p[r]), float(m[r]))[0]


def steps(type_, graph):
    """Prompts, six tokens, one request gone and another in its place, six more: every step's state."""
    rng, d, out = np.random.default_rng(9), Decoder(4, type_), []
    d.prompts(rng, PROMPTS, None if graph else d.check)
    out.append(d.state())
    run = None
    for i in range(12):
        if i == 6:
            ds3.kv_release(D.ints([0, 0, 0, 1]), d.lens, d.table, d.free, d.n_free, 4, MAX_BLOCKS, BLOCKS, BLOCK)
            tokens = d.tokens.read(np.int32, 4)
            d.prompts(rng, [0, 0, 0, 30])             # (the others' tokens are drawn anew below)
            tokens[3] = d.tokens.read(np.int32, 4)[3]
            d.tokens.write(tokens)
        d.uniform.write(rng.random(4).astype(np.float32))
        if graph and i == 1:
            with ds3.Graph() as run:
                d.step(4, d.tokens)
        if run:
            run.launch()
        else:
            d.step(4, d.tokens, d.check if not graph and i in (0, 5, 11) else None)
        assert d.status.read(np.int32, 4)[2:].tolist() == [0, 0]
        out.append(d.state())
    return out


@pytest.mark.parametrize("type_", [F32, F16])
def test_steps(hip_ready, type_):
    eager = steps(type_, False)
    assert eager[0][2].tolist() == PROMPTS and eager[-1][2].tolist() == [31, 13, 19, 36]
    assert all(((0 <= s[0]) & (s[0] < VOCAB)).all() and (s[1] > 0).all() for s in eager)
    replayed = steps(type_, True)
    for i, (a, b) in enumerate(zip(eager, replayed)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), i


def test_graphs_that_share_workspaces(hip_ready):
    """Two graphs of split attention and of few-row sampling, replayed in turn with eager calls between."""
    rng = np.random.default_rng(3)
    cases = []
    for new, lens, heads, kv, dim, type_ in (([1, 1], [4000, 2500], 8, 2, 128, F32), ([70, 2], [1500, 900], 4, 2, 64, F16)):
        pages = D.Pages(rng, lens, 16, kv, dim)
        q = rng.standard_normal((sum(new), heads, dim)).astype(D.NP[type_])
        args = (ds3.Buffer.from_array(q), pages.device(), D.ints(pages.table), D.ints(np.r_[0, np.cumsum(new)]), D.ints(lens))
        cases.append((args, ds3.Buffer.alloc(q.nbytes), q, (sum(new), len(new), heads, pages.max_blocks, 0.1, type_)))
    x = rng.standard_normal((2, 50000)).astype(np.float32)
    logits, u, tokens = ds3.Buffer.from_array(x), [D.floats([0.3, 0.9]), D.floats([0.7, 0.05])], [D.ints([0, 0]) for _ in "ab"]

    def call(i):
        args, out, _, more = cases[i]
        ds3.attention_paged(*args, out, *more)
        ds3.sample(logits, u[i], tokens[i], 2, 50000)

    def read(i):
        _, out, q, _ = cases[i]
        return out.read(q.dtype, q.shape), tokens[i].read(np.int32, 2)
    want = []
    for i in (0, 1):
        call(i)
        want.append(read(i))
    graphs = []
    for i in (0, 1):
        with ds3.Graph() as g:
            call(i)
        graphs.append(g)
    for turn in range(4):
        for i in (0, 1):
            cases[i][1].zero()
            tokens[i].write(np.zeros(2, np.int32))
        graphs[turn % 2].launch()
        graphs[1 - turn % 2].launch()
        if turn == 2:
            call(0)
        for i in (0, 1):
            assert all(np.array_equal(a, b) for a, b in zip(read(i), want[i])), (turn, i)


def test_caches_beyond_32_bits(hip_ready):
    """A cache of more than 2^31 values: blocks at both ends and around the middle."""
    rng, dim, block = np.random.default_rng(4), 128, 16
    blocks = (1 << 31) // (block * dim) + 40
    cache = ds3.KvCache.alloc(blocks, block, 1, dim)
    n, new = [75, 40], [70, 1]
    table = np.full((2, 5), -1, np.int32)
    table[0] = [blocks - 1, 3, blocks // 2, blocks - 30, blocks - 2]
    table[1, :3] = [blocks - 3, 0, blocks // 2 + 1]
    small = D.Pages(rng, n, block, 1, dim, spare=0)
    small.table = np.full((2, 5), -1, np.int32)
    at = 0
    for i in range(2):
        for j in range(-(-n[i] // block)):
            small.table[i, j] = at
            for buf, host in ((cache.k, small.k), (cache.v, small.v)):
                buf.write(host[at], offset=int(table[i, j]) * block * dim * 2)
            at += 1
    q, k, v = (rng.standard_normal((71, h, dim)).astype(np.float32) for h in (4, 1, 1))
    positions = np.r_[np.arange(5, 75), 39]
    slots = np.array([table[int(i == 70), p // block] * block + p % block for i, p in enumerate(positions)])
    assert slots.max() * dim > 2 ** 31
    turned, out = ds3.Buffer.alloc(q.nbytes), ds3.Buffer.alloc(q.nbytes)
    ds3.rope_append(ds3.Buffer.from_array(q), ds3.Buffer.from_array(k), ds3.Buffer.from_array(v), None, D.ints(slots), cache,
                    turned, 71, 4)
    for i, p in enumerate(positions):
        b = small.table[int(i == 70), p // block]
        small.k[b, :, p % block], small.v[b, :, p % block] = k[i], v[i]
    ds3.attention_paged(turned, cache, D.ints(table), D.ints([0, 70, 71]), D.ints(n), out, 71, 2, 4, 5, dim ** -0.5)
    want, tol = D.attention(q, small, new, n, dim ** -0.5)
    got = out.read(np.float32, q.shape)
    assert (np.abs(got - want) <= D.rounded_to(tol, want, F32)).all()
