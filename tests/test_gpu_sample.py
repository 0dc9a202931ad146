"""Sampling against its definition in whole numbers, row by row."""
import numpy as np
import pytest

import _decode as D
from qw3_amd import ds3

pytestmark = pytest.mark.gpu

TOP = np.float32(1 - 2.0 ** -24)                     # the largest number below 1


def check(x, u, t=None, k=None, p=None, m=None, pad=0):
    rows, vocab = x.shape
    host = np.full((rows, vocab + pad), 100, np.float32)
    host[:, :vocab] = x
    tokens, probs = D.ints(np.full(rows, -5)), D.floats(np.full(rows, -5))
    some = lambda v, f: None if v is None else f(v)                              # noqa: E731
    ds3.sample(ds3.Buffer.from_array(host), D.floats(u), tokens, rows, vocab, temperature=some(t, D.floats),
               top_k=some(k, D.ints), top_p=some(p, D.floats), min_p=some(m, D.floats), probs=probs,
               row_stride=4 * (vocab + pad))
    got, share = tokens.read(np.int32, rows), probs.read(np.float32, rows)
    for r in range(rows):
        of = lambda v, d: d if v is None else np.float32(v[r])                   # noqa: E731
        want, prob = D.sample_row(x[r], float(np.float32(u[r])), of(t, 1.0), 0 if k is None else int(k[r]),
                                  float(of(p, 1.0)), float(of(m, 0.0)))
        assert got[r] == want, (r, got[r], want, x[r][got[r]], x[r][want])
        # weights are off by 2^-45 each from the ratio's two sides, the quotient rounds to 32 bits
        assert abs(share[r] - prob) <= prob * 2.0 ** -22 + 2.0 ** -60, (r, share[r], prob)
    return got, share


def logits(rng, rows, vocab, peak=6):
    x = 2.5 * rng.standard_normal((rows, vocab))
    at = rng.integers(0, vocab, (rows, 12))
    np.put_along_axis(x, at, peak + 3 * np.abs(rng.standard_normal((rows, 12))), 1)
    return x.astype(np.float32)


SETTINGS = [dict(), dict(t=0.6, k=20, p=0.95), dict(t=1.3, p=0.8), dict(t=0.7, m=0.05), dict(t=1.0, k=1),
            dict(t=0.9, k=300, p=0.9, m=0.01), dict(t=2.0, p=0.999), dict(t=0.05), dict(t=0.0), dict(t=5.0, k=5000)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 64, 1000, 4097, 32000])
@pytest.mark.parametrize("rows", [1, 5])
def test_settings(hip_ready, vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    x = logits(rng, rows, vocab)
    for s in SETTINGS:
        u = rng.random(rows).astype(np.float32)
        u[0] = rng.choice(np.array([0.0, TOP, 0.5], np.float32))
        check(x, u, **{n: np.full(rows, v) for n, v in s.items()})


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (3, 262144), (40, 32000), (300, 5000), (1100, 300)])
def test_rows_with_settings_of_their_own(hip_ready, rows, vocab):
    rng = np.random.default_rng(rows)
    x = logits(rng, rows, vocab)
    pick = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
    of = lambda n, d: np.array([s.get(n, d) for s in pick])                      # noqa: E731
    check(x, rng.random(rows).astype(np.float32), of("t", 1.0), of("k", 0), of("p", 1.0), of("m", 0.0))


@pytest.mark.parametrize("vocab", [5, 3000, 9000, 100000])
def test_ties(hip_ready, vocab):
    """Equal logits go by index: steps of a quarter, few values, all equal, zeros of both signs."""
    rng = np.random.default_rng(vocab)
    rows = np.stack([np.round(4 * logits(rng, 1, vocab)[0]) / 4, rng.integers(0, 3, vocab), np.full(vocab, 1.5),
                     np.where(rng.random(vocab) < 0.5, 0.0, -0.0), np.full(vocab, -3e38)]).astype(np.float32)
    n = len(rows)
    for s in SETTINGS + [dict(k=vocab // 2 + 1, p=0.7), dict(k=vocab - 1), dict(p=0.5), dict(t=1e-3, p=0.3)]:
        for u in (0.0, 0.3, TOP):
            check(rows, np.full(n, u, np.float32), **{a: np.full(n, v) for a, v in s.items()})


def test_rows_that_are_not_finite(hip_ready):
    rng = np.random.default_rng(2)
    x = logits(rng, 9, 500)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2], x[2, 1::2] = -np.inf, np.nan
    x[3, 77:80] = np.inf
    x[4] = -np.inf
    x[4, 123] = -50
    x[5, :499] = np.nan
    x[6, 10] = np.nan
    x[7] = np.finfo(np.float32).min                   # a mask of the type's lowest value
    x[7, [5, 9]] = 3
    x[8, 100:] = np.finfo(np.float32).min
    for s in SETTINGS:
        got, share = check(x, rng.random(9).astype(np.float32), **{n: np.full(9, v) for n, v in s.items()})
        assert got[:5].tolist() == [-1, -1, -1, 77, 123] and got[5] == 499 and share[:5].tolist() == [0, 0, 0, 1, 1]


def test_settings_at_their_ends(hip_ready):
    rng = np.random.default_rng(5)
    x = logits(rng, 12, 2000)
    u = np.array([0.0, TOP, 0.5, 1.0, 2.0, -1.0, np.nan, 0.9, 0.1, 0.7, 0.3, 0.6], np.float32)
    held = np.where(np.isnan(u), 0, np.clip(u, 0, TOP)).astype(np.float32)
    nan, inf = np.nan, np.inf
    for s in (dict(t=[1, 1, inf, 1e-40, 1e30, -1, nan, 1, 0.5, 1, 1, 1]), dict(p=[0, 0, 1, 2, nan, -1, 1e-30, 0.5, 0, 1, inf, -inf]),
              dict(m=[0, 1, 2, nan, -1, 1e-30, 0.5, 1, 0, inf, -inf, 0.1]),
              dict(k=[-1, 0, 1, 2000, 2001, 2 ** 31 - 1, -2 ** 31, 1999, 2, 3, 5, 7])):
        a, _ = check(x, held, **s)
        some = {"t": "temperature", "k": "top_k", "p": "top_p", "m": "min_p"}
        name, v = next(iter(s.items()))
        tokens = ds3.Buffer.alloc(48)
        ds3.sample(ds3.Buffer.from_array(x), D.floats(u), tokens, 12, 2000, **{some[name]: (D.ints if name == "k" else D.floats)(v)})
        got = tokens.read(np.int32, 12)
        # u outside 0 <= u < 1 is held to it
        assert np.array_equal(got[np.isfinite(u) & (u < 1)], a[np.isfinite(u) & (u < 1)]) and np.array_equal(got[6], a[6])


def test_strides_and_alignment(hip_ready):
    rng = np.random.default_rng(7)
    for pad in (1, 3, 64):
        check(logits(rng, 4, 1001), rng.random(4).astype(np.float32), k=np.full(4, 40), pad=pad)
        check(logits(rng, 4, 1001), rng.random(4).astype(np.float32), p=np.full(4, 0.9), pad=pad)


@pytest.mark.parametrize("vocab", [6000, 120000])
def test_large_top_k_with_ties(hip_ready, vocab):
    """More tokens kept than a list holds, borders within values that many tokens share."""
    rng = np.random.default_rng(vocab)
    x = (np.round(logits(rng, 8, vocab) * 4) / 4).astype(np.float32)
    k = np.array([513, 600, 1000, 2000, 4000, 5999, vocab, 700])
    for p in (1.0, 0.9):
        check(x, rng.random(8), t=np.full(8, 1.5), k=k, p=np.full(8, p))


@pytest.mark.parametrize("rows", [1, 4, 260])
def test_rows_of_few_finite_logits(hip_ready, rows):
    """Minus infinity nearly everywhere: one token, three, a run at either end."""
    rng, vocab = np.random.default_rng(rows), 70000 if rows < 100 else 9000
    x = np.full((rows, vocab), -np.inf, np.float32)
    for r in range(rows):
        at = [[rng.integers(vocab)], rng.integers(0, vocab, 3), range(40), range(vocab - 40, vocab)][r % 4]
        x[r, list(at)] = rng.standard_normal(len(at))
    check(x, rng.random(rows), t=np.full(rows, 0.8))
    check(x, rng.random(rows), t=np.full(rows, 0.8), k=np.full(rows, 20), p=np.full(rows, 0.9))


def test_few_rows_draw_as_many_rows_do(hip_ready):
    """A row's token does not depend on how many rows the call has."""
    rng = np.random.default_rng(7)
    for vocab in (5000, 60000):
        x = logits(rng, 3, vocab)
        for s in ({}, dict(k=20, p=0.95), dict(k=1500), dict(m=0.001, p=0.999)):
            u = rng.random(3).astype(np.float32)
            full = {key: np.full(3, value) for key, value in s.items()}
            one = [check(x[i:i + 1], u[i:i + 1], **{key: v[:1] for key, v in full.items()}) for i in range(3)]
            many = 300
            wide = np.broadcast_to(x[:, None], (3, many // 3, vocab)).reshape(many, vocab)
            tokens, probs = D.ints([0] * many), D.floats([0] * many)
            of = {"k": ("top_k", D.ints), "p": ("top_p", D.floats), "m": ("min_p", D.floats)}
            ds3.sample(ds3.Buffer.from_array(np.ascontiguousarray(wide)), D.floats(np.repeat(u, many // 3)), tokens, many,
                       vocab, probs=probs, **{of[key][0]: of[key][1](np.full(many, value)) for key, value in s.items()})
            got, share = tokens.read(np.int32, many).reshape(3, -1), probs.read(np.float32, many).reshape(3, -1)
            for i in range(3):
                assert (got[i] == one[i][0][0]).all() and (share[i] == one[i][1][0]).all()


def test_graph_of_draws(hip_ready):
    """One row and many, replayed with new numbers: the eager call's tokens."""
    rng = np.random.default_rng(8)
    for rows, vocab in ((1, 151936), (70, 20000)):
        logit, u = ds3.Buffer.from_array(logits(rng, rows, vocab)), D.floats([0] * rows)
        tokens, k, p = D.ints([0] * rows), D.ints([50] * rows), D.floats([0.9] * rows)

        def call():
            ds3.sample(logit, u, tokens, rows, vocab, top_k=k, top_p=p)
        call()
        with ds3.Graph() as graph:
            call()
        for _ in range(4):
            u.write(rng.random(rows).astype(np.float32))
            logit.write(logits(rng, rows, vocab))
            graph.launch()
            got = tokens.read(np.int32, rows)
            tokens.write(np.full(rows, -9, np.int32))
            call()
            assert np.array_equal(tokens.read(np.int32, rows), got)
        graph.close()                                 # (while nothing is captured)


@pytest.mark.parametrize("rows,vocab", [(64, 151936), (40, 262144)])
def test_parts_that_begin_with_masked_logits(hip_ready, rows, vocab):
    """A part of a row of more than 32,768 logits, all of them masked but a few at its end, which are negative or lie
    below those of parts that are not masked."""
    rng = np.random.default_rng(rows)
    parts = 256 // rows
    x = np.full((rows, vocab), -np.inf, np.float32)
    ends = [vocab * (i + 1) // parts for i in range(parts)]
    for r in range(rows):
        for i, end in enumerate(ends):
            at = rng.integers(end - 4900, end - 100, 30)
            x[r, at] = [-30, -0.5, 4, -3][r % 4] + rng.standard_normal(len(at))
            if r % 8 >= 4 and i == r % parts:             # one part in full
                x[r, end - vocab // parts + 8:end - 8] = 2 * rng.standard_normal(vocab // parts - 16) - 20 * (r % 3)
    for s in (dict(), dict(t=0.3), dict(t=1e-4), dict(p=0.9), dict(m=0.1, t=2.0)):
        check(x, rng.random(rows).astype(np.float32), **{n: np.full(rows, v) for n, v in s.items()})


def test_numbers_beyond_their_range(hip_ready):
    """u of 1 and more draws what the largest number below 1 does: no token of weight 0, whatever masks the row."""
    rng = np.random.default_rng(11)
    lowest = np.finfo(np.float32).min
    for rows, vocab in ((6, 2000), (6, 40000), (300, 9000)):
        x = logits(rng, rows, vocab)
        x[1, 50:] = lowest
        x[2, ::2] = lowest
        x[3] = np.where(np.arange(vocab) % 7 == 0, x[3], -90)                    # a tail of small, equal weights
        x[4] = np.where(np.arange(vocab) < 5, x[4], x[4] - 60)
        x[5:] = x[5:] if rows == 6 else np.where(rng.random((rows - 5, vocab)) < 0.01, x[5:], lowest)
        high = np.resize(np.array([1, 2, np.inf, 1e30, 1.0000001], np.float32), rows)
        for s in SETTINGS + [dict(t=1e-3), dict(t=30.0)]:
            s = {n: np.full(rows, v) for n, v in s.items()}
            want, _ = check(x, np.full(rows, TOP), **s)
            tokens = D.ints([-5] * rows)
            some = {"t": ("temperature", D.floats), "k": ("top_k", D.ints), "p": ("top_p", D.floats), "m": ("min_p", D.floats)}
            for u in (high, high[::-1].copy()):
                ds3.sample(ds3.Buffer.from_array(x), D.floats(u), tokens, rows, vocab, **{some[n][0]: some[n][1](v) for n, v in s.items()})
                got = tokens.read(np.int32, rows)
                assert np.array_equal(got, want), np.argwhere(got != want)


@pytest.mark.parametrize("rows,vocab", [(2, 60000), (20, 20000), (300, 5000)])
def test_many_steps_of_temperature(hip_ready, rows, vocab):
    """Logits far from 0 in units of the temperature: their weights are as exact as those of others."""
    rng = np.random.default_rng(vocab)
    for centre, t in ((-50, 1e-3), (50, 1e-3), (-50, 0.3), (1000, 0.05), (-2e4, 2.0), (30, 1.0)):
        x = (centre + t * logits(rng, rows, vocab, peak=3)).astype(np.float32)
        for s in (dict(), dict(p=0.9), dict(p=0.99999), dict(m=1e-3)):
            s = {"t": t, **s}
            check(x, rng.random(rows).astype(np.float32), **{n: np.full(rows, v) for n, v in s.items()})
