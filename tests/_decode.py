"""Plain 64-bit forms of the attention and sampling operators, and their device buffers."""
from __future__ import annotations

import math

import numpy as np

from qw3_amd import ds3

F32, F16 = ds3.TYPE_F32, ds3.TYPE_F16
NP = {F32: np.float32, F16: np.float16}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -140, F16: 2.0 ** -25}           # half the distance of the smallest numbers


def ints(v):
    return ds3.Buffer.from_array(np.asarray(v, np.int32))


def floats(v):
    return ds3.Buffer.from_array(np.asarray(v, np.float32))


def frequencies(rotary, base, scaling=ds3.ROPE_PLAIN, factor=1.0, low=0.0, high=0.0, original=0):
    """Radians a position of each pair, the factor of rotated values."""
    out, m = [], 1.0
    for i in range(rotary // 2):
        theta = base ** (-2 * i / rotary)
        turns = original * theta / (2 * math.pi)
        if scaling == ds3.ROPE_LINEAR:
            theta /= factor
        elif scaling == ds3.ROPE_WAVELENGTH:
            s = min(1.0, max(0.0, (turns - low) / (high - low)))
            theta *= s + (1 - s) / factor
        elif scaling == ds3.ROPE_YARN:
            at = [rotary * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (high, low)]
            a, b = max(0, math.floor(at[0])), min(rotary - 1, math.ceil(at[1]))
            s = min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))
            theta *= 1 - s + s / factor
            m = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        out.append(theta)
    return np.array(out), m


def rope(x, positions, theta, m, norm=None, eps=1e-6, interleaved=False):
    """(values, bounds of the error before the output's rounding) of heads x [tokens][heads][dim].

    The bound.  A head's norm in 32 bits: squares and a sum of dim terms in chains of at most dim / lanes + log2 lanes
    additions (20 for any head_dim), root, quotient and two products, together 26 half steps of 2^-24 relative.
    Sine and cosine: the turn rounds by 2^-26 (9.4e-8 radians), sincospi by two steps (2.4e-7), the factor by 2^-24;
    two products and a sum: in all under 2^-20 of |a| + |b|, times the factor.  The angle itself: the turns a position
    are off by at most 2^-51 relative (a power, two quotients), as is their product."""
    x = x.astype(np.float64)
    slack = np.zeros(x.shape[:2] + (1,))
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
        slack = slack + 26 * 2.0 ** -24
    r = 2 * len(theta)
    out, tol = x.copy(), np.abs(x) * slack
    a = positions.astype(np.float64)[:, None, None] * theta
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    p, q = x[..., first], x[..., second]
    out[..., first], out[..., second] = m * (p * np.cos(a) - q * np.sin(a)), m * (q * np.cos(a) + p * np.sin(a))
    size = m * (np.abs(p) + np.abs(q))
    tol[..., first] = tol[..., second] = size * (2.0 ** -20 + slack + np.abs(a) * 2.0 ** -50)
    return out, tol


def rounded_to(tol, value, type_):
    return tol + (np.abs(value) + tol) * HALF_STEP[type_] + TINY[type_]


class Pages:
    """Host caches [blocks][kv heads][block][dim] in float16 with a block table of random order."""

    def __init__(self, rng, lens, block, n_kv, dim, spare=2, max_blocks=None):
        need = [-(-n // block) for n in lens]
        self.block, self.n_kv, self.dim = block, n_kv, dim
        self.n_blocks = sum(need) + spare
        self.max_blocks = max_blocks or max(max(need), 1)
        self.table = np.full((len(lens), self.max_blocks), -1, np.int32)
        order = rng.permutation(self.n_blocks).astype(np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_blocks, n_kv, block, dim)
        self.k = rng.standard_normal(shape).astype(np.float16)
        self.v = rng.standard_normal(shape).astype(np.float16)

    def device(self):
        return ds3.KvCache(ds3.Buffer.from_array(self.k), ds3.Buffer.from_array(self.v), self.n_blocks, self.block,
                           self.n_kv, self.dim)

    def rows(self, i, n):
        """(which of n positions lie in the cache, their k, their v: [n][kv heads][dim])."""
        pos = np.arange(n)
        b = self.table[i, pos // self.block]
        ok = (b >= 0) & (b < self.n_blocks)
        b = np.where(ok, b, 0)
        return ok, self.k[b, :, pos % self.block].astype(np.float64), self.v[b, :, pos % self.block].astype(np.float64)


def attention(q, pages, new, lens, scale, window=0, type_=F32):
    """(values, bounds) for q [tokens][heads][dim], the requests' new tokens and lengths.

    The bound.  A score s sums dim exact products (F16: q as it is; F32: q in parts of 22 bits, 2^-22 of each product)
    in 32 bits: off by d = scale sum|q k| (dim + 5) 2^-24, and by a rounding of the product with scale.  exp2's argument
    (s - m) log2 e rounds by 3 half steps of up to |s - m| log2 e, exp2 itself by two steps, so weights are off by
    e = exp(2 d + 4 |s - m| 2^-24) - 1 + 2^-22 relative, the rounding of weights adds 2^-22 (F32: two parts) or 2^-11
    (F16) and 2^-20 of the largest weight where the parts lose bits at the bottom of their range (weights below 2^-14 are
    held to 2^-25).  The sums over n keys, in any order with rescalings between: (2 n + 16) 2^-24."""
    t = 0
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    group = q.shape[1] // pages.n_kv
    dim = q.shape[2]
    for i, (m, n) in enumerate(zip(new, lens)):
        ok, k, v = pages.rows(i, max(0, min(n, pages.max_blocks * pages.block)))
        for j in range(m):
            pos = n - m + j
            lo = max(0, pos - window + 1) if window else 0
            see = np.arange(lo, max(lo, min(pos + 1, len(ok))))
            see = see[ok[see]]
            if len(see):
                for h in range(q.shape[1]):
                    x = q[t, h].astype(np.float64)
                    kk, vv = k[see, h // group], v[see, h // group]
                    s = kk @ x * scale
                    d = (np.abs(kk) @ np.abs(x) * abs(scale)).max() * (dim + 6) * 2.0 ** -24
                    w = np.exp(s - s.max())
                    spread = (s.max() - s).max()
                    e = math.expm1(2 * d + 4 * spread * 2.0 ** -24) + 2.0 ** -22
                    e += 2.0 ** -22 if type_ == F32 else 2.0 ** -11
                    e = 2 * e + (2 * len(see) + 16) * 2.0 ** -24
                    size = (w @ np.abs(vv)) / w.sum()
                    out[t, h] = w @ vv / w.sum()
                    tol[t, h] = size * e + 2.0 ** (-25 if type_ == F16 else -36) * np.abs(vv).sum(0) / w.sum()
            t += 1
    return out, tol


def sample_row(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, its share) of one row: the definition with whole-number weights."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float32)).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    s = x[order]
    if s[0] == -np.inf:
        return -1, 0.0
    if not t > 0 or s[0] == np.inf:
        return int(order[0]), 1.0
    order, s = order[s > -np.inf], s[s > -np.inf]
    real = np.exp((s - s[0]) * (1.0 / float(np.float32(t))))
    w = [int(v) for v in np.rint(real * 2.0 ** 44)]
    if k > 0:
        w = w[:k]
    if p < 1:
        least = max(1, math.ceil(max(p, 0.0) * float(sum(w))))
        c, n = 0, 0
        while n < len(w) and c < least:
            c += w[n]
            n += 1
        w = w[:n]
    if m > 0:
        w = [v for v, y in zip(w, real) if y >= m] or w[:1]
    total = sum(w)
    least, c = min(math.floor(max(u, 0.0) * float(total)) + 1, total), 0
    for j, v in enumerate(w):
        c += v
        if c >= least:
            return int(order[j]), real[j] * 2.0 ** 44 / total
    raise AssertionError
