"""Performance cases of a decoder's attention and sampling operators.

  rope    rotary positions on heads of F32 or F16 rows, each head RMS-normalised first where there is a norm weight
  append  new tokens' q, k and v: head norms, rotation, q out, k and v (F16) into a paged cache
  plan    block tables, positions and cache slots of new tokens from the requests' lengths
  attn    new tokens of each request over the paged cache: causal, grouped heads, an optional window
  sample  temperature, top-k, top-p and min-p, drawn by given uniform numbers

A cache is [blocks][kv heads][block size][head size] for k and for v; slot s is row s % block size of block s / block
size; a request's block table names its blocks in order.  The plain forms compute in 32 bits (angles of positions and
sampling weights in 64), exact() in 64.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

EPS = 1e-6
ROPES = {
    "plain": {"scaling": "plain", "base": 1e6},
    "linear": {"scaling": "linear", "base": 1e4, "factor": 4.0},
    "wavelength": {"scaling": "wavelength", "base": 5e5, "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"scaling": "yarn", "base": 1e6, "factor": 4.0, "low": 1.0, "high": 32.0, "original": 32768},
}
QWEN = {"heads": 32, "kv": 4, "dim": 128}


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the queries of one decoded token, normalised by head
        {"name": "rope_1", "kind": "rope", "tokens": 1, "heads": 32, "dim": 128, "rotary": 128, "type": "F32",
         "interleaved": False, "norm": True, "rope": "plain", "far": 40960},
        # a long prompt's queries far beyond the trained context, half of each head rotated, pairs side by side
        {"name": "rope_far_4001", "kind": "rope", "tokens": 4001, "heads": 64, "dim": 128, "rotary": 64, "type": "F16",
         "interleaved": True, "norm": False, "rope": "yarn", "far": 1 << 20},
        # one token each of eight decode streams into the cache
        {"name": "append_8", "kind": "append", "tokens": 8, **QWEN, "rotary": 128, "type": "F32", "out": "F32",
         "interleaved": False, "norm": True, "rope": "plain", "far": 40960, "block": 16},
        # a prefill chunk of several prompts, queries handed on in 16 bits
        {"name": "append_4096", "kind": "append", "tokens": 4096, **QWEN, "rotary": 128, "type": "F32", "out": "F16",
         "interleaved": False, "norm": True, "rope": "yarn", "far": 131072, "block": 64},
        # a decode step of eight streams
        {"name": "plan_8", "kind": "plan", "seqs": 8, "new": "one", "most": 1, "context": 8192, "block": 16},
        # a serving step: a thousand requests, some of them with prompt chunks, most with one token
        {"name": "plan_1000", "kind": "plan", "seqs": 1000, "new": "mixed", "most": 512, "context": 32768, "block": 16},
        # a single stream's decode
        {"name": "attn_1", "kind": "attn", "seqs": 1, "new": "one", "most": 1, "context": 4096, **QWEN, "type": "F32",
         "block": 16, "window": 0},
        # the decode step of 64 streams with contexts of unlike length
        {"name": "attn_64", "kind": "attn", "seqs": 64, "new": "one", "most": 1, "context": 16384, **QWEN, "type": "F16",
         "block": 16, "window": 0},
        # one prompt chunk among decode streams, in the engine's 32 bits
        {"name": "attn_mixed_16", "kind": "attn", "seqs": 16, "new": "mixed", "most": 512, "context": 4096, **QWEN,
         "type": "F32", "block": 32, "window": 0},
        # long prompts' last chunks
        {"name": "attn_chunks_4096", "kind": "attn", "seqs": 2, "new": "ragged", "most": 4096, "context": 12288, **QWEN,
         "type": "F16", "block": 64, "window": 0},
        # one decoded token, the model's recommended settings
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "settings": "model"},
        # a large batch, every request with its own settings
        {"name": "sample_256", "kind": "sample", "rows": 256, "vocab": 151936, "settings": "mixed"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("rope", "append", "plan", "attn", "attn", "attn", "sample", "sample"))
    dim = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 8, 16))
    kv = rng.choice((1, 2, 4, 8))
    heads = {"heads": group * kv, "kv": kv, "dim": dim}
    rotary = max(2, int(dim * rng.choice((1, 1, 0.5, 0.25))) // 2 * 2)
    turn = {"rotary": rotary, "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.5,
            "rope": rng.choice(tuple(ROPES)), "far": _log_int(rng, 64, 1 << 20)}
    block = rng.choice((8, 16, 16, 32, 64, 128))
    if kind == "rope":
        count = rng.choice((1, 4, 8, 20, 32, 64))
        return {"kind": kind, "tokens": _log_int(rng, 1, min(8192, (1 << 25) // (count * dim))), "heads": count, "dim": dim,
                "type": rng.choice(("F32", "F16")), **turn}
    if kind == "append":
        return {"kind": kind, "tokens": _log_int(rng, 1, min(8192, (1 << 24) // ((group + 2) * kv * dim))), **heads,
                "type": rng.choice(("F32", "F16")), "out": rng.choice(("F32", "F16")), "block": block, **turn}
    if kind == "plan":
        new = rng.choice(("one", "mixed", "ragged"))
        return {"kind": kind, "seqs": _log_int(rng, 1, 1000), "new": new, "most": 1 if new == "one" else _log_int(rng, 2, 512),
                "context": _log_int(rng, 1, 32768), "block": block}
    if kind == "sample":
        vocab = _log_int(rng, 32, 262144)
        return {"kind": kind, "rows": _log_int(rng, 1, max(1, min(512, (38 << 20) // vocab))), "vocab": vocab,
                "settings": rng.choice(("model", "mixed", "open"))}
    new = rng.choice(("one", "one", "mixed", "ragged"))
    seqs = _log_int(rng, 1, 96 if new == "one" else 12)
    most = 1 if new == "one" else _log_int(rng, 2, 2048)
    context = _log_int(rng, 1, 16384)
    cells = seqs * (context + most)
    context = max(1, int(context * min(1.0, (1 << 30) / (cells * kv * dim))))                  # values of the cache
    rows = seqs * group * kv * most
    context = max(1, min(context, (1 << 31) // rows - most))                                   # scores
    case = {"kind": kind, "seqs": seqs, "new": new, "most": most, "context": context, **heads,
            "type": rng.choice(("F32", "F16")), "block": block,
            "window": 0 if rng.random() < 0.75 else _log_int(rng, 1, 4096)}
    while case["most"] > 2 and work({**case, "window": 0})["flops"] > 5e11:
        case["most"] //= 2
    return case


def _lengths(case):
    """(cached tokens, new tokens) of each request: the case's own, whatever the seed."""
    n, most = case["seqs"], case["most"]
    rng = np.random.default_rng(n * 1000003 + most * 1009 + case["context"])
    cached = np.exp(rng.uniform(np.log(max(1, case["context"] / 8)), np.log(case["context"] + 1), n)).astype(np.int64)
    cached[-1] = case["context"]
    if case["new"] == "one":
        new = np.ones(n, np.int64)
    elif case["new"] == "mixed":                      # every sixteenth request has a chunk, the first the longest
        new = np.where(np.arange(n) % 16 == 0, rng.integers(most // 2, most + 1, n), 1)
        new[0] = most
    else:
        new = rng.integers(most // 2, most + 1, n)
        new[-1] = most
    if n > 2:
        cached[1] = 0                                 # a request that has just come
    return cached, new


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------

def _gen(seed, *what):
    h = int(seed) * 1000003 + 29
    for w in what:
        h = (h * 1000003 + int(w) + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(h)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _dtype(name):
    return torch.float32 if name == "F32" else torch.float16


def _ints(values):
    return torch.as_tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _rows(gen, tokens, heads, dim, type_):
    """Heads as a projection gives them: channels of unlike size."""
    size = torch.exp(0.4 * _normal(gen, heads * dim))
    return (_normal(gen, tokens, heads * dim) * size).reshape(tokens, heads, dim).to(_dtype(type_))


def _tables(case, gen):
    """(block table, blocks) for cached + new tokens of each request, over blocks in random order."""
    cached, new = _lengths(case)
    need = -(-(cached + new) // case["block"])
    blocks = int(need.sum()) + 3
    order = torch.randperm(blocks, generator=gen, device="cuda").int()
    most = int(need.max()) + 1
    first = torch.as_tensor(np.cumsum(need) - need, device="cuda")
    at = first[:, None] + torch.arange(most, device="cuda")
    table = torch.where(torch.arange(most, device="cuda") < torch.as_tensor(need, device="cuda")[:, None],
                        order[at.clamp(max=blocks - 1)], -1)
    return table.int().contiguous(), blocks


def _inputs(case, seed):
    s, kind = types.SimpleNamespace(case=case), case["kind"]
    if kind in ("rope", "append"):
        t, d = case["tokens"], case["dim"]
        s.q = _rows(_gen(seed, 1), t, case["heads"], d, case["type"])
        s.positions = torch.randint(0, case["far"], (t,), generator=_gen(seed, 2), device="cuda").int()
        s.q_norm = 1 + 0.2 * _normal(_gen(seed, 3), d) if case["norm"] else None
        s.k_norm = 1 + 0.2 * _normal(_gen(seed, 4), d) if case["norm"] else None
        s.turns = _frequencies(case["rope"], case["rotary"])
        if kind == "append":
            s.k = _rows(_gen(seed, 5), t, case["kv"], d, case["type"])
            s.v = _rows(_gen(seed, 6), t, case["kv"], d, case["type"])
            s.blocks = -(-t // case["block"]) + 5
            order = torch.randperm(s.blocks * case["block"], generator=_gen(seed, 7), device="cuda").int()
            s.slots = order[:t].clone()
            s.slots[t // 2::17] = -1                  # rows of a padded batch
            shape = (s.blocks, case["kv"], case["block"], d)
            s.k_cache = _normal(_gen(seed, 8), *shape).half()
            s.v_cache = _normal(_gen(seed, 9), *shape).half()
    elif kind == "plan":
        cached, new = _lengths(case)
        s.table, s.blocks = _tables(case, _gen(seed, 1))
        b = case["block"]
        had = torch.as_tensor(-(-cached // b), device="cuda")
        have = torch.as_tensor(-(-(cached + new) // b), device="cuda")
        at = torch.arange(s.table.shape[1], device="cuda")
        fresh = (at >= had[:, None]) & (at < have[:, None])
        taken = s.table[fresh]
        spare = torch.randperm(7, generator=_gen(seed, 2), device="cuda").int() + s.blocks
        s.free = torch.cat((spare, taken.flip(0)))    # a stack: the last is taken first
        s.n_free = _ints([s.free.numel()])
        s.blocks += 7
        s.table = torch.where(fresh, -1, s.table).contiguous()
        s.cached, s.new, s.tokens = _ints(cached), _ints(new), int(new.sum()) + 5
        s.free = torch.cat((s.free, torch.full((s.blocks - s.free.numel(),), -1, dtype=torch.int32, device="cuda")))
    elif kind == "attn":
        cached, new = _lengths(case)
        s.table, s.blocks = _tables(case, _gen(seed, 1))
        s.offsets = _ints(np.concatenate(([0], np.cumsum(new))))
        s.lens = _ints(cached + new)
        s.q = (1.5 * _normal(_gen(seed, 2), int(new.sum()), case["heads"], case["dim"])).to(_dtype(case["type"]))
        shape = (s.blocks, case["kv"], case["block"], case["dim"])
        s.k_cache = _normal(_gen(seed, 3), *shape).half()
        s.v_cache = _normal(_gen(seed, 4), *shape).half()
        s.most, s.longest = int(new.max()), int((cached + new).max())
    else:
        n, v = case["rows"], case["vocab"]
        gen = _gen(seed, 1)
        s.logits = 2.5 * _normal(gen, n, v)
        peaks = torch.randint(0, v, (n, 24), generator=gen, device="cuda")
        s.logits.scatter_reduce_(1, peaks, 6 + 4 * _normal(gen, n, 24).abs(), "amax")
        s.logits[:, v - v // 64:] = -math.inf         # the padding of a vocabulary
        s.uniform = torch.rand(n, generator=gen, device="cuda")
        rng = np.random.default_rng(seed)
        if case["settings"] == "model":
            got = [np.full(n, 0.6), np.full(n, 20), np.full(n, 0.95), np.full(n, 0.0)]
        elif case["settings"] == "open":              # nothing but the temperature
            got = [rng.uniform(0.5, 1.5, n), np.zeros(n), np.ones(n), np.zeros(n)]
        else:
            got = [rng.choice((0.0, 0.3, 0.6, 0.7, 1.0, 1.3), n), rng.choice((0, 0, 1, 20, 40, 200, 2000), n),
                   rng.choice((1.0, 0.95, 0.9, 0.8, 0.5), n), rng.choice((0.0, 0.0, 0.02, 0.1), n)]
        s.temperature, s.top_p, s.min_p = (torch.as_tensor(np.float32(got[i]), device="cuda") for i in (0, 2, 3))
        s.top_k = _ints(got[1])
    return s


# ---------------------------------------------------------------------------
# The library's buffers and calls
# ---------------------------------------------------------------------------

class _Memory:
    """A ds3 buffer's device memory for torch (a handle starts with its base address, size and offset)."""

    def __init__(self, buf, shape, typestr):
        import ctypes as C
        self.buf = buf
        base, _, offset = C.cast(buf.handle, C.POINTER(C.c_uint64))[0:3]
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (base + offset, False),
                                         "version": 2}


_TYPESTR = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4", torch.uint8: "|u1"}


def _tensor(buf, shape, dtype):
    return torch.as_tensor(_Memory(buf, shape, _TYPESTR[dtype]), device="cuda")


def _buffer(t):
    """A library buffer holding the tensor's bytes."""
    from qw3_amd import ds3
    t = t.contiguous()
    b = ds3.Buffer.alloc(max(16, t.numel() * t.element_size()))
    _tensor(b, t.shape, t.dtype).copy_(t)
    return b


def _type(name):
    from qw3_amd import ds3
    return getattr(ds3, "TYPE_" + name)


# A program enqueues its layers between begin_batch and end_batch and waits once.
_batch_open = False


def _batch(open_):
    global _batch_open
    from qw3_amd._native import hip
    if open_ and not _batch_open and hip().ds3_hip_begin_batch() != 0:
        raise RuntimeError("begin_batch failed")
    if _batch_open and not open_:
        hip().ds3_hip_end_batch()
    _batch_open = open_


def _library(s):
    """The inputs in the library's buffers, and buffers for what the calls write."""
    from qw3_amd import ds3
    c, kind, b = s.case, s.case["kind"], types.SimpleNamespace(case=s.case)
    b.outputs = {}

    def held(name, like):
        """A buffer that starts as `like` and that the call writes."""
        buf = _buffer(like)
        b.outputs[name] = _tensor(buf, like.shape, like.dtype)
        return buf

    def some(t):
        return None if t is None else _buffer(t)

    if kind in ("rope", "append"):
        r = ROPES[c["rope"]]
        b.table = ds3.rope_table(c["rotary"], r["base"], getattr(ds3, "ROPE_" + r["scaling"].upper()), r.get("factor", 1.0),
                                 r.get("low", 0.0), r.get("high", 0.0), r.get("original", 0))
        b.q, b.positions, b.q_norm, b.k_norm = _buffer(s.q), _buffer(s.positions), some(s.q_norm), some(s.k_norm)
        b.out = held("q", torch.zeros(s.q.shape, dtype=_dtype(c.get("out", c["type"])), device="cuda"))
        if kind == "append":
            b.k, b.v, b.slots = _buffer(s.k), _buffer(s.v), _buffer(s.slots)
            b.cache = ds3.KvCache(held("k_cache", s.k_cache), held("v_cache", s.v_cache), s.blocks, c["block"], c["kv"],
                                  c["dim"])
    elif kind == "plan":
        b.new, b.cached, b.free, b.n_free = _buffer(s.new), _buffer(s.cached), _buffer(s.free), _buffer(s.n_free)
        b.table, b.max_blocks, b.tokens, b.blocks = held("table", s.table), s.table.shape[1], s.tokens, s.blocks
        b.lens, b.left = held("lens", torch.zeros_like(s.cached)), held("left", torch.zeros_like(s.n_free))
        b.offsets = held("offsets", torch.zeros(c["seqs"] + 1, dtype=torch.int32, device="cuda"))
        b.positions = held("positions", torch.zeros(s.tokens, dtype=torch.int32, device="cuda"))
        b.slots = held("slots", torch.zeros(s.tokens, dtype=torch.int32, device="cuda"))
        b.status = held("status", torch.zeros(4, dtype=torch.int32, device="cuda"))
    elif kind == "attn":
        b.q, b.table, b.offsets, b.lens = _buffer(s.q), _buffer(s.table), _buffer(s.offsets), _buffer(s.lens)
        b.cache = ds3.KvCache(_buffer(s.k_cache), _buffer(s.v_cache), s.blocks, c["block"], c["kv"], c["dim"])
        b.out, b.tokens, b.max_blocks = held("out", torch.zeros_like(s.q)), s.q.shape[0], s.table.shape[1]
    else:
        b.logits, b.uniform, b.temperature = _buffer(s.logits), _buffer(s.uniform), _buffer(s.temperature)
        b.top_k, b.top_p, b.min_p = _buffer(s.top_k), _buffer(s.top_p), _buffer(s.min_p)
        b.tokens = held("tokens", torch.zeros(c["rows"], dtype=torch.int32, device="cuda"))
        b.probs = held("probs", torch.zeros(c["rows"], dtype=torch.float32, device="cuda"))
    return b


def _run_own(b):
    from qw3_amd import ds3
    c, kind = b.case, b.case["kind"]
    if kind == "rope":
        ds3.rope(b.q, b.positions, b.table, b.out, c["tokens"], c["heads"], c["dim"], c["rotary"], _type(c["type"]),
                 norm=b.q_norm, eps=EPS, interleaved=c["interleaved"])
    elif kind == "append":
        ds3.rope_append(b.q, b.k, b.v, b.positions, b.slots, b.cache, b.out, c["tokens"], c["heads"], _type(c["type"]),
                        _type(c["out"]), table=b.table, rotary_dim=c["rotary"], q_norm=b.q_norm, k_norm=b.k_norm, eps=EPS,
                        interleaved=c["interleaved"])
    elif kind == "plan":
        ds3.kv_plan(b.new, b.cached, b.table, b.free, b.n_free, b.offsets, b.positions, b.slots, b.status, c["seqs"],
                    b.max_blocks, b.blocks, c["block"], b.tokens, kv_lens_out=b.lens, n_free_out=b.left)
    elif kind == "attn":
        ds3.attention_paged(b.q, b.cache, b.table, b.offsets, b.lens, b.out, b.tokens, c["seqs"], c["heads"], b.max_blocks,
                            c["dim"] ** -0.5, _type(c["type"]), window=c["window"])
    else:
        ds3.sample(b.logits, b.uniform, b.tokens, c["rows"], c["vocab"], temperature=b.temperature, top_k=b.top_k,
                   top_p=b.top_p, min_p=b.min_p, probs=b.probs)
    return b.outputs


def prepare(case, seed):
    if own:
        from qw3_amd import ds3
        ds3.init()
        _batch(False)
    s = _inputs(case, seed)
    if own:
        s = _library(s)
        torch.cuda.synchronize()                      # the inputs were written on torch's stream
        _batch(True)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _frequencies(name, rotary):
    """(angle a position of each pair, in 64 bits, and the factor of the rotated values)."""
    r = ROPES[name]
    i = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    theta = r["base"] ** (-2 * i / rotary)
    if r["scaling"] == "linear":
        return theta / r["factor"], 1.0
    if r["scaling"] == "wavelength":
        rotations = r["original"] * theta / (2 * math.pi)
        smooth = ((rotations - r["low"]) / (r["high"] - r["low"])).clamp(0, 1)
        return theta * ((1 - smooth) / r["factor"] + smooth), 1.0
    if r["scaling"] == "yarn":
        def pair(rotations):
            return rotary * math.log(r["original"] / (rotations * 2 * math.pi)) / (2 * math.log(r["base"]))
        lo, hi = max(0, math.floor(pair(r["high"]))), min(rotary - 1, math.ceil(pair(r["low"])))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return theta * (1 - ramp) + theta / r["factor"] * ramp, 0.1 * math.log(r["factor"]) + 1
    return theta, 1.0


def _rotated(x, norm, s):
    """Heads in 32 bits: normalised, rotated."""
    c = s.case
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    theta, factor = s.turns
    angle = s.positions.double()[:, None] * theta
    cos, sin = (factor * torch.cos(angle)).float()[:, None], (factor * torch.sin(angle)).float()[:, None]
    head, rest = x[..., :c["rotary"]], x[..., c["rotary"]:]
    if c["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head.chunk(2, -1)
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((head, rest), -1)


def _plan_plain(s):
    c = s.case
    b, cached, new = c["block"], s.cached.long(), s.new.long()
    lens = cached + new
    had, have = (cached + b - 1) // b, (lens + b - 1) // b
    fresh = have - had
    first = fresh.cumsum(0) - fresh
    at = torch.arange(s.table.shape[1], device="cuda")
    taken = (at >= had[:, None]) & (at < have[:, None])
    rank = s.n_free.long() - 1 - (first[:, None] + at - had[:, None])
    table = torch.where(taken, s.free[rank.clamp(0, s.free.numel() - 1)], s.table)
    ends = new.cumsum(0)
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends))
    t = torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(ends, t, right=True).clamp(max=c["seqs"] - 1)
    live = t < ends[-1]
    position = torch.where(live, cached[seq] + t - offsets[seq], 0)
    slot = torch.where(live, table[seq, (position // b).clamp(max=s.table.shape[1] - 1)].long() * b + position % b, -1)
    zero = torch.zeros_like(ends[-1])
    return {"table": table, "lens": lens.int(), "left": (s.n_free - fresh.sum()).int(), "offsets": offsets.int(),
            "positions": position.int(), "slots": slot.int(),
            "status": torch.stack((ends[-1], fresh.sum(), zero, zero)).int()}


def _attention_plain(s):
    c = s.case
    g, b, d = c["heads"] // c["kv"], c["block"], c["dim"]
    new, lens = (s.offsets[1:] - s.offsets[:-1]).long(), s.lens.long()
    key = torch.arange(s.longest, device="cuda")
    blocks = s.table.long()[:, key // b].clamp(min=0)
    k = s.k_cache[blocks, :, key % b].float().permute(0, 2, 1, 3)                       # [seqs][kv][keys][dim]
    v = s.v_cache[blocks, :, key % b].float().permute(0, 2, 1, 3).contiguous()
    j = torch.arange(s.most, device="cuda")
    rows = (s.offsets[:-1].long()[:, None] + j).clamp(max=s.q.shape[0] - 1)
    q = s.q[rows].float().reshape(c["seqs"], s.most, c["kv"], g, d).permute(0, 2, 3, 1, 4).reshape(c["seqs"], c["kv"], -1, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(c["seqs"], c["kv"], g, s.most, -1)
    position = (lens - new)[:, None] + j
    seen = (key <= position[..., None]) & (key < lens[:, None, None])
    if c["window"]:
        seen &= key > position[..., None] - c["window"]
    scores = (scores * d ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    del scores
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(c["seqs"], c["kv"], -1, s.longest), v).reshape(c["seqs"], c["kv"], g, s.most, d)
    out = torch.where(total > 0, out / total, 0)
    out = out.permute(0, 3, 1, 2, 4).reshape(c["seqs"], s.most, c["heads"], d)
    return out[j < new[:, None]].to(s.q.dtype)


def _sample_plain(s):
    x, index = torch.sort(s.logits, dim=1, descending=True, stable=True)
    t = s.temperature.double()[:, None]
    greedy = t[:, 0] <= 0
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(t > 0, t, 1))
    rank = torch.arange(x.shape[1], device="cuda")
    kept = (s.top_k[:, None] <= 0) | (rank < s.top_k[:, None])
    w = torch.where(kept, w, 0)
    before = w.cumsum(1) - w
    kept &= (before < s.top_p.double()[:, None] * w.sum(1, keepdim=True)) | (rank == 0)
    kept &= (w >= s.min_p.double()[:, None]) | (rank == 0)
    w = torch.where(kept, w, 0)
    total = w.sum(1)
    drawn = (w.cumsum(1) > (s.uniform.double() * total)[:, None]).int().argmax(1)
    drawn = torch.where(greedy, 0, drawn)[:, None]
    probs = torch.where(greedy, 1, w.gather(1, drawn)[:, 0] / total)
    return {"tokens": index.gather(1, drawn)[:, 0].int(), "probs": probs.float()}


def run(state):
    if own:
        return _run_own(state)
    s, kind = state, state.case["kind"]
    if kind == "rope":
        return {"q": _rotated(s.q, s.q_norm, s).to(s.q.dtype)}
    if kind == "append":
        c, live = s.case, s.slots >= 0
        block, row = s.slots[live].long() // c["block"], s.slots[live].long() % c["block"]
        s.k_cache[block, :, row] = _rotated(s.k, s.k_norm, s)[live].half()
        s.v_cache[block, :, row] = s.v[live].half()
        return {"q": _rotated(s.q, s.q_norm, s).to(_dtype(c["out"])), "k_cache": s.k_cache, "v_cache": s.v_cache}
    if kind == "plan":
        return _plan_plain(s)
    if kind == "attn":
        return {"out": _attention_plain(s)}
    return _sample_plain(s)


# ---------------------------------------------------------------------------
# Work, 64-bit results
# ---------------------------------------------------------------------------

def _size(name):
    return 4 if name == "F32" else 2


def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * _size(case["type"]) + 4 * case["tokens"] + 4 * case["rotary"], "flops": 4 * n}
    if kind == "append":
        n, m = case["tokens"] * case["heads"] * case["dim"], 2 * case["tokens"] * case["kv"] * case["dim"]
        return {"bytes": (n + m) * _size(case["type"]) + n * _size(case["out"]) + 2 * m + 8 * case["tokens"],
                "flops": 4 * (n + m)}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    cached, new = _lengths(case)
    if kind == "plan":
        fresh = int((-(-(cached + new) // case["block"]) + -cached // case["block"]).sum())
        return {"bytes": 16 * case["seqs"] + 8 * fresh + 8 * int(new.sum()), "flops": 4 * int(new.sum())}
    position = np.concatenate([np.arange(a, a + b) for a, b in zip(cached, new)])
    seen = position + 1 if not case["window"] else np.minimum(position + 1, case["window"])
    read = cached + new if not case["window"] else np.minimum(cached + new, case["window"] - 1 + new)
    heads = case["heads"] * case["dim"]
    return {"bytes": 4 * case["kv"] * case["dim"] * int(read.sum()) + 2 * int(new.sum()) * heads * _size(case["type"]),
            "flops": 4 * heads * int(seen.sum())}


def _turned64(x, norm, s):
    """Heads in 64 bits, pairs as complex numbers."""
    c, r = s.case, ROPES[s.case["rope"]]
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * norm.double()
    half, factor = c["rotary"] // 2, 1.0
    theta = [math.exp(-2 * i / c["rotary"] * math.log(r["base"])) for i in range(half)]
    if r["scaling"] == "linear":
        theta = [f / r["factor"] for f in theta]
    elif r["scaling"] == "wavelength":
        for i, f in enumerate(theta):
            length = 2 * math.pi / f
            if length > r["original"] / r["low"]:
                theta[i] = f / r["factor"]
            elif length > r["original"] / r["high"]:
                part = (r["original"] / length - r["low"]) / (r["high"] - r["low"])
                theta[i] = (1 - part) * f / r["factor"] + part * f
    elif r["scaling"] == "yarn":
        factor = 1 + math.log(r["factor"]) / 10
        where = [c["rotary"] / 2 * math.log(r["original"] / (n * 2 * math.pi)) / math.log(r["base"]) for n in (r["high"], r["low"])]
        lo, hi = max(math.floor(where[0]), 0), min(math.ceil(where[1]), c["rotary"] - 1)
        for i, f in enumerate(theta):
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            theta[i] = part * f / r["factor"] + (1 - part) * f
    angle = s.positions.double()[:, None, None] * torch.tensor(theta, dtype=torch.float64, device="cuda")
    first = slice(0, 2 * half, 2) if c["interleaved"] else slice(0, half)
    second = slice(1, 2 * half, 2) if c["interleaved"] else slice(half, 2 * half)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, factor), angle)
    x = x.clone()
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _attention64(s):
    """Request by request, kv head by kv head."""
    c, out = s.case, torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    g, at, lens = c["heads"] // c["kv"], s.offsets.tolist(), s.lens.tolist()
    for i in range(c["seqs"]):
        n, new = lens[i], at[i + 1] - at[i]
        blocks = s.table[i, :-(-n // c["block"])].long()
        back = n - 1 - torch.arange(n, device="cuda") - (new - 1 - torch.arange(new, device="cuda"))[:, None]
        hidden = back < 0 if not c["window"] else (back < 0) | (back >= c["window"])
        for h in range(c["kv"]):
            k = s.k_cache[blocks, h].reshape(-1, c["dim"])[:n].double()
            v = s.v_cache[blocks, h].reshape(-1, c["dim"])[:n].double()
            for a in range(g):
                z = s.q[at[i]:at[i + 1], h * g + a].double() @ k.t() / math.sqrt(c["dim"])
                out[at[i]:at[i + 1], h * g + a] = torch.softmax(z.masked_fill_(hidden, -math.inf), 1) @ v
    return out


def _probability64(s, row):
    """The drawn token's probability in one row, from its sorted list."""
    x = s.logits[row].double().cpu().numpy()
    t, k, p, m, u = (float(v[row]) for v in (s.temperature, s.top_k, s.top_p, s.min_p, s.uniform))
    if t <= 0:
        return 1.0
    w = np.sort(np.exp((x - x.max()) / t))[::-1]
    w = w[:int(k)] if k > 0 else w
    w = w[:max(1, int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1)]
    w = w[w >= m]
    return float(w[min(len(w) - 1, int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")))] / w.sum())


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None                                   # whole numbers
    s = _inputs(case, seed)
    if kind == "rope":
        return {"q": _turned64(s.q, s.q_norm, s)}
    if kind == "append":
        k, v = s.k_cache.double(), s.v_cache.double()
        new = _turned64(s.k, s.k_norm, s)
        slots = s.slots.tolist()
        at = [t for t in range(case["tokens"]) if slots[t] >= 0]
        block = torch.tensor([slots[t] // case["block"] for t in at], device="cuda").long()
        row = torch.tensor([slots[t] % case["block"] for t in at], device="cuda").long()
        k[block, :, row], v[block, :, row] = new[at], s.v[at].double()
        return {"q": _turned64(s.q, s.q_norm, s), "k_cache": k, "v_cache": v}
    if kind == "attn":
        return {"out": _attention64(s)}
    return {"tokens": None, "probs": torch.tensor([_probability64(s, i) for i in range(case["rows"])], dtype=torch.float64)}
