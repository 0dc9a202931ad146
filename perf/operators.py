"""Performance cases of the microscaled (MX) operators: 4-bit weights, 8-bit rows, and what joins them.

An MX matrix holds, for every 32 consecutive values of a row, one power of two (E8M0: a byte c stands for
2^(c - 127), 255 for NaN) and 32 codes: MXFP4, a sign and the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6 in four bits
(value 2j in the low half of byte j), or MXINT8, a signed byte q for q / 64.

  quant    rows of F32, F16, Q8_0, Q4_K or Q6_K values to MXFP4 or MXINT8
  norm     residual addition, RMS norm and the rounding of the normalised rows to MXINT8
  matmul   C = X W^T of MXINT8 rows with MXFP4 weights
  gate_up  rows grouped by expert: silu(x Wg^T) * (x Wu^T), rounded to MXINT8
  grouped  rows grouped by expert: C = X W_e^T

The plain forms compute in 32 bits on the values that the codes stand for; exact() does so in 64.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

EPS = 1e-6
STD = 0.02
MXFP4, MXINT8 = "MXFP4", "MXINT8"
QWEN = {"embd": 2048, "ff": 768, "experts": 128, "used": 8}
BLOCK = {"F32": (1, 4), "F16": (1, 2), "Q8_0": (32, 34), "Q4_K": (256, 144), "Q6_K": (256, 210)}


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # activations of eight decode streams on their way into a product: the smallest call
        {"name": "quant_rows_8", "kind": "quant", "rows": 8, "cols": 2048, "src": "F32", "to": MXINT8},
        # a layer's gate experts converted once from the Q4_K blocks of a model file
        {"name": "quant_experts_q4k", "kind": "quant", "rows": 128 * 768, "cols": 2048, "src": "Q4_K", "to": MXFP4},
        # the FFN block's prologue for one decoded token
        {"name": "norm_1", "kind": "norm", "rows": 1, "cols": 2048, "delta": True, "keep": True},
        # the same for a whole long prompt of a wider model, ragged
        {"name": "norm_6001", "kind": "norm", "rows": 6001, "cols": 4096, "delta": True, "keep": False},
        # the output head of every decoded token
        {"name": "head_1", "kind": "matmul", "rows": 1, "n": 151936, "k": 2048},
        # the rows of one expert, or a short ragged prompt through a small projection
        {"name": "rows_27", "kind": "matmul", "rows": 27, "n": 768, "k": 2048},
        # a prefill projection of a 512-token chunk
        {"name": "projection_512", "kind": "matmul", "rows": 512, "n": 4096, "k": 2048},
        # gate and up of one decoded token's eight experts
        {"name": "gate_up_1", "kind": "gate_up", "tokens": 1, "zipf": False, **QWEN},
        # a short prompt: every expert has a few rows
        {"name": "gate_up_37", "kind": "gate_up", "tokens": 37, "zipf": False, **QWEN},
        # a large chunk with Zipf-skewed expert popularity: empty experts beside very full ones
        {"name": "gate_up_zipf_2048", "kind": "gate_up", "tokens": 2048, "zipf": True, **QWEN},
        # down of one decoded token's eight experts
        {"name": "down_1", "kind": "grouped", "tokens": 1, "zipf": False, "gather": False, "embd": 768, "ff": 2048,
         "experts": 128, "used": 8},
        # down of the engine's prefill chunk
        {"name": "down_512", "kind": "grouped", "tokens": 512, "zipf": False, "gather": False, "embd": 768, "ff": 2048,
         "experts": 128, "used": 8},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("quant", "norm", "matmul", "matmul", "gate_up", "gate_up", "grouped", "grouped"))
    if kind == "quant":
        src = rng.choice(("F32", "F16", "Q8_0", "Q4_K", "Q6_K"))
        cols = 256 * rng.randint(1, 16) if BLOCK[src][0] == 256 else 32 * _log_int(rng, 1, 160)
        return {"kind": kind, "rows": _log_int(rng, 1, max(1, (1 << 26) // cols)), "cols": cols, "src": src,
                "to": rng.choice((MXFP4, MXINT8))}
    if kind == "norm":
        cols = 32 * _log_int(rng, 1, 256)
        return {"kind": kind, "rows": _log_int(rng, 1, min(20000, (1 << 24) // cols)), "cols": cols,
                "delta": rng.random() < 0.7, "keep": rng.random() < 0.6}
    if kind == "matmul":
        k = 32 * _log_int(rng, 1, 160) if rng.random() < 0.5 else 512 * rng.randint(1, 8)
        rows = 1 if rng.random() < 0.2 else _log_int(rng, 1, 4096)
        n = _log_int(rng, 1, 8192)
        if rng.random() < 0.6:
            n = max(16, n // 16 * 16)
        if rows == 1:
            n *= 16                                # one token: the heads and decode projections
        n = max(1, min(n, int(25e9) // (rows * k)))
        return {"kind": kind, "rows": rows, "n": n, "k": k}
    shape = {"embd": 32 * _log_int(rng, 4, 64), "ff": 32 * _log_int(rng, 2, 32),
             "experts": rng.choice((4, 8, 32, 60, 64, 128)), "used": rng.choice((1, 2, 4, 8))}
    if rng.random() < 0.5:
        shape = {"embd": rng.choice((512, 1024, 2048)), "ff": rng.choice((256, 512, 768)),
                 "experts": rng.choice((32, 64, 128)), "used": rng.choice((4, 8))}
    shape["used"] = min(shape["used"], shape["experts"])
    if kind == "grouped":
        if rng.random() < 0.5:
            shape["embd"], shape["ff"] = shape["ff"], shape["embd"]
        if rng.random() < 0.3:
            shape["ff"] = max(1, shape["ff"] - rng.randint(1, 31))     # an output width of its own
        shape["gather"] = rng.random() < 0.5
    return {"kind": kind, "tokens": _log_int(rng, 1, 2000), "zipf": rng.random() < 0.3, **shape}


# ---------------------------------------------------------------------------
# The formats, in plain torch
# ---------------------------------------------------------------------------

def _blocks(v):
    return v.reshape(v.shape[0], -1, 32)


def _scale_codes(amax, m, shift):
    """E8M0 bytes of 2^(exponent - shift), where frexp's mantissa m over its bound moves the exponent up by one."""
    _, e = torch.frexp(amax)
    code = (e - 1 - shift + m.to(e.dtype) + 127).clamp(0, 254)
    code = torch.where(amax > 0, code, torch.zeros_like(code))
    return torch.where(torch.isfinite(amax), code, torch.full_like(code, 255))


def _pow2(code, bias):
    """2^(code - bias) as float64, from its bits (a device's pow and exp2 may be an ulp off)."""
    return ((code.long() - bias + 1023) << 52).view(torch.float64)


def _scaled(b, code, bias):
    """b / 2^(code - bias), exact in 32 bits: two factors, as one alone can pass their range."""
    k = bias - code
    return b * _pow2(k // 2, 0).float().unsqueeze(2) * _pow2(k - k // 2, 0).float().unsqueeze(2)


def _to_mxint8(v):
    """(codes int8 [rows][cols], scales uint8 [rows][cols / 32]) of float32 rows."""
    b = _blocks(v)
    amax = b.abs().amax(2)
    code = _scale_codes(amax, torch.zeros_like(amax, dtype=torch.bool), 0)
    q = _scaled(b, code, 133).round().clamp(-127, 127)
    q = torch.where((code == 255).unsqueeze(2), torch.zeros_like(q), q)
    return q.to(torch.int8).reshape(v.shape), code.to(torch.uint8)


def _to_mxfp4(v):
    """(codes uint8 [rows][cols / 2], scales uint8 [rows][cols / 32]) of float32 rows."""
    b = _blocks(v)
    amax = b.abs().amax(2)
    m, _ = torch.frexp(amax)
    code = _scale_codes(amax, m > 0.875, 2)          # the largest value is at most 7 steps of 2^exponent
    y = _scaled(b.abs(), code, 127)
    # nearest magnitude, halfway cases to the even code
    q = ((y > 0.25).byte() + (y >= 0.75).byte() + (y > 1.25).byte() + (y >= 1.75).byte() + (y > 2.5).byte()
         + (y >= 3.5).byte() + (y > 5).byte()) | (torch.signbit(b).byte() << 3)
    q = torch.where((code == 255).unsqueeze(2), torch.zeros_like(q), q).reshape(v.shape[0], -1, 2)
    return q[:, :, 0] | (q[:, :, 1] << 4), code.to(torch.uint8)


def _scales(s, dtype):
    """The powers of two of E8M0 bytes."""
    p = _pow2(s, 127)
    return torch.where(s == 255, torch.full_like(p, math.nan), p).to(dtype)


def _magnitudes(dtype):
    half = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(half + [-x for x in half], dtype=dtype, device="cuda")


def _values(codes, scales, to, dtype=torch.float32):
    """The values of an MX matrix, [..., cols]."""
    if to == MXINT8:
        q = codes.to(dtype) / 64
    else:
        q = _magnitudes(dtype)[torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1).int()]
    return (q.reshape(*scales.shape, 32) * _scales(scales, dtype).unsqueeze(-1)).reshape(q.shape)


def _f16_at(b, at, dtype):
    return b[:, at:at + 2].contiguous().view(torch.float16).to(dtype)


def _source_values(raw, src, cols, dtype=torch.float32):
    """The values of rows of a GGUF type (uint8 [rows][row bytes])."""
    if src in ("F32", "F16"):
        return raw.view(torch.float32 if src == "F32" else torch.float16).to(dtype).reshape(-1, cols)
    b = raw.reshape(-1, BLOCK[src][1])
    if src == "Q8_0":
        return (_f16_at(b, 0, dtype) * b[:, 2:].contiguous().view(torch.int8).to(dtype)).reshape(-1, cols)
    if src == "Q6_K":
        s = b[:, 192:208].contiguous().view(torch.int8).to(dtype)
        ql, qh = b[:, :128].reshape(-1, 2, 2, 32), b[:, 128:192].reshape(-1, 2, 32)
        q = torch.stack((ql[:, :, 0] & 15, ql[:, :, 1] & 15, ql[:, :, 0] >> 4, ql[:, :, 1] >> 4), 2)
        h = torch.stack((qh & 3, (qh >> 2) & 3, (qh >> 4) & 3, qh >> 6), 2)
        q = (q | (h << 4)).to(dtype) - 32
        return ((_f16_at(b, 208, dtype) * s).unsqueeze(2) * q.reshape(-1, 16, 16)).reshape(-1, cols)
    sb = b[:, 4:16]
    s = torch.cat((sb[:, :4] & 63, (sb[:, 8:] & 15) | ((sb[:, :4] >> 6) << 4)), 1).to(dtype)
    m = torch.cat((sb[:, 4:8] & 63, (sb[:, 8:] >> 4) | ((sb[:, 4:8] >> 6) << 4)), 1).to(dtype)
    qs = b[:, 16:].reshape(-1, 4, 32)
    q = torch.stack((qs & 15, qs >> 4), 2).reshape(-1, 8, 32).to(dtype)
    return ((_f16_at(b, 0, dtype) * s).unsqueeze(2) * q - (_f16_at(b, 2, dtype) * m).unsqueeze(2)).reshape(-1, cols)


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------

def _gen(seed, *what):
    h = int(seed) * 1000003 + 17
    for w in what:
        h = (h * 1000003 + int(w) + 1) % (1 << 62)
    return torch.Generator(device="cuda").manual_seed(h)


def _normal(gen, rows, cols, std=1.0):
    return torch.randn(rows, cols, generator=gen, device="cuda") * std


def _hidden(gen, rows, cols):
    """Rows as a decoder's residual stream has them: channels of unlike size, a few of them large."""
    size = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    return _normal(gen, rows, cols) * size


def _weights(gen, rows, cols):
    """MXFP4 codes and scales of N(0, 0.02) weights, a slice of rows at a time."""
    codes = torch.empty(rows, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // cols)
    for r in range(0, rows, step):
        codes[r:r + step], scales[r:r + step] = _to_mxfp4(_normal(gen, min(step, rows - r), cols, STD))
    return codes, scales


def _source(gen, rows, cols, src):
    """uint8 [rows][row bytes]: values, or blocks with codes of every pattern and scales as a model's weights have."""
    if src in ("F32", "F16"):
        v = _normal(gen, rows, cols, STD) * torch.exp(torch.randn(rows, 1, generator=gen, device="cuda"))
        return v.to(torch.float32 if src == "F32" else torch.float16).view(torch.uint8)
    per, nb = BLOCK[src]
    n = rows * cols // per
    b = torch.randint(0, 256, (n, nb), dtype=torch.uint8, generator=gen, device="cuda")
    for at in {"Q8_0": (0,), "Q6_K": (208,), "Q4_K": (0, 2)}[src]:
        d = (1e-4 + 1e-3 * torch.rand(n, 1, generator=gen, device="cuda")).to(torch.float16)
        b[:, at:at + 2] = d.view(torch.uint8)
    return b.reshape(rows, -1)


def _zipf_bias(n):
    """Logit bias ln(rank^-1.2) over a fixed permutation of the experts."""
    p = (np.random.default_rng(7).permutation(n) + 1.0) ** -1.2
    return np.log(p / p.sum()).astype(np.float32)


def _routing(case, seed):
    """(offsets int32 [experts + 1], ids int32 [tokens * used]): the tokens of each expert, in token order."""
    e, t, u = case["experts"], case["tokens"], case["used"]
    z = torch.randn(t, e, generator=_gen(seed, 3), device="cuda")
    if case["zipf"]:
        z = z + torch.from_numpy(_zipf_bias(e)).cuda()
    chosen = torch.topk(z, u, dim=1).indices.reshape(-1)
    order = torch.argsort(chosen, stable=True)
    counts = torch.bincount(chosen, minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, (order // u).int()


def _inputs(case, seed):
    """The case's inputs as torch tensors."""
    s = types.SimpleNamespace(case=case)
    kind = case["kind"]
    if kind == "quant":
        s.raw = _source(_gen(seed, 1), case["rows"], case["cols"], case["src"])
    elif kind == "norm":
        s.x = _hidden(_gen(seed, 1), case["rows"], case["cols"])
        s.delta = 0.3 * _hidden(_gen(seed, 2), case["rows"], case["cols"]) if case["delta"] else None
        s.gain = 1.0 + _normal(_gen(seed, 3), 1, case["cols"], 0.2)
    elif kind == "matmul":
        s.x = _to_mxint8(_hidden(_gen(seed, 1), case["rows"], case["k"]))
        s.w = _weights(_gen(seed, 2), case["n"], case["k"])
    else:
        k, f, e, t = case["embd"], case["ff"], case["experts"], case["tokens"]
        s.offsets, s.ids = _routing(case, seed)
        gather = kind == "gate_up" or case["gather"]
        s.x = _to_mxint8(_hidden(_gen(seed, 1), t if gather else t * case["used"], k))
        if not gather:
            s.ids = None                           # the rows lie in the experts' order already
        s.w = [_weights(_gen(seed, 4 + i), e * f, k) for i in range(2 if kind == "gate_up" else 1)]
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


def _tensor(buf, shape, typestr):
    return torch.as_tensor(_Memory(buf, shape, typestr), device="cuda")


def _buffer(t):
    """A library buffer holding the tensor's bytes."""
    from qw3_amd import ds3
    t = t.contiguous()
    b = ds3.Buffer.alloc(t.numel() * t.element_size())
    _tensor(b, (b.nbytes,), "|u1").copy_(t.view(torch.uint8).reshape(-1))
    return b


def _matrix(pair, to, rows, cols):
    from qw3_amd import ds3
    return ds3.MxMatrix(_buffer(pair[0]), _buffer(pair[1]), _type(to), rows, cols)


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

    def out(name, rows, cols, typestr="<f4"):
        buf = ds3.Buffer.alloc(max(1, rows * cols * int(typestr[2])))
        b.outputs[name] = _tensor(buf, (rows, cols), typestr)
        return buf

    b.outputs = {}
    if kind == "quant":
        b.src = _buffer(s.raw)
        b.q = ds3.MxMatrix.alloc(_type(c["to"]), c["rows"], c["cols"])
        b.values = out("values", c["rows"], c["cols"])
    elif kind == "norm":
        b.x, b.gain = _buffer(s.x), _buffer(s.gain)
        b.delta = _buffer(s.delta) if c["delta"] else None
        b.sum = out("sum", c["rows"], c["cols"]) if c["delta"] else None
        b.x_norm = out("x_norm", c["rows"], c["cols"]) if c["keep"] else None
        b.q = ds3.MxMatrix.alloc(ds3.TYPE_MXINT8, c["rows"], c["cols"])
        b.values = out("values", c["rows"], c["cols"], "<f2")
    elif kind == "matmul":
        b.x, b.w = _matrix(s.x, MXINT8, c["rows"], c["k"]), _matrix(s.w, MXFP4, c["n"], c["k"])
        b.c = out("c", c["rows"], c["n"])
    else:
        k, f, rows = c["embd"], c["ff"], c["tokens"] * c["used"]
        b.x = _matrix(s.x, MXINT8, s.x[0].shape[0], k)
        b.w = [_matrix(w, MXFP4, c["experts"] * f, k) for w in s.w]
        b.offsets, b.ids, b.rows = _buffer(s.offsets), None if s.ids is None else _buffer(s.ids), rows
        if kind == "gate_up":
            b.h = ds3.MxMatrix.alloc(ds3.TYPE_MXINT8, rows, f)
            b.values = out("h", rows, f, "<f2")
        else:
            b.c = out("c", rows, f)
    return b


def _run_own(b):
    from qw3_amd import ds3
    c, kind = b.case, b.case["kind"]
    if kind == "quant":
        ds3.mx_quantize(b.src, _type(c["src"]), b.q)
        ds3.mx_dequantize(b.q, b.values)
    elif kind == "norm":
        ds3.add_rms_norm_mx(b.x, b.gain, EPS, b.q, delta=b.delta, sum_out=b.sum, x_norm=b.x_norm)
        ds3.mx_dequantize(b.q, b.values, ds3.TYPE_F16)
    elif kind == "matmul":
        ds3.matmul_mx(b.x, b.w, b.c)
    elif kind == "gate_up":
        ds3.moe_gate_up_mx(b.x, b.w[0], b.w[1], b.offsets, b.h, c["experts"], ids=b.ids)
        ds3.mx_dequantize(b.h, b.values, ds3.TYPE_F16)
    else:
        ds3.matmul_mx_grouped(b.x, b.w[0], b.offsets, b.c, b.rows, c["experts"], ids=b.ids)
    return b.outputs


def prepare(case, seed):
    if own:
        from qw3_amd import ds3
        ds3.init()
        _batch(False)
    s = _inputs(case, seed)
    if own:
        s = _library(s)
        torch.cuda.synchronize()                   # the inputs were written on torch's stream
        _batch(True)
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _grouped_plain(s, *weights):
    """x of every row times each of the weights of its group, [rows][n]: the groups that have rows, padded to the widest."""
    c = s.case
    x = _values(*s.x, MXINT8)
    if s.ids is not None:
        x = x[s.ids.long()]
    counts = (s.offsets[1:] - s.offsets[:-1]).long()
    active = torch.nonzero(counts).squeeze(1)
    widest, rows = int(counts.max()), x.shape[0]
    group = torch.repeat_interleave(torch.arange(active.numel(), device="cuda"), counts[active])
    at = torch.arange(rows, device="cuda") - s.offsets[:-1].long()[active][group]
    padded = torch.zeros(active.numel(), widest, x.shape[1], device="cuda")
    padded[group, at] = x
    out = []
    for codes, scales in weights:
        w = _values(codes.reshape(c["experts"], c["ff"], -1)[active], scales.reshape(c["experts"], c["ff"], -1)[active],
                    MXFP4)
        out.append(torch.bmm(padded, w.transpose(1, 2))[group, at])
    return out


def run(state):
    if own:
        return _run_own(state)
    s, c, kind = state, state.case, state.case["kind"]
    if kind == "quant":
        v = _source_values(s.raw, c["src"], c["cols"])
        quantised = _to_mxint8(v) if c["to"] == MXINT8 else _to_mxfp4(v)
        return {"values": _values(*quantised, c["to"])}
    if kind == "norm":
        x = s.x + s.delta if c["delta"] else s.x
        y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s.gain
        out = {"values": _values(*_to_mxint8(y), MXINT8).to(torch.float16)}
        return {**out, **({"sum": x} if c["delta"] else {}), **({"x_norm": y} if c["keep"] else {})}
    if kind == "matmul":
        return {"c": _values(*s.x, MXINT8) @ _values(*s.w, MXFP4).t()}
    if kind == "gate_up":
        g, u = _grouped_plain(s, *s.w)
        return {"h": _values(*_to_mxint8(g / (1 + torch.exp(-g)) * u), MXINT8).to(torch.float16)}
    return {"c": _grouped_plain(s, *s.w)[0]}


# ---------------------------------------------------------------------------
# Work, 64-bit results
# ---------------------------------------------------------------------------

def _mx_bytes(to, rows, cols):
    return rows * (cols // 2 if to == MXFP4 else cols) + rows * (cols // 32)


def _distinct(case):
    """Experts that the tokens are expected to choose between them (sampled logits of the inputs' distribution)."""
    e, u = case["experts"], case["used"]
    z = np.random.default_rng(3).standard_normal((case["tokens"], e))
    if case["zipf"]:
        z += _zipf_bias(e)
    return len(np.unique(np.argpartition(-z, u - 1, axis=1)[:, :u]))


def work(case):
    kind = case["kind"]
    if kind == "quant":
        per, nb = BLOCK[case["src"]]
        n = case["rows"] * case["cols"]
        return {"bytes": n // per * nb + _mx_bytes(case["to"], case["rows"], case["cols"]), "flops": 2 * n}
    if kind == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * (1 + 2 * case["delta"] + case["keep"]) + 4 * case["cols"]
                + _mx_bytes(MXINT8, case["rows"], case["cols"]), "flops": 6 * n}
    if kind == "matmul":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": _mx_bytes(MXFP4, n, k) + _mx_bytes(MXINT8, m, k) + 4 * m * n, "flops": 2 * m * n * k}
    k, f, t, rows = case["embd"], case["ff"], case["tokens"], case["tokens"] * case["used"]
    gate_up = kind == "gate_up"
    gather = gate_up or case["gather"]
    return {"bytes": _distinct(case) * (2 if gate_up else 1) * _mx_bytes(MXFP4, f, k)
            + _mx_bytes(MXINT8, t if gather else rows, k) + 4 * (case["experts"] + 1) + (4 * rows if gather else 0)
            + (_mx_bytes(MXINT8, rows, f) if gate_up else 4 * rows * f),
            "flops": (4 if gate_up else 2) * rows * f * k}


def _decode64(codes, scales, to):
    """The float64 values of an MX matrix, byte by byte of its codes."""
    if to == MXINT8:
        v = codes.double() * 2.0 ** -6
    else:
        fp4 = [(1 - 2 * (c >> 3)) * (c & 1) / 2 if not c & 6 else
               (1 - 2 * (c >> 3)) * (2 + (c & 1)) * 2.0 ** ((c >> 1 & 3) - 2) for c in range(16)]
        pairs = torch.tensor([[fp4[byte & 15], fp4[byte >> 4]] for byte in range(256)], dtype=torch.float64, device="cuda")
        v = pairs[codes.long()].reshape(codes.shape[0], -1)
    power = torch.tensor([2.0 ** (c - 127) for c in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
    return v * power[scales.long()].repeat_interleave(32, dim=1)


def _source64(raw, src, cols):
    """The float64 values of rows of a GGUF type, value by value of a block (places in bytes)."""
    if src in ("F32", "F16"):
        return raw.view(torch.float32 if src == "F32" else torch.float16).double()
    per, nb = BLOCK[src]
    b = raw.reshape(-1, nb)
    i = torch.arange(per, device="cuda")

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).double()

    def low(at, bits, shift):                       # `bits` bits of the byte at each place
        return (b[:, at].int() >> shift) & ((1 << bits) - 1)

    if src == "Q8_0":
        v = half(0) * b[:, 2:].contiguous().view(torch.int8).double()
    elif src == "Q6_K":
        h, r = i // 128, i % 128
        q = low(64 * h + r % 64, 4, 4 * (r // 64)) | (low(128 + 32 * h + r % 32, 2, 2 * (r // 32)) << 4)
        v = half(208) * b[:, 192 + i // 16].contiguous().view(torch.int8).double() * (q - 32).double()
    else:
        j = i // 32
        late, k = (j >= 4).int(), j % 4
        first, second, both = low(4 + k, 8, 0), low(8 + k, 8, 0), low(12 + k, 8, 0)
        sc = torch.where(late == 1, (both & 15) | (first >> 6 << 4), first & 63)
        mn = torch.where(late == 1, (both >> 4) | (second >> 6 << 4), second & 63)
        v = half(0) * sc * low(16 + 32 * (j // 2) + i % 32, 4, 4 * (j % 2)) - half(2) * mn
    return v.reshape(-1, cols)


def _floor_pow2(v):
    """The largest power of two that is at most v > 0 (float64 normal numbers)."""
    return ((v.view(torch.int64) >> 52) << 52).view(torch.float64)


def _round64(v):
    """MXINT8 values of float64 rows, by the format's definition."""
    b = v.reshape(v.shape[0], v.shape[1] // 32, 32)
    step = _floor_pow2(b.abs().amax(2, keepdim=True).clamp(min=2.0 ** -127)) / 64
    return (torch.clamp(torch.round(b / step), -127, 127) * step).reshape(v.shape)


def _fp4_round64(v):
    """MXFP4 values of float64 rows: the smallest power of two with at most seven of it to the largest value."""
    b = v.reshape(v.shape[0], v.shape[1] // 32, 32)
    amax = b.abs().amax(2, keepdim=True)
    p = _floor_pow2(amax.clamp(min=2.0 ** -125)) / 4
    p = torch.where(amax > 7 * p, 2 * p, p)
    y = b.abs() / p
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return (torch.clamp(torch.round(y / step) * step, max=6) * torch.sign(b) * p).reshape(v.shape)


def _decode64(codes, scales, to):
    """The float64 values of an MX matrix, byte by byte of its codes."""
    if to == MXINT8:
        v = codes.double() * 2.0 ** -6
    else:
        fp4 = [(1 - 2 * (c >> 3)) * (c & 1) / 2 if not c & 6 else
               (1 - 2 * (c >> 3)) * (2 + (c & 1)) * 2.0 ** ((c >> 1 & 3) - 2) for c in range(16)]
        pairs = torch.tensor([[fp4[byte & 15], fp4[byte >> 4]] for byte in range(256)], dtype=torch.float64, device="cuda")
        v = pairs[codes.long()].reshape(codes.shape[0], -1)
    power = torch.tensor([2.0 ** (c - 127) for c in range(255)] + [math.nan], dtype=torch.float64, device="cuda")
    return v * power[scales.long()].repeat_interleave(32, dim=1)


def _source64(raw, src, cols):
    """The float64 values of rows of a GGUF type, value by value of a block (places in bytes)."""
    if src in ("F32", "F16"):
        return raw.view(torch.float32 if src == "F32" else torch.float16).double()
    per, nb = BLOCK[src]
    b = raw.reshape(-1, nb)
    i = torch.arange(per, device="cuda")

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).double()

    def low(at, bits, shift):                       # `bits` bits of the byte at each place
        return (b[:, at].int() >> shift) & ((1 << bits) - 1)

    if src == "Q8_0":
        v = half(0) * b[:, 2:].contiguous().view(torch.int8).double()
    elif src == "Q6_K":
        h, r = i // 128, i % 128
        q = low(64 * h + r % 64, 4, 4 * (r // 64)) | (low(128 + 32 * h + r % 32, 2, 2 * (r // 32)) << 4)
        v = half(208) * b[:, 192 + i // 16].contiguous().view(torch.int8).double() * (q - 32).double()
    else:
        j = i // 32
        late, k = (j >= 4).int(), j % 4
        first, second, both = low(4 + k, 8, 0), low(8 + k, 8, 0), low(12 + k, 8, 0)
        sc = torch.where(late == 1, (both & 15) | (first >> 6 << 4), first & 63)
        mn = torch.where(late == 1, (both >> 4) | (second >> 6 << 4), second & 63)
        v = half(0) * sc * low(16 + 32 * (j // 2) + i % 32, 4, 4 * (j % 2)) - half(2) * mn
    return v.reshape(-1, cols)


def _round64(v):
    """MXINT8 values of float64 rows, by the format's definition."""
    b = v.reshape(v.shape[0], v.shape[1] // 32, 32)
    amax = b.abs().amax(2, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -127))) - 6)
    return (torch.clamp(torch.round(b / step), -127, 127) * step).reshape(v.shape)


def _fp4_round64(v):
    """MXFP4 values of float64 rows: the smallest power of two with at most seven steps to the largest value."""
    b = v.reshape(v.shape[0], v.shape[1] // 32, 32)
    amax = b.abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -130) / 7))
    e = torch.where(amax > 7 * torch.exp2(e), e + 1, e)
    e = torch.where(amax <= 7 * torch.exp2(e - 1), e - 1, e).clamp(min=-127)
    y = b.abs() / torch.exp2(e)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return (torch.clamp(torch.round(y / step) * step, max=6) * torch.sign(b) * torch.exp2(e)).reshape(v.shape)


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        v = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        step = max(1, (1 << 25) // case["cols"])
        for r in range(0, case["rows"], step):
            x = _source64(s.raw[r:r + step], case["src"], case["cols"])
            x = x.float().double()                  # a block's value is the nearest of 32 bits
            v[r:r + step] = _round64(x) if case["to"] == MXINT8 else _fp4_round64(x)
        return {"values": v}
    if kind == "norm":
        x = s.x.double() + (s.delta.double() if case["delta"] else 0)
        y = x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * s.gain.double()
        out = {"values": _round64(y)}
        return {**out, **({"sum": x} if case["delta"] else {}), **({"x_norm": y} if case["keep"] else {})}
    x = _decode64(*s.x, MXINT8)
    if kind == "matmul":
        codes, scales = s.w
        return {"c": torch.cat([x @ _decode64(codes[r:r + 8192], scales[r:r + 8192], MXFP4).t()
                                for r in range(0, case["n"], 8192)], 1)}
    f, out = case["ff"], []
    at = s.offsets.tolist()
    for e in range(case["experts"]):
        rows = x[at[e]:at[e + 1]] if s.ids is None else x[s.ids[at[e]:at[e + 1]].long()]
        y = [rows @ _decode64(codes[e * f:(e + 1) * f], scales[e * f:(e + 1) * f], MXFP4).t()
             for codes, scales in s.w]
        out.append(y[0] if kind == "grouped" else _round64(y[0] / (1 + torch.exp(-y[0])) * y[1]))
    return {"h" if kind == "gate_up" else "c": torch.cat(out)}
