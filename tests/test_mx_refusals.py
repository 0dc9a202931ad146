"""Calls of the microscaled operators that the library refuses, each with its
diagnostic and before any device or buffer access: stand-in handles are enough,
and no device is needed."""
import ctypes as C

import numpy as np
import pytest

import _mx as X
from qw3_amd import _native, ds3

FP4, I8, F32 = X.FP4, X.I8, ds3.TYPE_F32


class Handle(C.Structure):
    """What a ds3_hip_buffer_t holds."""
    _fields_ = [("base", C.c_uint64), ("bytes", C.c_size_t), ("offset", C.c_size_t), ("owner", C.c_bool),
                ("readonly", C.c_bool)]


def buf(nbytes, at, readonly=False):
    return Handle(at, nbytes, 0, False, readonly)


@pytest.fixture
def lib():
    lib = _native._bind(C.CDLL(str(_native.LIB_DIR / "libds3_hip.so")), _native.SIGNATURES)
    if lib.ds3_hip_debug_simulate_capture(1) != 0:        # a device context is open in this process
        pytest.skip("a device context is open in this process")
    lib.ds3_hip_debug_simulate_capture(0)
    return lib


MB = 1 << 20
# far apart, all on multiples of 16 bytes
A, B, D, E, G, H, J, K, L = (buf(64 * MB, (i + 1) << 30) for i in range(9))
small = buf(1, 100 << 30)
odd = buf(64 * MB, (200 << 30) + 8)
odder = buf(64 * MB, (201 << 30) + 2)
locked = buf(64 * MB, 202 << 30, readonly=True)


def ref(v):
    return C.cast(C.byref(v), C.c_void_p) if isinstance(v, Handle) else v


def refused(lib, capfd, name, args, *words):
    capfd.readouterr()
    assert getattr(lib, "ds3_hip_" + name)(*map(ref, args)) == -1
    err = capfd.readouterr().err
    for w in words:
        assert w in err, err
    assert "no HIP device" not in err, "accepted as far as the device"


def changed(args, **at):
    args = list(args)
    for i, v in at.items():
        args[int(i[1:])] = v
    return args


QUANT = [A, F32, 4 * 64, B, D, I8, 3, 64]
VALUES = [A, B, I8, 3, 64, D, F32]
NORM = [A, B, D, 1e-6, E, G, H, J, 64, 3]
DENSE = [A, B, D, E, G, 3, 5, 64]
GROUPED = [A, B, D, E, G, H, J, 4, 6, 2, 5, 64]
GATE_UP = [A, B, D, E, G, H, J, K, L, buf(MB, 99 << 30), 4, 6, 2, 32, 64]


@pytest.mark.parametrize("name,args", [("mx_quantize", QUANT), ("mx_dequantize", VALUES), ("add_rms_norm_mx", NORM),
                                       ("matmul_mx", DENSE), ("matmul_mx_grouped", GROUPED), ("moe_gate_up_mx", GATE_UP)])
def test_missing_and_small_buffers(lib, capfd, name, args):
    optional = {("add_rms_norm_mx", 1), ("add_rms_norm_mx", 4), ("add_rms_norm_mx", 5), ("matmul_mx_grouped", 5),
                ("moe_gate_up_mx", 7)}
    for i, v in enumerate(args):
        if not isinstance(v, Handle):
            continue
        if (name, i) not in optional:
            refused(lib, capfd, name, changed(args, **{f"a{i}": None}))
        refused(lib, capfd, name, changed(args, **{f"a{i}": small}), "holds")


def test_sizes_and_types(lib, capfd):
    refused(lib, capfd, "mx_quantize", changed(QUANT, a7=48), "n_cols=48 must be a multiple of 32")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a7=0), "must be a multiple of 32")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a5=F32), "no microscaled type")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a1=99), "unsupported")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a1=ds3.TYPE_Q4_K, a2=144), "unsupported")      # 64 of 256
    refused(lib, capfd, "mx_quantize", changed(QUANT, a2=4 * 63), "shorter than one row")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a2=4 * 64 + 2), "multiple of 4 bytes")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a0=odder), "multiple of 4 bytes")
    refused(lib, capfd, "mx_quantize", changed(QUANT, a6=1 << 31), "out of range")
    huge = [buf(1 << 40, (i + 1) << 44) for i in range(2)]
    # the span of the rows passes 64 bits
    refused(lib, capfd, "mx_quantize", changed(QUANT, a2=1 << 40, a3=huge[0], a4=huge[1], a6=(1 << 24) + 1), "out of range")
    refused(lib, capfd, "matmul_mx_grouped", changed(GROUPED, a9=1024, a10=1 << 30, a11=1 << 27), "holds")
    refused(lib, capfd, "mx_dequantize", changed(VALUES, a2=F32), "unsupported")
    refused(lib, capfd, "mx_dequantize", changed(VALUES, a6=ds3.TYPE_Q8_0), "unsupported")
    refused(lib, capfd, "mx_dequantize", changed(VALUES, a4=33), "multiple of 32")
    refused(lib, capfd, "mx_dequantize", changed(VALUES, a5=odder), "multiple of 4 bytes")
    refused(lib, capfd, "add_rms_norm_mx", changed(NORM, a8=100), "multiple of 32")
    refused(lib, capfd, "add_rms_norm_mx", changed(NORM, a3=-1.0))
    refused(lib, capfd, "add_rms_norm_mx", changed(NORM, a3=float("nan")))
    refused(lib, capfd, "add_rms_norm_mx", changed(NORM, a1=odder), "multiple of 4 bytes")
    refused(lib, capfd, "matmul_mx", changed(DENSE, a7=16), "K=16 must be a multiple of 32")
    refused(lib, capfd, "matmul_mx", changed(DENSE, a4=odder), "multiple of 4 bytes")
    refused(lib, capfd, "matmul_mx", changed(DENSE, a5=0xffffffff), "out of range")
    refused(lib, capfd, "matmul_mx_grouped", changed(GROUPED, a9=0), "n_group=0")
    refused(lib, capfd, "matmul_mx_grouped", changed(GROUPED, a9=1025), "n_group=1025")
    refused(lib, capfd, "matmul_mx_grouped", changed(GROUPED, a5=None), "needs n_rows=6")
    refused(lib, capfd, "matmul_mx_grouped", changed(GROUPED, a4=odder), "multiple of 4 bytes")
    refused(lib, capfd, "moe_gate_up_mx", changed(GATE_UP, a13=33), "n_ff=33 must be a multiple of 32")


def test_unaligned_codes(lib, capfd):
    for name, args, places in (("mx_quantize", QUANT, (3,)), ("mx_dequantize", VALUES, (0,)), ("add_rms_norm_mx", NORM, (6,)),
                               ("matmul_mx", DENSE, (0, 2)), ("matmul_mx_grouped", GROUPED, (0, 2)),
                               ("moe_gate_up_mx", GATE_UP, (0, 2, 4, 8))):
        for i in places:
            refused(lib, capfd, name, changed(args, **{f"a{i}": odd}), "codes must start on a multiple of 16 bytes")


def test_outputs_that_overlap_or_are_read_only(lib, capfd):
    for name, args, places in (("mx_quantize", QUANT, (3, 4)), ("mx_dequantize", VALUES, (5,)),
                               ("add_rms_norm_mx", NORM, (4, 5, 6, 7)), ("matmul_mx", DENSE, (4,)),
                               ("matmul_mx_grouped", GROUPED, (6,)), ("moe_gate_up_mx", GATE_UP, (8, 9))):
        for i in places:
            refused(lib, capfd, name, changed(args, **{f"a{i}": locked}), "read-only")
            for j, v in enumerate(args):
                if j == i or not isinstance(v, Handle) or (name == "add_rms_norm_mx" and i == 4 and j in (0, 1)):
                    continue
                # the last bytes of the other operand's first 16
                refused(lib, capfd, name, changed(args, **{f"a{i}": buf(MB, v.base)}), "overlaps")
    # the sum may be x or delta, but no other part of them
    refused(lib, capfd, "add_rms_norm_mx", changed(NORM, a4=buf(64 * MB, A.base + 64)), "overlaps")


def test_calls_that_are_accepted(lib, capfd):
    """The same arguments unchanged reach the device, which is not there: the refusals above are for their reasons."""
    if _native_device():
        pytest.skip("a device is there")
    for name, args in (("mx_quantize", QUANT), ("mx_dequantize", VALUES), ("add_rms_norm_mx", NORM),
                       ("add_rms_norm_mx", changed(NORM, a4=A)), ("add_rms_norm_mx", changed(NORM, a4=B)),
                       ("matmul_mx", DENSE), ("matmul_mx_grouped", GROUPED), ("moe_gate_up_mx", GATE_UP)):
        capfd.readouterr()
        assert getattr(lib, "ds3_hip_" + name)(*map(ref, args)) == -1
        assert "no HIP device" in capfd.readouterr().err


def _native_device():
    import torch
    return torch.cuda.device_count() > 0


def test_zero_rows_return_at_once(lib):
    for name, args in (("mx_quantize", changed(QUANT, a6=0)), ("mx_dequantize", changed(VALUES, a3=0)),
                       ("add_rms_norm_mx", changed(NORM, a9=0)), ("matmul_mx", changed(DENSE, a5=0)),
                       ("matmul_mx", changed(DENSE, a6=0)), ("matmul_mx_grouped", changed(GROUPED, a8=0)),
                       ("matmul_mx_grouped", changed(GROUPED, a7=0)), ("moe_gate_up_mx", changed(GATE_UP, a11=0))):
        assert getattr(lib, "ds3_hip_" + name)(*map(ref, args)) == 0, name


def test_python_refusals():
    m = ds3.MxMatrix(None, None, I8, 4, 64)
    w = ds3.MxMatrix(None, None, FP4, 6, 64)
    for call in (lambda: ds3.MxMatrix.nbytes(I8, 2, 40), lambda: ds3.MxMatrix.nbytes(F32, 2, 64),
                 lambda: ds3.matmul_mx(w, w, None), lambda: ds3.matmul_mx(m, m, None),
                 lambda: ds3.matmul_mx(ds3.MxMatrix(None, None, I8, 4, 96), w, None),
                 lambda: ds3.matmul_mx_grouped(m, w, None, None, 4, 4),
                 lambda: ds3.moe_gate_up_mx(m, w, w, None, ds3.MxMatrix(None, None, I8, 4, 64), 2),
                 lambda: ds3.add_rms_norm_mx(None, None, 1e-6, w)):
        with pytest.raises(ValueError):
            call()


def test_the_formats():
    """The test's own formats: every code is its own nearest value, and ties go to the even code."""
    for t in (FP4, I8):
        codes = np.tile(np.arange(256, dtype=np.uint8), (3, 1))
        scales = np.full((3, (512 if t == FP4 else 256) // 32), 127, np.uint8)
        v = X.values(t, codes, scales)
        v[np.abs(v) > 127 / 64] = 0 if t == I8 else v[np.abs(v) > 127 / 64]
        assert np.array_equal(X.values(t, *X.encode(t, v)), v)
    c, s = X.encode(FP4, np.r_[6.0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, np.zeros(24)][None])
    assert s[0, 0] == 127 and np.array_equal(X.values(FP4, c, s)[0, :8], [6, 0, 1, 1, 2, 2, 4, 4])
    c, s = X.encode(FP4, np.r_[7.0, 1, np.zeros(30)][None])
    assert s[0, 0] == 127 and np.array_equal(X.values(FP4, c, s)[0, :2], [6, 1])
    c, s = X.encode(FP4, np.r_[7.000001, 1, np.zeros(30)][None])
    assert s[0, 0] == 128
    c, s = X.encode(I8, np.r_[1.9999, 1 / 128, 3 / 128, np.zeros(29)][None])
    assert s[0, 0] == 127 and c[0, :3].tolist() == [127, 0, 2]
