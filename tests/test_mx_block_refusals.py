"""Calls of the microscaled FFN block and of the combine that the library
refuses, before any device or buffer access (no device is needed)."""
import pytest

from qw3_amd import ds3
from test_mx_refusals import (A, B, D, E, F32, FP4, G, H, I8, J, K, L, MB, Handle, _native_device, buf, changed, lib, locked,
                              odd, odder, ref, refused, small)

M, N, O, Q, R, S = (buf(64 * MB, (i + 300) << 30) for i in range(6))
COMBINE = [A, B, D, E, 3, 2, 5, 64, True]
#        hidden delta norm eps  router gate  up    down  logits idx scores T E  X  k  F  stride
BLOCK = [A, B, D, 1e-6, E, G, H, J, K, L, M, N, O, Q, 3, 64, 8, 2, 32, 256, F32, True]
OUT = {"moe_combine": (3,), "moe_block_mx": (0, 11, 12, 13)}
OPTIONAL = {"moe_combine": (), "moe_block_mx": (1, 11, 12, 13)}
BOTH = pytest.mark.parametrize("name,args", [("moe_combine", COMBINE), ("moe_block_mx", BLOCK)])


@BOTH
def test_missing_and_small_buffers(lib, capfd, name, args):
    for i, v in enumerate(args):
        if isinstance(v, Handle):
            if i not in OPTIONAL[name]:
                refused(lib, capfd, name, changed(args, **{f"a{i}": None}))
            refused(lib, capfd, name, changed(args, **{f"a{i}": small}), "holds")


@BOTH
def test_outputs_that_overlap_or_are_read_only(lib, capfd, name, args):
    for i in OUT[name]:
        refused(lib, capfd, name, changed(args, **{f"a{i}": locked}), "read-only")
        for j, v in enumerate(args):
            if j != i and isinstance(v, Handle):
                refused(lib, capfd, name, changed(args, **{f"a{i}": buf(MB, v.base)}), "overlaps")


@BOTH
def test_accepted_and_empty(lib, capfd, name, args):
    tokens = {"moe_combine": 4, "moe_block_mx": 14}[name]
    assert getattr(lib, "ds3_hip_" + name)(*map(ref, changed(args, **{f"a{tokens}": 0}))) == 0
    if _native_device():
        pytest.skip("a device is there")
    for a in (args, changed(args, **{f"a{i}": None for i in OPTIONAL[name]})):
        capfd.readouterr()
        assert getattr(lib, "ds3_hip_" + name)(*map(ref, a)) == -1
        assert "no HIP device" in capfd.readouterr().err


def test_sizes_and_types(lib, capfd):
    refused(lib, capfd, "moe_combine", changed(COMBINE, a5=0))
    refused(lib, capfd, "moe_combine", changed(COMBINE, a7=0))
    refused(lib, capfd, "moe_combine", changed(COMBINE, a4=1 << 31), "out of range")
    refused(lib, capfd, "moe_combine", changed(COMBINE, a0=odder), "multiple of 4 bytes")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a3=-1.0))
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a14=0xffffffff), "out of range")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a14=0x40000000), "out of range")       # tokens x slots
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a15=48, a19=192), "n_embd=48 must be a multiple of 32")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a18=16), "n_ff_exp=16 must be a multiple of 32")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a16=0))
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a17=9))                                # more slots than experts
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a16=257), "n_expert=257")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a16=32, a17=17), "n_used=17")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a19=252), "router rows")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a20=99), "router rows")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a1=odder), "multiple of 4 bytes")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a4=odder), "multiple of 4 bytes")
    for i in (5, 7, 9):
        refused(lib, capfd, "moe_block_mx", changed(BLOCK, **{f"a{i}": odd}), "codes must start on a multiple of 16 bytes")


def test_python_refusals():
    g, d, bad = (ds3.MxMatrix(None, None, t, r, c) for t, r, c in ((FP4, 8 * 32, 64), (FP4, 8 * 64, 32), (I8, 8 * 32, 64)))
    for mats, n_expert in (((g, bad, d), 8), ((g, g, g), 8), ((g, g, d), 7), ((g, d, d), 8)):
        with pytest.raises(ValueError):
            ds3.moe_block_mx(None, None, 1e-6, None, F32, *mats, 3, n_expert, 2)


def test_more_tokens_than_a_launch_routes(lib, capfd):
    """The router's launch ends below 2^26 tokens; the call says so before hidden is written."""
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a14=1 << 26), "n_tokens=67108864 is out of range")
    refused(lib, capfd, "moe_block_mx", changed(BLOCK, a14=(1 << 26) - 1), "holds")
