"""Calls of the attention and sampling operators that the library refuses, each
with its diagnostic and before any device or buffer access."""
import ctypes as C

import pytest

from qw3_amd import _native, ds3
from test_mx_refusals import MB, Handle, buf, changed, lib, ref, refused          # noqa: F401

F32, F16 = ds3.TYPE_F32, ds3.TYPE_F16
A = [buf(64 * MB, (i + 1) << 30) for i in range(16)]
small = buf(1, 100 << 30)
odd = buf(64 * MB, (200 << 30) + 2)
eight = buf(64 * MB, (201 << 30) + 8)
locked = buf(64 * MB, 202 << 30, readonly=True)

TABLE = [A[0], 64, 1e6, 0, 1.0, 0.0, 0.0, 0]
ROPE = [A[0], F32, 1024, A[1], A[2], A[3], 1e-6, A[4], F32, 1024, 3, 4, 64, 64, False]
APPEND = [A[0], A[1], A[2], F32, 1024, 512, 512, A[3], A[4], A[5], A[6], A[7], 1e-6, A[8], F16, A[9], A[10], 3, 4, 2, 64, 64,
          False, 5, 16]
PLAN = [A[0], A[1], A[2], A[3], A[4], A[5], A[6], A[7], A[8], A[9], A[10], 3, 4, 20, 16, 64]
RELEASE = [A[0], A[1], A[2], A[3], A[4], 3, 4, 20, 16]
ATTN = [A[0], F32, 1024, A[1], A[2], A[3], A[4], A[5], A[6], 1024, 3, 2, 4, 2, 64, 5, 16, 4, 0.125, 0]
SAMPLE = [A[0], 400, A[1], A[2], A[3], A[4], A[5], A[6], A[7], 3, 100]
CALLS = {"rope_table": TABLE, "rope": ROPE, "rope_append": APPEND, "kv_plan": PLAN, "kv_release": RELEASE,
         "attention_paged": ATTN, "sample": SAMPLE}
OPTIONAL = {("rope", 5), ("rope_append", 10), ("rope_append", 11), ("rope_append", 9), ("sample", 3), ("sample", 4),
            ("sample", 5), ("sample", 6), ("sample", 8)}
OUTPUTS = {"rope_table": (0,), "rope": (7,), "rope_append": (13, 15, 16), "kv_plan": (2, 3, 6, 7, 8, 9, 10),
           "kv_release": (1, 3, 4), "attention_paged": (8,), "sample": (7, 8)}


@pytest.mark.parametrize("name", CALLS)
def test_missing_small_and_misplaced_buffers(lib, capfd, name):                  # noqa: F811
    args = CALLS[name]
    for i, v in enumerate(args):
        if not isinstance(v, Handle):
            continue
        if (name, i) not in OPTIONAL:
            refused(lib, capfd, name, changed(args, **{f"a{i}": None}))
        refused(lib, capfd, name, changed(args, **{f"a{i}": small}), "holds")
        refused(lib, capfd, name, changed(args, **{f"a{i}": odd}), "must start on a multiple")
        if i in OUTPUTS[name]:
            refused(lib, capfd, name, changed(args, **{f"a{i}": locked}), "read-only buffer")
            for j, w in enumerate(args):
                pairs = {("kv_plan", 2, 1), ("kv_plan", 6, 5), ("rope", 7, 0)}
                if isinstance(w, Handle) and j != i and (name, i, j) not in pairs and (name, j, i) not in pairs:
                    refused(lib, capfd, name, changed(args, **{f"a{i}": w}), "overlaps")


def test_heads(lib, capfd):                                                       # noqa: F811
    for name, args, dim, most in (("rope", ROPE, 12, 512), ("rope_append", APPEND, 20, 512), ("attention_paged", ATTN, 14, 256)):
        for bad in (0, 4, 12, most + 8):
            refused(lib, capfd, name, changed(args, **{f"a{dim}": bad}), "head_dim")
        refused(lib, capfd, name, changed(args, **{f"a{2 if dim != 20 else 4}": 1016}), "bytes apart")
        refused(lib, capfd, name, changed(args, **{f"a{2 if dim != 20 else 4}": 1032}), "multiple of 16")
        refused(lib, capfd, name, changed(args, a0=eight), "multiple of 16")
    for name, args, kv in (("rope_append", APPEND, 19), ("attention_paged", ATTN, 13)):
        for bad in (0, 3, 8):
            refused(lib, capfd, name, changed(args, **{f"a{kv}": bad}), "n_head")
    for name, args, types in (("rope", ROPE, (1, 8)), ("rope_append", APPEND, (3, 14)), ("attention_paged", ATTN, (1,))):
        for i in types:
            refused(lib, capfd, name, changed(args, **{f"a{i}": ds3.TYPE_Q8_0}), "neither F32 nor F16")


def test_rotary(lib, capfd):                                                      # noqa: F811
    for name, args, at in (("rope", ROPE, 13), ("rope_append", APPEND, 21)):
        for bad in (0, 7, 66):
            refused(lib, capfd, name, changed(args, **{f"a{at}": bad}), "rotary_dim")
    for bad in (0, 3, 514):
        refused(lib, capfd, "rope_table", changed(TABLE, a1=bad), "rotary_dim")
    nan, inf = float("nan"), float("inf")
    for at, bad in ((2, 1.0), (2, nan), (2, inf), (3, -1), (3, 4)):
        refused(lib, capfd, "rope_table", changed(TABLE, **{f"a{at}": bad}), "unsupported")
    refused(lib, capfd, "rope_table", changed(TABLE, a3=1, a4=0.0), "unsupported")
    for scaling in (2, 3):
        good = changed(TABLE, a3=scaling, a4=4.0, a5=1.0, a6=8.0, a7=4096)
        for at, bad in ((4, 0.0), (4, nan), (5, 0.0), (5, 8.0), (6, inf), (7, 0)):
            refused(lib, capfd, "rope_table", changed(good, **{f"a{at}": bad}), "unsupported")


def test_pages(lib, capfd):                                                       # noqa: F811
    for name, args, blocks, size in (("rope_append", APPEND, 23, 24), ("kv_plan", PLAN, 13, 14), ("kv_release", RELEASE, 7, 8),
                                     ("attention_paged", ATTN, 15, 16)):
        for bad in (0, 3, 48, 1 << 17):
            refused(lib, capfd, name, changed(args, **{f"a{size}": bad}), "no power of two")
        for bad in (0, 1 << 31, (1 << 27) + 1):
            refused(lib, capfd, name, changed(args, **{f"a{blocks}": bad}), "n_blocks")
    for name, args, at in (("kv_plan", PLAN, 12), ("kv_release", RELEASE, 6), ("attention_paged", ATTN, 17)):
        for bad in (0, 1 << 27):
            refused(lib, capfd, name, changed(args, **{f"a{at}": bad}), "max_blocks")
    for name, args, at in (("kv_plan", PLAN, 11), ("kv_release", RELEASE, 5), ("attention_paged", ATTN, 11)):
        for bad in (0, (1 << 20) + 1):
            refused(lib, capfd, name, changed(args, **{f"a{at}": bad}), "n_seq")
    refused(lib, capfd, "kv_plan", changed(PLAN, a15=0), "max_tokens")
    refused(lib, capfd, "rope_append", changed(APPEND, a0=None), "given together")
    refused(lib, capfd, "rope_append", changed(APPEND, a13=None), "given together")
    refused(lib, capfd, "rope_append", changed(APPEND, a7=None))


def test_attention_and_sampling_numbers(lib, capfd):                              # noqa: F811
    refused(lib, capfd, "attention_paged", changed(ATTN, a18=float("nan")), "scale")
    refused(lib, capfd, "attention_paged", changed(ATTN, a18=float("inf")), "scale")
    refused(lib, capfd, "attention_paged", changed(ATTN, a10=(1 << 20) + 1), "n_tokens")
    refused(lib, capfd, "attention_paged", changed(ATTN, a19=1 << 31), "window")
    refused(lib, capfd, "sample", changed(SAMPLE, a10=0), "n_vocab")
    refused(lib, capfd, "sample", changed(SAMPLE, a10=(1 << 18) + 1), "n_vocab")
    refused(lib, capfd, "sample", changed(SAMPLE, a9=(1 << 20) + 1), "n_rows")
    refused(lib, capfd, "sample", changed(SAMPLE, a1=396), "bytes apart")
    refused(lib, capfd, "sample", changed(SAMPLE, a1=402), "multiple of 4")


def test_table_during_a_capture(lib, capfd):                                      # noqa: F811
    assert lib.ds3_hip_debug_simulate_capture(1) == 0
    try:
        assert lib.ds3_hip_rope_table(*map(ref, TABLE)) == -1
        assert "rope_table is not allowed during graph capture" in capfd.readouterr().err
    finally:
        lib.ds3_hip_debug_simulate_capture(0)


def test_positions_near_the_end_of_int32(lib, capfd):                            # noqa: F811
    """Attention reads up to a few hundred keys ahead: its positions end 2^16 before 2^31."""
    huge = buf(1 << 40, 1 << 44)
    for block, most in ((1, 0x7fff0000), (16, 0x7fff000), (1 << 16, 0x7fff)):
        args = changed(ATTN, a4=huge, a15=1, a16=block)
        refused(lib, capfd, "attention_paged", changed(args, a17=most + 1), "max_blocks")


def test_scales_beyond_2_127(lib, capfd):                                        # noqa: F811
    for bad in (2.0 ** 127 * 1.001, -3e38, float("-inf")):
        refused(lib, capfd, "attention_paged", changed(ATTN, a18=bad), "scale")


def test_tiles_beyond_a_launch(lib, capfd):                                      # noqa: F811
    """2^23 workgroups of 256 or 512 threads are more than a launch has."""
    far = [buf(1 << 42, (i + 1) << 44) for i in range(7)]
    for heads, kv, tokens, seqs in ((8, 8, 1 << 20, 1 << 20), (1 << 16, 1 << 16, 1 << 15, 1), (1 << 16, 1, 1 << 20, 1)):
        stride = heads * 8 * 4
        args = [far[0], F32, stride, *far[1:6], far[6], stride, tokens, seqs, heads, kv, 8, 5, 16, 4, 0.125, 0]
        refused(lib, capfd, "attention_paged", args, "more than 2^23 - 1 tiles")


def test_heads_beyond_a_launch(lib, capfd):                                      # noqa: F811
    """2^24 workgroups of 256 threads are more than a launch has: here 2^26 groups of 64 lanes."""
    far = [buf(1 << 45, (i + 1) << 46) for i in range(11)]
    for tokens, heads, dim in ((1 << 26, 5, 512), (1 << 25, 6, 264), (1 << 12, 1 << 16, 512), (1 << 31, 1, 512)):
        row = heads * dim * 4
        args = [far[0], F32, row, far[1], far[2], far[3], 1e-6, far[4], F32, row, tokens, heads, dim, 64, False]
        refused(lib, capfd, "rope", args, "out of range" if tokens >> 31 else "more than 2^24 - 1 workgroups")
    args = [far[0], far[1], far[2], F32, 2048, 2048, 2048, far[3], far[4], far[5], far[6], far[7], 1e-6, far[8], F32, far[9],
            far[10], 1 << 26, 1, 1, 512, 64, False, 5, 16]
    refused(lib, capfd, "rope_append", args, "more than 2^24 - 1 workgroups")
