"""The microscaled products' launcher (no device is needed): the sizes that the
GPU tests take reach every kernel, variant and length of a wave's walk, the
lines of the rule, and counts near 2^31."""
import ctypes as C

import pytest

import _mx_plan as M
from qw3_amd import _native


@pytest.fixture(scope="module")
def lib():
    return _native._bind(C.CDLL(str(_native.LIB_DIR / "libds3_hip.so")), _native.SIGNATURES)


@pytest.mark.parametrize("kind", M.KINDS)
def test_the_sizes_take_their_kernels(lib, kind):
    got = {size: M.brief(M.plan(lib, kind, *size)) for size in M.KINDS[kind]}
    assert got == M.KINDS[kind]


def test_every_variant_is_reached():
    few = {(k, p[1]) for k, s in M.KINDS.items() for p in s.values() if p[0] == 0}
    assert few == {(k, w) for k in M.KINDS for w in (2, 4)}
    tile = {(k, p[1], p[2]) for k, s in M.KINDS.items() for p in s.values() if p[0] == 1}
    # one matrix: four waves only with 16 rows, eight otherwise; groups: all
    assert tile == {(k, w, r) for k in ("grouped", "gate_up") for w in (4, 8) for r in (16, 32, 48)} | \
        {("dense", 4, 16)} | {("dense", 8, r) for r in (16, 32, 48)}
    walks = {(k, p[1], p[2]) for k, s in M.KINDS.items() for p in s.values() if p[0] == 1 and p[4] >= 3}
    assert walks == tile - {("dense", 4, 16)}


def test_the_lines_of_the_rule(lib):
    def kernel(kind, *size):
        p = M.plan(lib, kind, *size)
        return p["kernel"], p["outputs"], p["waves"]
    # 16 x 64 blocks of products: 127 / 128, 255 / 256 (two chunks), 511 / 512
    assert kernel("dense", 9, 0, 127 * 64, 2048)[:2] == (0, 16) and kernel("dense", 9, 0, 128 * 64, 2048)[:2] == (0, 32)
    assert kernel("dense", 9, 0, 255 * 64, 1024) == (0, 32, 4) and kernel("dense", 9, 0, 256 * 64, 1024) == (0, 64, 2)
    assert kernel("dense", 9, 0, 511 * 64, 2048) == (0, 32, 4) and kernel("dense", 9, 0, 512 * 64, 2048)[0] == 1
    assert kernel("dense", 8, 0, 512 * 64, 2048) == (0, 64, 2)
    # the digits of 16, 32 and 48 rows fill the shared memory at 16, 7 and 5 chunks
    assert kernel("dense", 500, 0, 4128, 7680)[0] == 1 and kernel("dense", 500, 0, 4128, 7712)[0] == 0
    rows = [M.plan(lib, "dense", 6000, 0, 1056, k)["rows"] for k in (2560, 2592, 3584, 3616)]
    assert rows == [48, 32, 32, 16]
    # at most one row a group
    assert kernel("gate_up", 128, 128, 768, 2048)[0] == 0 and kernel("gate_up", 129, 128, 768, 2048)[0] == 1
    # two waves a SIMD with a tile each
    assert [M.plan(lib, "dense", m, 0, 4096, 2048)["beside"] for m in (512, 992, 1024)] == [0, 0, 1]


def test_counts_near_2_31(lib):
    top = 2 ** 31 - 1
    for n in (top, top - 62, top - 63, top - 64):
        for rows in (1, 9):
            p = M.plan(lib, "dense", rows, 0, n, 32)
            assert p["tiles"] == -(-n // p["outputs"]) and 0 < p["span"] <= p["tiles"]
    for groups, kind, n in ((1, "grouped", 1), (1024, "grouped", 1), (7, "gate_up", 32)):
        p = M.plan(lib, kind, top, groups, n, 32)
        assert p["kernel"] == 1 and p["tiles"] == p["span"] == 1


def test_sizes_that_no_product_takes(lib):
    v = (C.c_int64 * 7)()
    for size in ((0, 0, 5, 64, False), (3, 0, 0, 64, False), (3, 0, 5, 48, False), (3, 1025, 5, 64, False), (3, 0, 32, 64, True),
                 (3, 2, 33, 64, True), (1 << 31, 0, 5, 64, False)):
        assert lib.ds3_hip_debug_mx_plan(*size, v) == -1, size
    assert lib.ds3_hip_debug_mx_plan(3, 0, 5, 64, False, None) == -1
