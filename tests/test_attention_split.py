"""The split of paged attention's work (no device is needed): every run of keys is
one that the launch, the workspace and the join have room for, lengths near 2^30
and 2^31 included."""
import ctypes as C

import numpy as np
import pytest

from qw3_amd import _native

LAST = 2 ** 31 - 2 ** 16                             # positions that a table may have
NAMES = ("run", "tiles", "units", "grid", "joined", "partial")


@pytest.fixture(scope="module")
def lib():
    return _native._bind(C.CDLL(str(_native.LIB_DIR / "libds3_hip.so")), _native.SIGNATURES)


def split(lib, new, lens, heads, kv, dim, positions, block=1 << 16, window=0, rows=None):
    offsets = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    lens, out = np.asarray(lens, np.int32), (C.c_int64 * 12)()
    assert lib.ds3_hip_debug_attention_split(offsets.ctypes.data, lens.ctypes.data, rows or int(offsets[-1]), len(new), heads, kv,
                                             dim, block, positions // block, window, out) == 0
    return [dict(zip(NAMES, out[6 * i:6 * i + 6])) for i in range(2)]


def check(lib, new, lens, heads, kv, dim, positions, **more):
    group = heads // kv
    rows = [m * group for m in new]
    window = more.get("window", 0)
    both = split(lib, new, lens, heads, kv, dim, positions, **more)
    large = 256 if dim <= 128 else 128
    only_few = sum(new) <= len(new) or sum(rows) <= 64
    of = [[i for i, r in enumerate(rows) if r > 0 and not only_few and (r > 64 or len(new) == 1)]]
    of.append([i for i, r in enumerate(rows) if r > 0 and i not in of[0]])
    for s, mine, m in zip(both, of, (large, 16)):
        tiles = sum(-(-rows[i] // m) for i in mine)
        assert s["tiles"] == tiles
        if not mine:
            assert s["units"] == 0
            continue
        spans = {i: max(1, min(lens[i], positions)) for i in mine}
        if window:
            spans = {i: min(n, window + m // group + 130) for i, n in spans.items()}
        assert s["run"] > 0
        runs = {i: -(-n // s["run"]) for i, n in spans.items()}
        assert s["units"] == sum(runs[i] * -(-rows[i] // m) for i in mine)
        assert tiles <= s["units"] <= s["grid"], s
        if max(runs.values()) > 1:
            assert s["units"] <= s["partial"] and tiles <= s["joined"], s
            assert max(runs.values()) <= 512
    return both


@pytest.mark.parametrize("n", [1, 5000, 2 ** 29, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 2 ** 22, LAST - 1, LAST])
@pytest.mark.parametrize("new", [1, 40, 5000])
def test_one_request(lib, n, new):
    for heads, kv, dim in ((1, 1, 8), (32, 4, 128), (2048, 2048, 8), (16, 1, 256), (4096, 4, 8)):
        check(lib, [new], [n], heads, kv, dim, LAST)


@pytest.mark.parametrize("n_seq", [2, 3, 64, 65, 300, 2047, 2048, 2049, 5000])
def test_many_requests(lib, n_seq):
    """Single tokens and chunks, some beyond 2^30 keys, with fewer tiles than units are aimed at, as many and more."""
    rng = np.random.default_rng(n_seq)
    for most in (300, 2 ** 30 + 1, 2 ** 31 - 2 ** 22 + 1, LAST):
        for some in (1, n_seq // 2, n_seq):
            lens = rng.integers(1, 300, n_seq)
            lens[rng.permutation(n_seq)[:some]] = most
            for heads, kv, dim in ((8, 1, 8), (8, 4, 64), (64, 64, 8)):
                one = check(lib, [1] * n_seq, lens.tolist(), heads, kv, dim, LAST)
                if n_seq > 1 and n_seq * kv >= 2048:  # as many tiles as units: none is split
                    assert one[1]["units"] == one[1]["tiles"]
            new = rng.choice([0, 1, 1, 1, 20, 700], n_seq)
            new[0] = 700
            if new.sum() < 2 ** 20:
                check(lib, new.tolist(), lens.tolist(), 8, 2, 64, LAST)
                check(lib, new.tolist(), lens.tolist(), 8, 2, 256, LAST, window=2 ** 30 + 7)
                check(lib, new.tolist(), lens.tolist(), 8, 2, 64, LAST, window=1000)


def test_lengths_beyond_the_table(lib):
    """A table that holds less than a length: its positions count."""
    for positions in (1 << 16, 1 << 20):
        both = check(lib, [1, 1], [2 ** 31 - 1, 5], 8, 2, 64, positions)
        assert both[1]["units"] <= 2 + positions // both[1]["run"]
