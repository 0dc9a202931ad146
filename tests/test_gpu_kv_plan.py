"""The step's plan of blocks, positions and slots against the rule, request by request."""
import numpy as np
import pytest

import _decode as D
from qw3_amd import ds3

pytestmark = pytest.mark.gpu


class State:
    def __init__(self, seed, n_seq, block, n_blocks, max_blocks):
        self.rng = np.random.default_rng(seed)
        self.block, self.n_blocks, self.max_blocks = block, n_blocks, max_blocks
        self.lens = np.zeros(n_seq, np.int32)
        self.table = np.full((n_seq, max_blocks), -7, np.int32)
        self.free = self.rng.permutation(n_blocks).astype(np.int32)
        self.n_free = n_blocks
        self.dev = [D.ints(self.lens), D.ints(self.table), D.ints(self.free), D.ints([n_blocks])]

    def want(self, new, max_tokens):
        """The plan by the rule; (carried out, offsets, positions, slots, status)."""
        new, b = np.maximum(new, 0).astype(np.int64), self.block
        lens, table = self.lens + new, self.table.copy()
        had, have = -(-self.lens.astype(np.int64) // b), -(-lens // b)
        most = 2 ** 31 - 1                            # counts are held to int32
        fresh = int(np.where(new > 0, have - had, 0).sum())
        status = [min(int(new.sum()), most), min(fresh, most), min(max(0, fresh - self.n_free), most),
                  int((have > self.max_blocks).sum())]
        done = status[2] == 0 and status[3] == 0 and status[0] <= max_tokens
        taken, pos, slots = 0, [], []
        for i in range(len(new) if done else 0):
            for j in range(had[i], have[i] if new[i] else had[i]):
                table[i, j] = self.free[self.n_free - 1 - taken]
                taken += 1
            for p in range(int(self.lens[i]), int(lens[i])):
                pos.append(p)
                slots.append(table[i, p // b] * b + p % b)
        offsets = np.concatenate(([0], np.cumsum(new))) if done else np.zeros(len(new) + 1, int)
        pad = max_tokens - len(pos)
        if done:
            self.lens, self.table, self.n_free = lens.astype(np.int32), table, self.n_free - taken
        return done, offsets, np.r_[pos, np.zeros(pad)].astype(int), np.r_[slots, -np.ones(pad)].astype(int), status

    def step(self, new, max_tokens, apart=False):
        lens, table, free, n_free = self.dev
        n = len(new)
        out = [ds3.Buffer.from_array(np.full(k, 99, np.int32)) for k in (n + 1, max_tokens, max_tokens, 4)]
        lens2, n_free2 = (D.ints(np.full(n, 5)), D.ints([5])) if apart else (None, None)
        ds3.kv_plan(D.ints(new), lens, table, free, n_free, *out, n, self.max_blocks, self.n_blocks, self.block, max_tokens,
                    kv_lens_out=lens2, n_free_out=n_free2)
        if apart:
            assert np.array_equal(lens.read(np.int32, n), self.lens) and n_free.read(np.int32, 1)[0] == self.n_free
            self.dev[0], self.dev[3] = lens2, n_free2
        done, *want, status = self.want(np.asarray(new), max_tokens)
        for buf, w in zip(out, want):
            assert np.array_equal(buf.read(np.int32, len(w)), w)
        assert out[3].read(np.int32, 4).tolist() == status
        self.check()
        return done

    def check(self):
        n = len(self.lens)
        assert np.array_equal(self.dev[0].read(np.int32, n), self.lens)
        assert np.array_equal(self.dev[1].read(np.int32, self.table.shape), self.table)
        assert np.array_equal(self.dev[2].read(np.int32, self.n_blocks), self.free)
        assert self.dev[3].read(np.int32, 1)[0] == self.n_free

    def release(self, done):
        lens, table, free, n_free = self.dev
        n = len(done)
        ds3.kv_release(D.ints(done), lens, table, free, n_free, n, self.max_blocks, self.n_blocks, self.block)
        for i in range(n):
            if done[i]:
                for j in range(-(-int(self.lens[i]) // self.block)):
                    self.free[self.n_free] = self.table[i, j]
                    self.n_free += 1
                self.lens[i] = 0
        self.check()


@pytest.mark.parametrize("n_seq,block,max_tokens", [(1, 16, 40), (3, 1, 64), (8, 16, 200), (70, 4, 2048), (70, 4, 2049),
                                                    (1100, 8, 9000), (2500, 2, 2048)])
def test_steps(hip_ready, n_seq, block, max_tokens):
    s = State(n_seq, n_seq, block, 40 * n_seq, 60)
    for i in range(8):
        most = max(1, min(30, 2 * max_tokens // n_seq)) if i % 3 == 0 else 1
        new = s.rng.integers(-1, most + 1, n_seq)
        if new.clip(0).sum() > max_tokens:
            new = (s.rng.random(n_seq) < 0.5 * max_tokens / n_seq).astype(int)
        assert s.step(new, max_tokens, apart=i % 2 == 1)
        if i % 3 == 2:
            s.release((s.rng.random(n_seq) < 0.4).astype(int))
    used = s.table[np.arange(s.max_blocks) < -(-s.lens // block)[:, None]]
    assert sorted([*used, *s.free[:s.n_free]]) == list(range(s.n_blocks))        # every block in one place


def test_plans_that_are_not_carried_out(hip_ready):
    s = State(1, 4, 8, 10, 5)
    assert s.step([9, 0, 8, 1], 32)                   # 2 + 1 + 1 blocks of 10
    assert not s.step([20, 20, 20, 0], 64)            # lacks blocks
    assert not s.step([40, 0, 0, 0], 64)              # a table row too short
    assert not s.step([2 ** 31 - 1, 2 ** 31 - 1, 5, 5], 64)
    assert not s.step([1, 1, 1, 1], 3)                # more tokens than rows
    assert s.step([1, 1, 1, 1], 4)
    assert s.step([0, 0, 0, 0], 4)
    assert not s.step([3000] * 4, 4000)
    s.release([1, 1, 1, 1])
    assert s.step([40, 40, 0, 0], 4000)               # every block
    lens, table, free, n_free = s.dev
    ds3.kv_release(D.ints([1, 0, 0, 0]), D.ints([40, 0, 0, 0]), table, free, D.ints([8]), 4, 5, 10, 8)
    assert np.array_equal(free.read(np.int32, 10), s.free)                       # five more do not fit


def test_tables_that_name_no_block(hip_ready):
    """Entries outside the cache, as a caller may have left them: no slot."""
    table = D.ints([[0, 50, 2], [-3, 1, 1]])
    pos, slots, offsets, status = (ds3.Buffer.alloc(4 * k) for k in (8, 8, 3, 4))
    ds3.kv_plan(D.ints([2, 2]), D.ints([6, 1]), table, D.ints([3, 4, 0, 0, 0]), D.ints([99]), offsets, pos, slots, status, 2, 3, 5, 4, 8,
                kv_lens_out=ds3.Buffer.alloc(8), n_free_out=ds3.Buffer.alloc(4))
    assert slots.read(np.int32, 8).tolist() == [-1, -1, -1, -1, -1, -1, -1, -1]
    assert pos.read(np.int32, 8).tolist() == [6, 7, 1, 2, 0, 0, 0, 0]


@pytest.mark.parametrize("n_seq", [64, 1024, 3000])
def test_requests_too_long_in_every_wave(hip_ready, n_seq):
    """One request longer than its table row, in any wave, refuses the plan; the count of such requests is exact."""
    s = State(n_seq + 1, n_seq, 4, 8 * n_seq, 6)
    assert s.step([1] * n_seq, n_seq)
    for at in [*range(0, n_seq, 61), n_seq - 1]:
        new = np.zeros(n_seq, int)
        new[at] = 24                                  # 25 tokens of at most 24
        assert not s.step(new, 4096)
    assert not s.step([24] * n_seq, 24 * n_seq)
    assert s.step([23] + [0] * (n_seq - 1), 4096)
