"""Attention over the 8-bit cache for sequences that begin alike, of tables that have parted from their prefix: the
answer, against the plain form in 64 bits (prompts_model.py derives the tolerances), and what it costs.  Needs an MI355X."""
import sys
import time

import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prompts import DT, Dev, normal, off

pytestmark = pytest.mark.gpu


def say(*a):
    print("[gpu]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    c = X.Context(0)
    yield c
    c.close()


class Call:
    """N sequences of one new token after BLOCKS blocks alike, whose tables name PAGES pages again and again, and a call of
    attend_shared with SPLITS splits' scratch (None: all)."""

    def __init__(self, ctx, heads, kv, hd, n, blocks, splits=None, pages=96, part=None, new=1):
        rng = np.random.default_rng([61, n, blocks])
        table = np.tile(rng.integers(0, pages, blocks + 2), (n, 1))
        if part:
            part(table)
        self.ctx, self.heads, self.new = ctx, heads, [new] * n
        self.m = m = pm.Cache("fp16", n, kv, hd, pages, blocks + 2, table, rng)
        m.scales[:] = (np.abs(rng.standard_normal(m.scales.shape)) * 0.01 + 0.02).astype(np.float32)
        m.scales.view(np.uint32)[:] &= np.uint32(0xFFFFF000)
        m.tk[:], m.tv[:] = normal(rng, m.tk.shape, "fp16")[0], normal(rng, m.tv.shape, "fp16")[0]
        m.lens[:] = 64 * blocks + 1 + 3 * np.arange(n)
        self.d = Dev(ctx, m)
        self.s = X.Seqs(ctx, self.new)
        self.p = X.Prefixes(ctx, self.s, [0] * n, [blocks])
        qb, self.q = normal(rng, (n * new, heads, hd), "fp16")
        self.dq, self.o = X.DevBuf.of(ctx, qb), X.DevBuf(ctx, qb.shape, np.uint16)
        self.floats = X.attend_shared_part(self.s, self.p, heads, kv, hd, m.cols)
        assert self.floats != X.kv8_attend_part(self.s, heads, kv, hd, m.cols)
        if splits:
            assert new == 1
            self.floats = min(self.floats, splits * 2 * n * heads * (hd + 2) + 4 * n)
        self.part = X.DevBuf(ctx, (self.floats,), np.float32)

    def __call__(self):
        m, w = self.m, self.heads * self.m.hd
        X.attend_shared(self.ctx, self.d.h, self.s, self.p, self.heads, self.dq.h, w, 0.1, self.o.h, DT["bf16"], w, self.part.h,
                        self.floats)

    def worst(self):
        self()
        want, tol = self.m.attend(self.q, self.new, 0.1, "bf16")
        return off(pm.value(self.o.get(), "bf16"), want, tol)

    def took(self):
        self()
        self.ctx.sync()
        best = 1e9
        for _ in range(5):
            t = time.perf_counter()
            for _ in range(3):
                self()
            self.ctx.sync()
            best = min(best, (time.perf_counter() - t) / 3)
        return best


def parting(rows):
    def part(table):
        for i, at in rows.items():
            table[i, at] = (table[i, at] + 1 + i) % 96
    return part


# by sequence, the entries that are another page than the prefix's
PARTED = {"first block": {1: [0]}, "last block": {1: [299], 7: [298, 299]}, "middle": {1: [150], 2: [151], 3: [64], 4: [63]},
          "first sequence": {0: [100]}, "every split": {1: list(range(0, 300, 7)), 2: list(range(5, 300, 64))},
          "all": {i: list(range(300)) for i in range(8)}}


@pytest.mark.parametrize("heads,kv,hd", [(2, 2, 64), (4, 1, 64), (4, 2, 128), (16, 2, 128)])
@pytest.mark.parametrize("splits", [1, 2, 5, None], ids=str)
@pytest.mark.parametrize("where", PARTED)
def test_parted(ctx, where, splits, heads, kv, hd):
    """Splits of a few blocks and of hundreds."""
    say("parted", where, splits, heads, kv, hd)
    r = Call(ctx, heads, kv, hd, 8, 300, splits, part=parting(PARTED[where])).worst()
    say("worst", r)
    assert r <= 1


def test_a_parted_table_costs_no_more_than_its_blocks(ctx):
    """With scratch for one split, a table that parts half-way: twice the blocks take about twice the time (not four times,
    as a walk back through the split for each block would)."""
    took = []
    for blocks in (8000, 16000):
        c = Call(ctx, 1, 1, 64, 8, blocks, 1, part=parting({1: [blocks // 2]}))
        took.append(c.took())
        say(blocks, "blocks", took[-1])
    assert took[1] < 3 * took[0]
