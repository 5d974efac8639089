"""Attention over the 8-bit cache for sequences that begin alike, on the GPU, against the plain form in 64
bits that the cache's attention is tested with (prompts_model.py, which derives the tolerances: sums in
any order, joined or not, are within them).  Needs an MI355X."""
import ctypes
import sys

import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prompts import DT, Dev, normal, off, strided

pytestmark = pytest.mark.gpu


def say(*a):
    print("[gpu]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    c = X.Context(0)
    yield c
    c.close()


def alike(ctx, dt, kv, hd, of, blocks, before, rng, cols=None, spare=4):
    """A cache of sequences with BEFORE tokens each, the first BLOCKS[OF] blocks of them on shared pages."""
    n = len(of)
    cols = cols or max(before) // 64 + 4
    pages = sum(blocks) + n * cols + spare
    free = list(rng.permutation(pages))
    shared = [[free.pop() for _ in range(b)] for b in blocks]
    table = [(shared[g] if g >= 0 else [])[:cols] for g in of]
    table = [t + [free.pop() for _ in range(cols - len(t))] for t in table]
    m = pm.Cache(dt, n, kv, hd, pages, cols, table, rng)
    # what the pages and tails would hold after the tokens before
    m.scales[:] = (np.abs(rng.standard_normal((pages, kv, 2))) * 0.01 + 0.02).astype(np.float32)
    u = m.scales.view(np.uint32)
    u &= np.uint32(0xFFFFF000)
    m.tk[:], m.tv[:] = normal(rng, m.tk.shape, dt)[0], normal(rng, m.tv.shape, dt)[0]
    m.lens[:] = before
    return m, Dev(ctx, m)


def step(ctx, m, d, of, blocks, new, heads, odt, rng, cap=None, scale=None):
    """Append NEW tokens and attend with shared prefixes: the worst distance over its tolerance."""
    rows, kv, hd = sum(new), m.kv, m.hd
    kb, _ = normal(rng, (rows, kv, hd), m.dt)
    vb, _ = normal(rng, (rows, kv, hd), m.dt)
    qb, q = normal(rng, (rows, heads, hd), m.dt)
    scale = hd ** -0.5 if scale is None else scale
    s = X.Seqs(ctx, new)
    p = X.Prefixes(ctx, s, of, blocks)
    dk, dv, dq = X.DevBuf.of(ctx, kb), X.DevBuf.of(ctx, vb), X.DevBuf.of(ctx, strided(qb, 24))
    o = X.DevBuf.of(ctx, np.full((rows + 1, heads * hd + 8), 0x1234, np.uint16))
    X.kv8_append(ctx, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    floats = floats if cap is None else cap(floats)
    scratch = X.DevBuf.of(ctx, np.full(floats + 4, np.nan, np.float32))
    X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd + 24, scale, o.h, DT[odt], heads * hd + 8,
                    scratch.h if floats else None, floats)
    m.append(kb, vb, new)
    got = o.get()
    assert np.isnan(scratch.get()[floats:]).all()
    assert (got[rows:] == 0x1234).all() and (got[:, heads * hd:] == 0x1234).all()
    want, tol = m.attend(q, new, scale, odt)
    r = off(pm.value(got[:rows, :heads * hd], odt).reshape(want.shape), want, tol)
    X.kv8_advance(ctx, d.h, s)
    m.advance(new)
    return r


# of, blocks, tokens of its own before the step, new tokens
SHAPES = {
    "two": ([0, 0], [2], [5, 60], [1, 1]),
    "new blocks": ([0, 0, 0], [1], [63, 0, 127], [1, 1, 1]),
    "chunks": ([0, 0, 0], [3], [10, 64, 0], [40, 1, 129]),
    "mixed": ([1, 0, -1, 0, 1, -1], [4, 2], [3, 70, 100, 0, 64, 0], [1, 1, 1, 1, 1, 2]),
    "waiting": ([0, 0, 0, 0], [2], [0, 5, 9, 70], [0, 3, 0, 1]),
    "many": ([i % 3 - 1 for i in range(40)], [5, 1], [(7 * i) % 90 for i in range(40)], [1] * 40),
    "long rows": ([0, 0], [6], [30, 0], [300, 65]),
    "one alone": ([0, 1], [3, 2], [9, 9], [1, 1]),
}


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (8, 1, 64), (3, 3, 128), (12, 4, 64), (5, 1, 128), (32, 2, 64),
                                         (11, 1, 128), (17, 1, 64)])
@pytest.mark.parametrize("shape", SHAPES)
def test_shared(ctx, shape, heads, kv, hd, dt, odt):
    of, blocks, own, new = SHAPES[shape]
    rng = np.random.default_rng([len(of), heads, hd])
    say("shared", shape, heads, kv, hd, dt, odt)
    before = [n + 64 * (blocks[g] if g >= 0 else 0) for n, g in zip(own, of)]
    m, d = alike(ctx, dt, kv, hd, of, blocks, before, rng)
    for _ in range(2):
        r = step(ctx, m, d, of, blocks, new, heads, odt, rng)
        say("worst", r)
        assert r <= 1


# as above, with prefixes long enough, and of enough sequences, that their blocks are read once for all (the plan decides by
# both): rows of a prefix that fill one tile of 16, two, half a tile of 128, several
LONG = {
    "eight": ([0] * 8, [17], [5, 60, 0, 63, 64, 127, 1, 300], [1] * 8),
    "new blocks": ([0] * 9, [18], [63] * 4 + [126] * 5, [1] * 9),
    "two prefixes and some alone": ([i % 3 - 1 for i in range(24)], [17, 29], [(31 * i) % 200 for i in range(24)], [1] * 24),
    "waiting": ([0] * 12, [20], [(17 * i) % 70 for i in range(12)], [i % 2 for i in range(12)]),
    "three tokens": ([0] * 10 + [-1], [19], [(41 * i) % 150 for i in range(10)] + [700], [3, 1, 2, 3, 0, 3, 2, 2, 1, 3, 3]),
    "sixteen": ([0] * 16, [21], [(13 * i) % 130 for i in range(16)], [1] * 16),
    "forty": ([0] * 40, [17], [(7 * i) % 90 for i in range(40)], [1] * 40),
    "long tails": ([0] * 8, [17], [1200, 3, 900, 0, 2000, 640, 64, 63], [1] * 8),
    "a long and a short": ([0, 0, 0, 0, 1, 1, 1, 1], [50, 1], [3, 70, 64, 0, 9, 500, 64, 1], [1] * 8),
}


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 1, 64), (3, 3, 128), (4, 2, 64), (5, 1, 128), (16, 1, 64), (2, 2, 64)])
@pytest.mark.parametrize("shape", LONG)
def test_long_shared(ctx, shape, heads, kv, hd, dt, odt):
    of, blocks, own, new = LONG[shape]
    rng = np.random.default_rng([len(of), heads, hd])
    say("long shared", shape, heads, kv, hd, dt, odt)
    before = [n + 64 * (blocks[g] if g >= 0 else 0) for n, g in zip(own, of)]
    m, d = alike(ctx, dt, kv, hd, of, blocks, before, rng)
    for _ in range(2):
        r = step(ctx, m, d, of, blocks, new, heads, odt, rng)
        say("worst", r)
        assert r <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,seqs,tokens", [(2, 1, 64, 2, 30000), (4, 1, 64, 8, 70000), (4, 1, 128, 8, 66000),
                                                     (4, 2, 128, 3, 14000), (8, 1, 128, 8, 20000), (8, 1, 64, 30, 9000)])
def test_very_long_prefixes(ctx, heads, kv, hd, seqs, tokens, dt):
    """Tens of thousands of keys: two tiles of rows a workgroup, few sequences, 128 splits."""
    rng = np.random.default_rng([32, seqs])
    of, blocks = [0] * seqs, [tokens // 64]
    say("very long", heads, kv, hd, seqs, tokens, dt)
    m, d = alike(ctx, dt, kv, hd, of, blocks, [blocks[0] * 64 + (37 * i) % 400 for i in range(seqs)], rng)
    assert step(ctx, m, d, of, blocks, [1] * seqs, heads, "bf16", rng) <= 1


def test_long_tables_that_are_not_alike(ctx):
    """Tables that part at a split's first block, within one, at the last, at several; that meet again; lengths under the
    prefix; pages that are none, alike and not; the first sequence's own table and length odd."""
    rng = np.random.default_rng(33)
    say("long not alike")
    for heads, kv, hd, n in ((2, 2, 64, 12), (4, 2, 128, 12), (4, 1, 64, 30), (4, 1, 128, 14)):
        of, blocks, b = [0] * n, [30], 30
        before = [b * 64 + (29 * i) % 150 for i in range(n)]
        before[3], before[5], before[7] = 100, 0, 64 * 17 + 63
        m, d = alike(ctx, "fp16", kv, hd, of, blocks, before, rng, cols=36)
        other = lambda i, j: m.table[i, 35 - j % 3]
        m.table[1, 0] = other(1, 0)
        m.table[2, 29] = other(2, 1)
        m.table[4, [7, 8, 20]] = [other(4, 0), other(4, 1), -1]
        m.table[6, 2:30:3] = [other(6, j) for j in range(10)]
        m.table[8, 10:] = m.table[9, 10:][::-1]
        m.table[[0, 9, 10], 16] = 1 << 30          # no page, in some and in the first's
        m.table[11, 12] = -7
        d.b["table"].upload(m.table)
        for blocks in ([30], [20], [36], [1 << 20]):
            r = step(ctx, m, d, of, blocks, [1] * n, heads, "bf16", rng)
            say(blocks, "worst", r)
            assert r <= 1
        m.lens[0] = 0                              # the first sequence begins anew: its table is what counts
        d.b["lens"].upload(m.lens)
        assert step(ctx, m, d, of, [30], [1] * n, heads, "fp16", rng) <= 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [None, 0.5, 0.2, 0.05, 0], ids=str)
def test_scratch(ctx, cap, hd):
    """All of the scratch, some (fewer splits), too little for one split of each, none: the same answer."""
    rng = np.random.default_rng(21)
    of, blocks, new = [0] * 5 + [1] * 3, [40, 33], [1] * 8
    say("scratch", cap, hd)
    before = [64 * blocks[g] + 11 * i for i, g in enumerate(of)]
    m, d = alike(ctx, "fp16", 2, hd, of, blocks, before, rng)
    assert step(ctx, m, d, of, blocks, new, 8, "fp16", rng, None if cap is None else lambda n: int(n * cap) // 4 * 4) <= 1


@pytest.mark.parametrize("heads,kv,hd,seqs,new", [(8, 2, 128, 2, 1), (8, 2, 128, 40, 1), (16, 1, 64, 20, 1), (8, 2, 64, 3, 50)])
def test_long_prefixes(ctx, heads, kv, hd, seqs, new):
    """Thousands of keys, split over the chip."""
    rng = np.random.default_rng([22, seqs])
    of, blocks = [0] * seqs, [90]
    say("long prefix", heads, kv, hd, seqs, new)
    m, d = alike(ctx, "bf16", kv, hd, of, blocks, [90 * 64 + (37 * i) % 400 for i in range(seqs)], rng)
    assert step(ctx, m, d, of, blocks, [new] * seqs, heads, "bf16", rng) <= 1


def test_tables_that_are_not_alike(ctx):
    """What the plan calls shared is a hint: tables that part early, at the first block, lengths under the prefix, pages
    that are none, a prefix longer than the table -- each sequence sees its own."""
    rng = np.random.default_rng(23)
    say("not alike")
    for heads, kv, hd, new in ((4, 2, 64, [1] * 9), (8, 1, 128, [30, 1, 2, 40, 1, 5, 9, 1, 70])):
        of, blocks = [0] * 8 + [-1], [5]
        before = [330, 331, 400, 322, 350, 100, 0, 321, 10]
        m, d = alike(ctx, "fp16", kv, hd, of, blocks, before, rng, cols=9)
        m.table[1, 3] = m.table[8, 3]          # parts at its fourth block
        m.table[2, 0] = m.table[8, 0]          # at its first
        m.table[3, 4] = -1                     # at its last, which is no page
        m.table[0, 2] = m.table[4, 2] = m.table[7, 2] = 1 << 30        # no page, alike
        d.b["table"].upload(m.table)
        for blocks in ([5], [9], [1 << 20]):
            assert step(ctx, m, d, of, blocks, new, heads, "bf16", rng) <= 1
    # the first sequence's own length under the prefix: its table is what the others are held against all the same
    m, d = alike(ctx, "fp16", 2, 64, [0] * 3, [4], [20, 300, 301], rng)
    assert step(ctx, m, d, [0] * 3, [4], [1] * 3, 4, "bf16", rng) <= 1


def test_full_tables(ctx):
    """A sequence whose table is full keeps no new token; with all its blocks shared it has none of its own."""
    rng = np.random.default_rng(24)
    say("full tables")
    for new in (1, 2):
        n = 9
        m, d = alike(ctx, "bf16", 2, 128, [0] * n, [18], [18 * 64] * 4 + [18 * 64 - 1, 18 * 64 - 64] + [1 << 30, -5, 1], rng, cols=18)
        assert step(ctx, m, d, [0] * n, [18], [new] * n, 4, "bf16", rng) <= 1
    for new in ([1, 1, 1], [20, 3, 70]):
        m, d = alike(ctx, "bf16", 2, 128, [0] * 3, [4], [256, 256, 250], rng, cols=4)
        assert step(ctx, m, d, [0] * 3, [4], new, 4, "bf16", rng) <= 1
    m, d = alike(ctx, "bf16", 2, 64, [0] * 3, [4], [1 << 30, -5, 256], rng, cols=4)
    assert step(ctx, m, d, [0] * 3, [4], [1, 1, 1], 4, "fp16", rng) <= 1


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_blocks_that_are_not_finite(ctx, dt, bad, new):
    """A block of the prefix that is not finite, seen by the sequences that share it and by no other; a hidden value of a
    tail that is not finite, by none."""
    rng = np.random.default_rng(25)
    say("not finite", dt, bad, new)
    kv, hd, heads, of, blocks = 2, 64, 8, [0, 0, 0, -1], [3]
    m, d = alike(ctx, dt, kv, hd, of, blocks, [200, 202, 210, 70], rng)
    m.table[2, 1] = m.table[3, 2]              # the third parts before the spoilt block
    spoilt = m.table[0, 1]
    m.scales[spoilt, 1, 1] = np.nan
    # its tail's later rows hold anything
    pat = pm.bits(np.float32(bad), dt)[0]
    total = [n + new for n in (200, 202, 210, 70)]
    for i, n in enumerate(total):
        m.tk[i, :, n % 64:], m.tv[i, :, n % 64:] = pat, pat
    for n in ("table", "scales", "tk", "tv"):
        d.b[n].upload(getattr(m, n))
    s = X.Seqs(ctx, [new] * 4)
    p = X.Prefixes(ctx, s, of, blocks)
    qb, q = normal(rng, (4 * new, heads, hd), dt)
    kb, _ = normal(rng, (4 * new, kv, hd), dt)
    vb, _ = normal(rng, (4 * new, kv, hd), dt)
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (4 * new, heads, hd), np.uint16)
    X.kv8_append(ctx, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd, 0.125, o.h, DT[dt], heads * hd, part.h, floats)
    got = pm.value(o.get(), dt).reshape(4, new, heads, hd)
    with np.errstate(invalid="ignore"):
        m.append(kb, vb, [new] * 4)
    m.scales[spoilt, 1, 1] = 0.03
    # a tail whose live rows were spoilt too and that the step filled: its block is not finite as a whole
    filled = [i for i in range(4) if np.isnan(m.scales[m.table[i, :total[i] // 64]]).any()]
    assert filled == ([2] if new == 50 else []) and np.isnan(got[filled]).all()
    m.scales[np.isnan(m.scales)] = 0.03
    m.tk[~np.isfinite(pm.value(m.tk, dt))] = 0
    m.tv[~np.isfinite(pm.value(m.tv, dt))] = 0
    want, tol = (x.reshape(got.shape) for x in m.attend(q, [new] * 4, 0.125, dt))
    assert np.isnan(got[:2, :, heads // 2:]).all()
    same = np.ones(got.shape, bool)
    same[:2, :, heads // 2:] = False
    same[filled] = False
    assert (abs(got - want)[same] <= tol[same]).all()


@pytest.mark.parametrize("heads", [2, 4, 8])
@pytest.mark.parametrize("bad", [np.nan, np.inf, "scale"])
def test_long_prefix_with_a_block_that_is_not_finite(ctx, bad, heads):
    """A spoilt block of the prefix is seen by the sequences that share it, and by none whose table has parted before it; a
    sequence's own spoilt block by itself alone; infinite scores in the prefix as in a sequence's own."""
    rng = np.random.default_rng(34)
    say("long not finite", bad, heads)
    kv, hd, n, of, blocks = 2, 128, 14, [0] * 14, [24]
    m, d = alike(ctx, "bf16", kv, hd, of, blocks, [24 * 64 + 70 + 5 * i for i in range(n)], rng)
    m.table[3, 2] = m.table[3, -1]
    m.table[4, 11] = m.table[4, -1]
    value = np.nan if bad == "scale" else bad
    m.scales[m.table[0, 11], 1, 1] = value                  # values of the second head's twelfth block
    m.scales[m.table[6, 24], 0, 0] = np.nan                 # a sequence's own keys
    d.b["table"].upload(m.table)
    d.b["scales"].upload(m.scales)
    s = X.Seqs(ctx, [1] * n)
    p = X.Prefixes(ctx, s, of, blocks)
    qb, q = normal(rng, (n, heads, hd), "bf16")
    dq, o = X.DevBuf.of(ctx, qb), X.DevBuf(ctx, (n, heads, hd), np.uint16)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
    got = pm.value(o.get(), "bf16")
    half = heads // 2
    sees = [i for i in range(n) if i != 4]                  # the fourth has parted there and only there
    assert not np.isfinite(got[sees][:, half:]).any() and np.isnan(got[6, :half]).all()
    m.scales[~np.isfinite(m.scales)] = 0.03
    want, tol = m.attend(q, [1] * n, 0.09, "bf16")
    same = np.zeros(got.shape, bool)
    same[:, :half] = True
    same[4] = True
    same[6, :half] = False
    assert (abs(got - want)[same] <= tol[same]).all()


@pytest.mark.parametrize("scale", [0.0, 3.0, 1e-4])
def test_sharp_and_flat(ctx, scale):
    """Scores of hundreds, in the prefix or outside of it, and of nothing."""
    rng = np.random.default_rng(26)
    say("scale", scale)
    for heads, kv in ((2, 2), (4, 2), (4, 1)):
        of, blocks = [0] * 12, [19]
        m, d = alike(ctx, "fp16", kv, 128, of, blocks, [19 * 64 + 51 * i for i in range(12)], rng)
        assert step(ctx, m, d, of, blocks, [1] * 12, heads, "bf16", rng, scale=scale) <= 1
    for new in (1, 40):
        of, blocks = [0] * 4, [7]
        m, d = alike(ctx, "bf16", 2, 128, of, blocks, [448, 460, 500, 700], rng)
        assert step(ctx, m, d, of, blocks, [new] * 4, 8, "bf16", rng, scale=scale) <= 1


def test_large_values_meet_small_ones(ctx):
    """A prefix of values 2^17 times the rest's, and the other way round: neither takes the other's bits."""
    rng = np.random.default_rng(27)
    say("sizes")
    for at in (0, 1):
        for heads, kv in ((2, 2), (4, 2), (4, 1)):
            of, blocks, n = [0] * 16, [20], 16
            m, d = alike(ctx, "bf16", kv, 128, of, blocks, [1280 + 33 * i for i in range(n)], rng)
            shared = m.table[0, :20]
            rest = np.setdiff1d(np.arange(m.pages), shared)
            m.scales[shared if at == 0 else rest, :, 1] *= np.float32(2.0 ** 17)
            d.b["scales"].upload(m.scales)
            assert step(ctx, m, d, of, blocks, [1] * n, heads, "bf16", rng) <= 1
        of, blocks = [0] * 3, [3]
        m, d = alike(ctx, "bf16", 1, 128, of, blocks, [250, 330, 200], rng)
        shared = m.table[0, :3]
        rest = np.setdiff1d(np.arange(m.pages), shared)
        m.scales[shared if at == 0 else rest, :, 1] *= np.float32(2.0 ** 17)
        d.b["scales"].upload(m.scales)
        assert step(ctx, m, d, of, blocks, [1] * 3, 4, "bf16", rng) <= 1
        assert step(ctx, m, d, of, blocks, [30] * 3, 4, "bf16", rng) <= 1


def test_two_runs_are_bit_identical(ctx):
    rng = np.random.default_rng(28)
    kv, hd, heads, n = 8, 128, 32, 16
    of, blocks = [0] * 12 + [1] * 4, [30, 17]
    m, d = alike(ctx, "fp16", kv, hd, of, blocks, [64 * blocks[g] + 9 * i for i, g in enumerate(of)], rng)
    say("twice")
    s = X.Seqs(ctx, [1] * n)
    p = X.Prefixes(ctx, s, of, blocks)
    dq = X.DevBuf.of(ctx, normal(rng, (n, heads, hd), "fp16")[0])
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    outs = []
    for fill in (0.0, np.nan):
        part = X.DevBuf.of(ctx, np.full(floats, fill, np.float32))
        o = X.DevBuf(ctx, (n, heads, hd), np.uint16)
        X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
        outs.append(o.get())
    assert np.array_equal(*outs)


def test_pages_past_4_gb(ctx):
    """A shared page whose codes lie past 2^32 bytes."""
    rng = np.random.default_rng(29)
    kv, hd, pages = 8, 128, 66000
    say("past 4 GB")
    m, d = alike(ctx, "fp16", kv, hd, [0, 0], [2], [130, 140], rng)
    big = {n: X.DevBuf(ctx, (pages, kv, 64, hd), np.int8) for n in ("k", "v")}
    sc = X.DevBuf(ctx, (pages, kv, 2), np.float32)
    move = {int(p): pages - 1 - i for i, p in enumerate(np.unique(m.table))}
    for a, b in move.items():
        for n in ("k", "v"):
            x = np.ascontiguousarray(getattr(m, n)[a])
            X.call("exn_upload", ctx.h, big[n].at(b * x.nbytes), X.ptr(x), x.nbytes)
        x = np.ascontiguousarray(m.scales[a])
        X.call("exn_upload", ctx.h, sc.at(b * x.nbytes), X.ptr(x), x.nbytes)
    far = np.vectorize(move.get)(m.table).astype(np.int32)
    d.b["table"].upload(far)
    h = X.Kv8(X.DT_F16, kv, hd, pages, 2, m.cols, big["k"].ptr, big["v"].ptr, sc.ptr,
              *(d.b[n].ptr for n in ("tk", "tv", "table", "lens")))
    s = X.Seqs(ctx, [1, 1])
    p = X.Prefixes(ctx, s, [0, 0], [2])
    qb, q = normal(rng, (2, 16, hd), "fp16")
    dq, o = X.DevBuf.of(ctx, qb), X.DevBuf(ctx, (2, 16, hd), np.uint16)
    floats = X.attend_shared_part(s, p, 16, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    X.attend_shared(ctx, h, s, p, 16, dq.h, 16 * hd, 0.09, o.h, X.DT_F16, 16 * hd, part.h, floats)
    got = pm.value(o.get(), "fp16")
    for b in (*big.values(), sc):
        b.free()
    want, tol = m.attend(q, [1, 1], 0.09, "fp16")
    assert off(got, want, tol) <= 1


def test_no_rows_and_no_prefixes(ctx):
    rng = np.random.default_rng(30)
    say("nothing")
    m, d = alike(ctx, "fp16", 2, 64, [0, 0], [1], [64, 70], rng)
    s = X.Seqs(ctx, [0, 0])
    p = X.Prefixes(ctx, s, [0, 0], [1])
    o = X.DevBuf.of(ctx, np.full((2, 256), 0x1234, np.uint16))
    assert X.attend_shared_part(s, p, 4, 2, 64, m.cols) == 0
    X.attend_shared(ctx, d.h, s, p, 4, o.h, 256, 1.0, o.h, X.DT_F16, 256)
    assert (o.get() == 0x1234).all()
    assert step(ctx, m, d, [-1, -1], [], [1, 3], 4, "bf16", rng) <= 1


def test_captured_steps_with_tables_that_change(ctx):
    """A captured step (rows turned by the cache's lengths, appended, attended, counted) replayed as the cache grows and
    as a sequence leaves its prefix: each replay against the plain form, with eager work between the replays."""
    import prompts_rope as pr
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    rng = np.random.default_rng(31)
    heads, kv, hd, n = 8, 2, 128, 12
    of, blocks, new = [0] * 8 + [1] * 4, [18, 17], [1] * 12
    say("captured")
    m, d = alike(ctx, "fp16", kv, hd, of, blocks, [64 * blocks[g] + (60 + 3 * i) % 90 for i, g in enumerate(of)], rng)
    s = X.Seqs(ctx, new)
    p = X.Prefixes(ctx, s, of, blocks)
    freqs = X.rope_freqs(hd, 5e6)
    rope = X.Rope(ctx, freqs)
    q0, k0, v0 = (X.DevBuf(ctx, (n, h, hd), np.uint16) for h in (heads, kv, kv))
    q1, k1 = (X.DevBuf(ctx, (n, h, hd), np.uint16) for h in (heads, kv))
    wq, wk = (X.DevBuf.of(ctx, (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)) for _ in range(2))
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    o = X.DevBuf(ctx, (n, heads, hd), np.uint16)

    def call():
        X.rope_rows(ctx, rope, s, hd, X.DT_F16, X.DT_F16, (heads, q0.h, heads * hd, wq.h, q1.h, heads * hd),
                    (kv, k0.h, kv * hd, wk.h, k1.h, kv * hd), 1e-6, lens=d.b["lens"].h)
        X.kv8_append(ctx, d.h, s, k1.h, kv * hd, v0.h, kv * hd)
        X.attend_shared(ctx, d.h, s, p, heads, q1.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
        X.kv8_advance(ctx, d.h, s)

    stream, g, ge = vp(), vp(), vp()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    try:
        X.call("exn_set_stream", ctx.h, stream)
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        call()
        assert hip.hipStreamEndCapture(stream, ctypes.byref(g)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(ge), g, None, None, 0) == 0
        for i in range(6):
            qb, kb, vb = (normal(rng, (n, h, hd), "fp16")[0] for h in (heads, kv, kv))
            for b, x in ((q0, qb), (k0, kb), (v0, vb)):
                b.upload(x)
            if i == 3:      # the second sequence leaves its prefix at the second block
                m.table[1, 1] = m.table[1, m.cols - 1]
                d.b["table"].upload(m.table)
            assert hip.hipGraphLaunch(ge, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            # the rows as the kernel left them (within what is derived for it), then the attention over them
            for x, w, y in ((qb, wq, q1), (kb, wk, k1)):
                want, tol = pr.rope_rows(pm.value(x, "fp16"), w.get(), 1e-6, m.lens[:, None], freqs, None, 0, 1.0, "fp16")
                assert off(pm.value(y.get(), "fp16"), want, tol) <= 1
            m.append(k1.get(), vb, new)
            want, tol = m.attend(pm.value(q1.get(), "fp16"), new, 0.09, "bf16")
            r = off(pm.value(o.get(), "bf16"), want, tol)
            say("replay", i, "worst", r)
            assert r <= 1
            m.advance(new)
            assert (d.b["lens"].get() == m.lens).all()
    finally:
        if ge.value:
            hip.hipGraphExecDestroy(ge)
        if g.value:
            hip.hipGraphDestroy(g)
        X.call("exn_set_stream", ctx.h, None)
        hip.hipStreamSynchronize(stream)
        hip.hipStreamDestroy(stream)


def test_two_streams_at_once(ctx):
    """One plan and its prefixes, one cache, in calls of two contexts that overlap: scratch and results of their own."""
    rng = np.random.default_rng(35)
    kv, hd, heads, n = 2, 128, 8, 24
    of, blocks = [0] * n, [40]
    m, d = alike(ctx, "fp16", kv, hd, of, blocks, [2560 + 17 * i for i in range(n)], rng)
    say("two streams")
    s = X.Seqs(ctx, [1] * n)
    p = X.Prefixes(ctx, s, of, blocks)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    with X.Context(0) as other:
        runs = []
        for c in (ctx, other):
            qb, q = normal(rng, (n, heads, hd), "fp16")
            runs.append((c, X.DevBuf.of(c, qb), X.DevBuf(c, (floats,), np.float32), X.DevBuf(c, (n, heads, hd), np.uint16), q))
        for _ in range(20):
            for c, dq, part, o, _q in runs:
                X.attend_shared(c, d.h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
        for c, dq, part, o, q in runs:
            want, tol = m.attend(q, [1] * n, 0.09, "bf16")
            assert off(pm.value(o.get(), "bf16"), want, tol) <= 1
        for b in runs[1][1:4]:
            b.free()


def test_the_same_page_many_times(ctx):
    """Tables that name one page again and again, in the prefix and after it."""
    rng = np.random.default_rng(36)
    say("same page")
    n, of, blocks = 9, [0] * 9, [20]
    m, d = alike(ctx, "bf16", 2, 64, of, blocks, [20 * 64 + 1 + 64 * (i % 3) for i in range(n)], rng)
    m.table[:, :20] = m.table[0, 0]
    m.table[4, :22] = m.table[4, 21]
    d.b["table"].upload(m.table)
    assert step(ctx, m, d, of, blocks, [1] * n, 4, "bf16", rng) <= 1


def test_plans_of_many_sequences(ctx):
    """Thousands of sequences over one prefix, and as many prefixes as sequences allow."""
    rng = np.random.default_rng(37)
    say("many sequences")
    n, kv, hd = 1500, 1, 64
    of = [0] * 700 + [1 + i % 80 for i in range(n - 700)]
    blocks = [17] + [18] * 80
    before = [64 * blocks[g] + i % 5 for i, g in enumerate(of)]
    m, d = alike(ctx, "fp16", kv, hd, of, blocks, before, rng, cols=20)
    assert step(ctx, m, d, of, blocks, [1] * n, 1, "fp16", rng) <= 1


# sequences of several tokens, of 17 to 64 rows a key/value head: new tokens, by the sequence's number
STEPS = {
    "even": lambda i, most: most,
    "ragged": lambda i, most: 1 + (5 * i) % most if i else most,
    "waiting": lambda i, most: [0, 1, most][i % 3],
}


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,hd,most", [(8, 2, 128, 16), (8, 2, 128, 5), (8, 1, 64, 8), (5, 1, 128, 12), (2, 2, 64, 64),
                                              (2, 2, 128, 17), (16, 1, 64, 8), (32, 1, 128, 3), (3, 3, 128, 30), (7, 1, 64, 3)])
@pytest.mark.parametrize("tokens", STEPS)
def test_steps_of_several_tokens(ctx, tokens, heads, kv, hd, most, dt, odt):
    rng = np.random.default_rng([37, heads, most])
    of = [-1 if i % 7 == 6 else i % 9 // 8 for i in range(28)]
    blocks = [33, 17]
    own = [(37 * i) % 130 if i % 5 else 900 - i for i in range(28)]
    new = [STEPS[tokens](i, most) for i in range(28)]
    say("steps", tokens, heads, kv, hd, most, dt, odt)
    m, d = alike(ctx, dt, kv, hd, of, blocks, [n + 64 * (blocks[g] if g >= 0 else 0) for n, g in zip(own, of)], rng)
    for _ in range(2):
        r = step(ctx, m, d, of, blocks, new, heads, odt, rng)
        say("worst", r)
        assert r <= 1


@pytest.mark.parametrize("heads,kv,hd,seqs,most,tokens", [(8, 2, 128, 3, 8, 14000), (4, 1, 64, 9, 9, 20000), (4, 2, 128, 30, 10, 5000)])
def test_steps_of_several_tokens_after_long_prefixes(ctx, heads, kv, hd, seqs, most, tokens):
    rng = np.random.default_rng([38, seqs])
    of, blocks = [0] * seqs, [tokens // 64]
    say("steps, long", heads, kv, hd, seqs, most, tokens)
    m, d = alike(ctx, "bf16", kv, hd, of, blocks, [blocks[0] * 64 + (37 * i) % 400 for i in range(seqs)], rng)
    assert step(ctx, m, d, of, blocks, [most - i % 3 for i in range(seqs)], heads, "bf16", rng) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,most", [(8, 2, 128, 17), (4, 1, 64, 40), (2, 2, 64, 80), (8, 1, 128, 10), (1, 1, 128, 160)])
def test_steps_of_many_tokens(ctx, heads, kv, hd, most, dt):
    """More than 64 rows a key/value head and sequence, in several tiles each."""
    rng = np.random.default_rng([43, heads, most])
    of, blocks, n = [0] * 13 + [-1], [80], 14
    say("many tokens", heads, kv, hd, most, dt)
    m, d = alike(ctx, dt, kv, hd, of, blocks, [80 * 64 * (g == 0) + (37 * i) % 150 for i, g in enumerate(of)], rng)
    m.table[5, 33] = m.table[5, -1]
    d.b["table"].upload(m.table)
    new = [most - (i % 3) * (most // 4) for i in range(n)]
    s = X.Seqs(ctx, new)
    assert X.attend_shared_part(s, X.Prefixes(ctx, s, of, blocks), heads, kv, hd, m.cols) != X.kv8_attend_part(s, heads, kv, hd, m.cols)
    assert step(ctx, m, d, of, blocks, new, heads, "bf16", rng) <= 1


def test_steps_whose_tables_are_not_alike(ctx):
    """As for single tokens: tables that part and meet again, pages that are none, odd lengths and hints."""
    rng = np.random.default_rng(39)
    say("steps not alike")
    for heads, kv, hd, n, most in ((8, 2, 128, 24, 5), (8, 1, 64, 20, 8), (2, 2, 64, 16, 40)):
        of, b = [0] * n, 30
        before = [b * 64 + (29 * i) % 150 for i in range(n)]
        before[3], before[5], before[7] = 100, 0, 64 * 17 + 63
        m, d = alike(ctx, "fp16", kv, hd, of, [b], before, rng, cols=36)
        other = lambda i, j: m.table[i, 35 - j % 3]
        m.table[1, 0] = other(1, 0)
        m.table[2, 29] = other(2, 1)
        m.table[4, [7, 8, 20]] = [other(4, 0), other(4, 1), -1]
        m.table[6, 2:30:3] = [other(6, j) for j in range(10)]
        m.table[8, 10:] = m.table[9, 10:][::-1]
        m.table[[0, 9, 10], 16] = 1 << 30
        m.table[11, 12] = -7
        d.b["table"].upload(m.table)
        new = [most - i % 4 for i in range(n)]
        for blocks in ([30], [36], [1 << 20]):
            r = step(ctx, m, d, of, blocks, new, heads, "bf16", rng)
            say(blocks, "worst", r)
            assert r <= 1
        m.lens[0] = 0
        d.b["lens"].upload(m.lens)
        assert step(ctx, m, d, of, [30], new, heads, "fp16", rng) <= 1


@pytest.mark.parametrize("cap", [0.5, 0.1, 0.02, 0], ids=str)
def test_steps_and_scratch(ctx, cap):
    rng = np.random.default_rng(40)
    of, blocks, new = [0] * 18, [24], [5, 3, 8] * 6
    say("steps, scratch", cap)
    m, d = alike(ctx, "fp16", 2, 128, of, blocks, [24 * 64 + 23 * i for i in range(18)], rng)
    assert step(ctx, m, d, of, blocks, new, 8, "fp16", rng, lambda n: int(n * cap) // 4 * 4) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_steps_with_values_that_are_not_finite(ctx, bad, dt):
    """A step's last token is not finite: those before it do not see it, also where its sequence's table parts from its
    prefix and meets it again; a spoilt block of the prefix is not seen by the sequences that have parted there."""
    rng = np.random.default_rng(41)
    say("steps, not finite", bad, dt)
    kv, hd, heads, n, most = 2, 128, 8, 20, 6
    of, blocks, new = [0] * n, [24], [most] * n
    m, d = alike(ctx, dt, kv, hd, of, blocks, [24 * 64 + 3 + 2 * i for i in range(n)], rng)
    m.table[2, 5] = m.table[2, -1]
    m.table[3, 11] = m.table[3, -1]
    m.scales[m.table[0, 11], 1, 1] = bad
    d.b["table"].upload(m.table)
    d.b["scales"].upload(m.scales)
    s = X.Seqs(ctx, new)
    p = X.Prefixes(ctx, s, of, blocks)
    kb, _ = normal(rng, (n * most, kv, hd), dt)
    vb, _ = normal(rng, (n * most, kv, hd), dt)
    qb, q = normal(rng, (n * most, heads, hd), dt)
    spoilt = vb.reshape(n, most, kv, hd).copy()
    spoilt[:, -1, 0, :] = pm.bits(np.float32(bad), dt)[()]
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, spoilt))
    o = X.DevBuf(ctx, (n, most, heads, hd), np.uint16)
    X.kv8_append(ctx, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    assert floats != X.kv8_attend_part(s, heads, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
    got = pm.value(o.get(), "bf16")
    m.append(kb, vb, new)
    m.scales[~np.isfinite(m.scales)] = 0.03
    want, tol = (x.reshape(got.shape) for x in m.attend(q, new, 0.09, "bf16"))
    half = heads // 2
    assert not np.isfinite(got[:, -1, :half]).any()
    sees = [i for i in range(n) if i != 3]
    assert not np.isfinite(got[sees][:, :, half:]).any()
    assert (abs(got - want)[:, :-1, :half] <= tol[:, :-1, :half]).all()
    assert (abs(got - want)[3, :, half:] <= tol[3, :, half:]).all()


def test_two_runs_of_steps_are_bit_identical(ctx):
    rng = np.random.default_rng(42)
    kv, hd, heads, n = 8, 128, 32, 16
    of, blocks = [0] * 12 + [1] * 4, [40, 17]
    m, d = alike(ctx, "fp16", kv, hd, of, blocks, [64 * blocks[g] + 9 * i for i, g in enumerate(of)], rng)
    say("steps twice")
    new = [7, 12, 1, 5] * 4
    s = X.Seqs(ctx, new)
    p = X.Prefixes(ctx, s, of, blocks)
    dq = X.DevBuf.of(ctx, normal(rng, (sum(new), heads, hd), "fp16")[0])
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    outs = []
    for fill in (0.0, np.nan):
        part = X.DevBuf.of(ctx, np.full(floats, fill, np.float32))
        o = X.DevBuf(ctx, (sum(new), heads, hd), np.uint16)
        X.attend_shared(ctx, d.h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_BF16, heads * hd, part.h, floats)
        outs.append(o.get())
    assert np.array_equal(*outs)
