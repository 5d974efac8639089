"""The prompt side's attention on the GPU: packed causal attention, the cache in 8 bits and the
attention over it, against plain forms in 64 bits (prompts_model.py, which derives the tolerances).
Needs an MI355X."""
import ctypes
import sys

import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm

pytestmark = pytest.mark.gpu
DT = {"fp16": X.DT_F16, "bf16": X.DT_BF16}


def say(*a):
    print("[gpu]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    c = X.Context(0)
    yield c
    c.close()


def normal(rng, shape, t, spread=1.0):
    """Normal values of the type, as patterns and as 64-bit values."""
    b = pm.bits(pm.rounded((spread * rng.standard_normal(shape)).astype(np.float32), t), t)
    return b, pm.value(b, t)


def strided(b, pad):
    """Rows with PAD unused values after each (NaN patterns: nothing may depend on them)."""
    n = b.shape[0]
    out = np.full((n, b[0].size + pad), 0x7FFF, np.uint16)
    out[:, :b[0].size] = b.reshape(n, -1)
    return out


def off(got, want, tol):
    """How far over the tolerance the worst value is (at most 1: within)."""
    assert np.isfinite(got).all()
    return float((abs(got - want) / tol).max(initial=0))


# --- packed prompts --------------------------------------------------------------------------

LENS = [[1], [1, 1, 1], [0, 5, 0], [24], [63, 64, 65], [127, 128, 129, 1, 2], [257, 21, 0, 100], [300, 3, 33]]


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "bf16"), ("bf16", "fp16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (8, 1, 64), (3, 3, 128), (6, 2, 64), (5, 1, 128), (32, 2, 64),
                                         (11, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_packed(ctx, lens, heads, kv, hd, dt, odt):
    rng = np.random.default_rng([sum(lens), heads, hd])
    rows = sum(lens)
    qb, q = normal(rng, (rows, heads, hd), dt)
    kb, k = normal(rng, (rows, kv, hd), dt, 1.5)
    vb, v = normal(rng, (rows, kv, hd), dt)
    say("packed", lens, heads, kv, hd, dt, odt)
    s = X.Seqs(ctx, lens)
    dq, dk, dv = (X.DevBuf.of(ctx, strided(b, p)) for b, p in ((qb, 8), (kb, 0), (vb, 16)))
    o = X.DevBuf.of(ctx, np.full((rows + 1, heads * hd + 8), 0x1234, np.uint16))
    scale = hd ** -0.5
    X.attend_packed(ctx, s, DT[dt], heads, kv, hd, dq.h, heads * hd + 8, dk.h, kv * hd, dv.h, kv * hd + 16, scale, o.h,
                    DT[odt], heads * hd + 8)
    got = o.get()
    assert (got[rows:] == 0x1234).all() and (got[:, heads * hd:] == 0x1234).all()
    want, tol = pm.packed(q, k, v, lens, scale, dt, odt)
    r = off(pm.value(got[:rows, :heads * hd], odt).reshape(want.shape), want, tol)
    say("worst", r)
    assert r <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("spread", [30.0, 1e-3])
def test_packed_sharp_and_flat(ctx, dt, spread):
    """Scores of hundreds (one key takes all) and scores of nothing."""
    rng = np.random.default_rng(5)
    lens, heads, kv, hd = [200, 70], 4, 1, 128
    qb, q = normal(rng, (270, heads, hd), dt, spread)
    kb, k = normal(rng, (270, kv, hd), dt)
    vb, v = normal(rng, (270, kv, hd), dt)
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (270, heads, hd), np.uint16)
    say("packed spread", spread, dt)
    X.attend_packed(ctx, X.Seqs(ctx, lens), DT[dt], heads, kv, hd, dq.h, heads * hd, dk.h, kv * hd, dv.h, kv * hd, 0.125,
                    o.h, DT[dt], heads * hd)
    want, tol = pm.packed(q, k, v, lens, 0.125, dt, dt)
    assert off(pm.value(o.get(), dt), want, tol) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_packed_hidden_values_weigh_nothing(ctx, dt, bad):
    """Keys and values that a row does not see (later in its sequence, or of another sequence) may
    be anything; a row that sees one is not finite itself there."""
    rng = np.random.default_rng(6)
    lens, heads, kv, hd = [100, 70, 200], 4, 2, 64
    rows = sum(lens)
    qb, q = normal(rng, (rows, heads, hd), dt)
    kb, k = normal(rng, (rows, kv, hd), dt)
    vb, v = normal(rng, (rows, kv, hd), dt)
    say("packed hidden", dt, bad)
    want, tol = pm.packed(q, k, v, lens, 0.1, dt, dt)
    clean = [150, 165]                       # the middle sequence, rows 50 and 65 of it
    pat = pm.bits(np.float32(bad), dt)[0]
    vb2, kb2 = vb.copy(), kb.copy()
    vb2[clean[0], 0, 5] = pat
    kb2[clean[1]] = pat
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb2, vb2))
    o = X.DevBuf(ctx, (rows, heads, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, lens), DT[dt], heads, kv, hd, dq.h, heads * hd, dk.h, kv * hd, dv.h, kv * hd, 0.1,
                    o.h, DT[dt], heads * hd)
    got = pm.value(o.get(), dt)
    same = np.ones(got.shape, bool)
    same[clean[0]:170, :heads // kv, 5] = False
    same[clean[1]:170] = False
    assert (abs(got - want)[same] <= tol[same]).all()
    seen = got[clean[0]:clean[1], :heads // kv, 5]
    assert np.isnan(seen).all() if np.isnan(bad) else (seen == bad).all()
    if not np.isinf(bad):
        assert np.isnan(got[clean[1]:170]).all()


def test_packed_parts_of_one_row(ctx):
    """q, k and v as parts of one row, as a fused product leaves them."""
    rng = np.random.default_rng(7)
    lens, heads, kv, hd = [129, 40], 32, 8, 128
    b, x = normal(rng, (169, heads + 2 * kv, hd), "fp16")
    d = X.DevBuf.of(ctx, b)
    o = X.DevBuf(ctx, (169, heads, hd), np.uint16)
    ld = (heads + 2 * kv) * hd
    say("packed fused rows")
    X.attend_packed(ctx, X.Seqs(ctx, lens), X.DT_F16, heads, kv, hd, d.h, ld, d.at(heads * hd * 2), ld,
                    d.at((heads + kv) * hd * 2), ld, hd ** -0.5, o.h, X.DT_BF16, heads * hd)
    want, tol = pm.packed(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], lens, hd ** -0.5, "fp16", "bf16")
    assert off(pm.value(o.get(), "bf16"), want, tol) <= 1


def test_packed_rows_far_apart(ctx):
    """Strides with which a sequence's rows are over 2^32 bytes apart."""
    rng = np.random.default_rng(8)
    n, hd, ld = 150, 64, 1 << 24
    say("packed far rows")
    buf = X.DevBuf(ctx, (n * ld,), np.uint16)     # 5 GB: k at 0, v at 64 of each row
    kb, k = normal(rng, (n, 1, hd), "bf16")
    vb, v = normal(rng, (n, 1, hd), "bf16")
    qb, q = normal(rng, (n, 2, hd), "bf16")
    for i in range(n):
        row = np.concatenate([kb[i, 0], vb[i, 0]])
        X.call("exn_upload", ctx.h, buf.at(2 * i * ld), X.ptr(row), row.nbytes)
    dq, o = X.DevBuf.of(ctx, qb), X.DevBuf(ctx, (n, 2, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, [n]), X.DT_BF16, 2, 1, hd, dq.h, 2 * hd, buf.h, ld, buf.at(2 * hd), ld, 0.125, o.h,
                    X.DT_BF16, 2 * hd)
    want, tol = pm.packed(q, k, v, [n], 0.125, "bf16", "bf16")
    got = pm.value(o.get(), "bf16")
    buf.free()
    assert off(got, want, tol) <= 1


# --- the cache ----------------------------------------------------------------------------------


class Dev:
    """A pm.Cache's arrays on the device."""

    def __init__(self, ctx, m):
        self.m, self.ctx = m, ctx
        self.b = {n: X.DevBuf.of(ctx, getattr(m, n)) for n in ("k", "v", "scales", "tk", "tv", "table", "lens")}
        self.h = X.Kv8(DT[m.dt], m.kv, m.hd, m.pages, len(m.lens), m.cols,
                       *(self.b[n].ptr for n in ("k", "v", "scales", "tk", "tv", "table", "lens")))

    def same(self, new=None):
        """The device's cache is the model's, bit for bit (NaN scales as NaN; tails as far as their
        blocks have tokens, NEW of them after the step's)."""
        for n in ("k", "v", "table", "lens"):
            assert (self.b[n].get() == getattr(self.m, n)).all(), n
        for n in ("tk", "tv"):
            got = self.b[n].get()
            for i in range(len(self.m.lens)):
                live = self.m.total(i, new[i] if new else 0) % 64
                assert (got[i, :, :live] == getattr(self.m, n)[i, :, :live]).all(), n
        s = self.b["scales"].get()
        assert ((s == self.m.scales) | (np.isnan(s) & np.isnan(self.m.scales))).all()


def cache_of(ctx, dt, seqs, kv, hd, cols, rng, pages=None, table=None):
    pages = pages or seqs * cols + 2
    if table is None:
        table = rng.permutation(pages)[:seqs * cols]
    m = pm.Cache(dt, seqs, kv, hd, pages, cols, table, rng)
    return m, Dev(ctx, m)


def step(ctx, m, d, new, heads, odt, rng, part=True, scale=None, spread=1.0):
    """Append, read, attend and advance by NEW tokens: the worst distance over its tolerance."""
    rows, kv, hd = sum(new), m.kv, m.hd
    kb, _ = normal(rng, (rows, kv, hd), m.dt, spread)
    vb, _ = normal(rng, (rows, kv, hd), m.dt)
    qb, q = normal(rng, (rows, heads, hd), m.dt)
    scale = hd ** -0.5 if scale is None else scale
    s = X.Seqs(ctx, new)
    dk, dv, dq = X.DevBuf.of(ctx, strided(kb, 8)), X.DevBuf.of(ctx, vb), X.DevBuf.of(ctx, strided(qb, 24))
    o = X.DevBuf.of(ctx, np.full((rows + 1, heads * hd + 8), 0x1234, np.uint16))
    X.kv8_append(ctx, d.h, s, dk.h, kv * hd + 8, dv.h, kv * hd)
    floats = X.kv8_attend_part(s, heads, kv, hd, m.cols) if part else 0
    scratch = X.DevBuf.of(ctx, np.full(floats + 4, np.nan, np.float32))
    X.kv8_attend(ctx, d.h, s, heads, dq.h, heads * hd + 24, scale, o.h, DT[odt], heads * hd + 8,
                 scratch.h if floats else None, floats)
    rk, rv = (X.DevBuf.of(ctx, np.full((rows + 1, kv * hd), 0x1234, np.uint16)) for _ in range(2))
    X.kv8_read(ctx, d.h, s, rk.h, kv * hd, rv.h, kv * hd)
    m.append(kb, vb, new)
    d.same(new)
    got = o.get()
    assert (got[rows:] == 0x1234).all() and (got[:, heads * hd:] == 0x1234).all()
    want, tol = m.attend(q, new, scale, odt)
    r = off(pm.value(got[:rows, :heads * hd], odt).reshape(want.shape), want, tol)
    for b, w in zip((rk, rv), m.read(new)):
        x = b.get()
        assert (x[rows:] == 0x1234).all()
        assert np.array_equal(pm.value(x[:rows], m.dt).reshape(w.shape), w)
    X.kv8_advance(ctx, d.h, s)
    m.advance(new)
    d.same()
    return r


STEPS = [
    [[1], [1], [63], [64], [1], [130]],
    [[200, 0, 65], [1, 1, 1], [0, 1, 0], [56, 62, 63], [1, 1, 1]],
    [[64, 128, 127, 63], [1, 1, 1, 1], [70, 5, 20, 100], [16, 16, 16, 16]],
]


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (8, 1, 64), (3, 3, 128), (12, 4, 64), (5, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("steps", STEPS, ids=["one", "three", "four"])
def test_cache_steps(ctx, steps, heads, kv, hd, dt, odt):
    """Whole prompts, single tokens and chunks, appended and attended in turn."""
    rng = np.random.default_rng([len(steps[0]), heads, hd])
    say("cache steps", steps[0], heads, kv, hd, dt, odt)
    m, d = cache_of(ctx, dt, len(steps[0]), kv, hd, 6, rng)
    for new in steps:
        r = step(ctx, m, d, new, heads, odt, rng)
        say(new, "worst", r)
        assert r <= 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("part", [True, False])
def test_cache_long(ctx, hd, part):
    """Thousands of keys to a token, with and without scratch to split them."""
    rng = np.random.default_rng(11)
    m, d = cache_of(ctx, "fp16", 2, 2, hd, 80, rng)
    say("cache long", hd, part)
    assert step(ctx, m, d, [4700, 3001], 2, "fp16", rng, part) <= 1
    assert step(ctx, m, d, [1, 1], 8, "fp16", rng, part) <= 1
    assert step(ctx, m, d, [2, 31], 8, "fp16", rng, part) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_one_by_one_is_all_at_once(ctx, dt):
    rng = np.random.default_rng(12)
    rows, kv, hd = 150, 2, 64
    kb, _ = normal(rng, (rows, kv, hd), dt)
    vb, _ = normal(rng, (rows, kv, hd), dt)
    dk, dv = X.DevBuf.of(ctx, kb), X.DevBuf.of(ctx, vb)
    say("one by one", dt)
    m, d = cache_of(ctx, dt, 1, kv, hd, 3, rng)
    m.append(kb, vb, [rows])
    m.advance([rows])
    one = X.Seqs(ctx, [1])
    for i in range(rows):
        X.kv8_append(ctx, d.h, one, dk.at(2 * i * kv * hd), kv * hd, dv.at(2 * i * kv * hd), kv * hd)
        X.kv8_advance(ctx, d.h, one)
    d.same()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("power", [-20, -8, 0, 9])
def test_codes_on_and_next_to_ties(ctx, dt, power):
    """Blocks of values exactly between two codes, and next to there; the smallest and largest ones."""
    rng = np.random.default_rng([20, power + 40])
    kv, hd, rows = 4, 128, 128
    x = (2.0 ** power * rng.standard_normal((rows, kv, hd))).astype(np.float32)
    x[0] = x[64] = 0
    x[0, :, 0] = x[64, :, 0] = 2.0 ** power * rng.choice([4.0, 5.0625, 6.5, 7.984375], kv)
    x = pm.rounded(np.clip(x, -4 * 2.0 ** power, 4 * 2.0 ** power), dt)
    for b in range(2):
        for h in range(kv):
            d = np.float64(pm.scale_of(x[64 * b:64 * b + 64, h]))
            tie = (rng.integers(-64, 64, (63, hd)) + 0.5) * d
            x[64 * b + 1:64 * b + 64, h] = pm.rounded(tie.astype(np.float32), dt)
    if power == -20:      # the second block: values of the type's smallest
        x[64:] = pm.rounded((2.0 ** (-23 if dt == "fp16" else -132) * rng.standard_normal((64, kv, hd))).astype(np.float32), dt)
    if power == 9:        # and of its largest
        x[64:] = pm.rounded((x[64:] / 4096 * (65000 if dt == "fp16" else 3e38)).astype(np.float32), dt)
    say("ties", dt, power)
    b = pm.bits(x, dt)
    m, d = cache_of(ctx, dt, 1, kv, hd, 2, rng)
    db = X.DevBuf.of(ctx, b)
    X.kv8_append(ctx, d.h, X.Seqs(ctx, [rows]), db.h, kv * hd, db.h, kv * hd)
    m.append(b, b, [rows])
    d.same([rows])


def test_cache_edges(ctx):
    """Rows past the table's end, pages that are none, lengths out of range: hidden, never written."""
    rng = np.random.default_rng(13)
    say("cache edges")
    table = np.array([[0, -1, 2], [3, 999, 5], [1 << 30, 6, -(1 << 31)]])
    m, d = cache_of(ctx, "bf16", 3, 2, 64, 3, rng, pages=7, table=table)
    assert step(ctx, m, d, [70, 130, 64], 4, "bf16", rng) <= 1
    assert step(ctx, m, d, [150, 1, 3], 4, "bf16", rng) <= 1      # the first past its end
    assert step(ctx, m, d, [5, 100, 60], 4, "bf16", rng) <= 1     # and again
    m.lens[:] = [-5, 1 << 30, 100]
    d.b["lens"].upload(m.lens)
    assert step(ctx, m, d, [1, 2, 1], 4, "bf16", rng) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_cache_blocks_that_are_not_finite(ctx, dt, bad):
    """A value that is not finite: its row from the tail, its whole block once that is full; rows that
    do not see it are as they were."""
    rng = np.random.default_rng(14)
    kv, hd, heads = 1, 64, 2
    m, d = cache_of(ctx, dt, 2, kv, hd, 3, rng)
    say("cache not finite", dt, bad)
    for new, spoil in (([100, 100], None), ([10, 10], 3), ([30, 30], None)):
        rows = sum(new)
        kb, _ = normal(rng, (rows, kv, hd), dt)
        vb, _ = normal(rng, (rows, kv, hd), dt)
        qb, q = normal(rng, (rows, heads, hd), dt)
        if spoil is not None:
            vb[spoil, 0, 7] = pm.bits(np.float32(bad), dt)[0]       # sequence 0, place 103
        s = X.Seqs(ctx, new)
        dk, dv, dq = (X.DevBuf.of(ctx, b) for b in (kb, vb, qb))
        o = X.DevBuf(ctx, (rows, heads, hd), np.uint16)
        X.kv8_append(ctx, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
        X.kv8_attend(ctx, d.h, s, heads, dq.h, heads * hd, 0.125, o.h, DT[dt], heads * hd)
        with np.errstate(invalid="ignore"):
            m.append(kb, vb, new)
        d.same(new)
        got = pm.value(o.get(), dt)
        clean = pm.Cache(dt, 2, kv, hd, m.pages, 3, m.table, rng)
        for n in ("k", "v", "scales", "tk", "tv", "lens"):
            setattr(clean, n, getattr(m, n).copy())
        clean.scales[np.isnan(clean.scales)] = 0
        clean.tv[~np.isfinite(pm.value(clean.tv, dt))] = 0
        want, tol = clean.attend(q, new, 0.125, dt)
        same = np.ones(got.shape, bool)
        if new == [10, 10]:
            same[3:10, :, 7] = False
            assert not np.isfinite(got[3:10, :, 7]).any()
        if new == [30, 30]:
            same[:30] = False                 # the block is full, and as a whole not finite
            assert np.isnan(got[:30]).all()
        assert (abs(got - want)[same] <= tol[same]).all()
        X.kv8_advance(ctx, d.h, s)
        m.advance(new)


def test_cache_past_4_gb(ctx):
    """Pages whose codes lie past 2^32 bytes."""
    rng = np.random.default_rng(15)
    kv, hd, pages = 8, 128, 66000                      # 4.3 GB of keys, as much of values
    say("cache past 4 GB")
    m = pm.Cache("fp16", 1, kv, hd, 4, 4, [[0, 1, 2, 3]], rng)
    d = Dev(ctx, m)
    big = {n: X.DevBuf(ctx, (pages, kv, 64, hd), np.int8) for n in ("k", "v")}
    sc = X.DevBuf(ctx, (pages, kv, 2), np.float32)
    far = np.array([[pages - 1, 0, pages - 2, 65536]], np.int32)
    d.b["table"].upload(far)
    h = X.Kv8(X.DT_F16, kv, hd, pages, 1, 4, big["k"].ptr, big["v"].ptr, sc.ptr,
              *(d.b[n].ptr for n in ("tk", "tv", "table", "lens")))
    for new in ([200], [1], [40]):
        rows = sum(new)
        kb, _ = normal(rng, (rows, kv, hd), "fp16")
        vb, _ = normal(rng, (rows, kv, hd), "fp16")
        qb, q = normal(rng, (rows, 8, hd), "fp16")
        s = X.Seqs(ctx, new)
        dk, dv, dq = (X.DevBuf.of(ctx, b) for b in (kb, vb, qb))
        o = X.DevBuf(ctx, (rows, 8, hd), np.uint16)
        X.kv8_append(ctx, h, s, dk.h, kv * hd, dv.h, kv * hd)
        X.kv8_attend(ctx, h, s, 8, dq.h, 8 * hd, 0.1, o.h, X.DT_F16, 8 * hd)
        X.kv8_advance(ctx, h, s)
        m.append(kb, vb, new)
        want, tol = m.attend(q, new, 0.1, "fp16")
        m.advance(new)
        assert off(pm.value(o.get(), "fp16"), want, tol) <= 1
    for b in (*big.values(), sc):
        b.free()


def test_shared_prefix(ctx):
    """Two sequences on one prefix's pages, each with its own tail, are two sequences."""
    rng = np.random.default_rng(16)
    kv, hd = 2, 128
    say("shared prefix")
    m, d = cache_of(ctx, "fp16", 2, kv, hd, 4, rng, pages=8, table=[[0, 1, 2, 3], [4, 5, 6, 7]])
    assert step(ctx, m, d, [150, 0], 8, "bf16", rng) <= 1
    m.table[1] = [0, 1, 4, 5]
    m.lens[1] = m.lens[0]
    m.tk[1], m.tv[1] = m.tk[0], m.tv[0]
    for n in ("table", "lens", "tk", "tv"):
        d.b[n].upload(getattr(m, n))
    assert step(ctx, m, d, [30, 80], 8, "bf16", rng) <= 1
    assert step(ctx, m, d, [1, 1], 8, "bf16", rng) <= 1


def test_two_runs_are_bit_identical(ctx):
    rng = np.random.default_rng(17)
    kv, hd, heads = 8, 128, 32
    m, d = cache_of(ctx, "fp16", 3, kv, hd, 40, rng)
    say("two runs")
    step(ctx, m, d, [2000, 700, 64], heads, "bf16", rng)
    s = X.Seqs(ctx, [1, 1, 1])
    qb, _ = normal(rng, (3, heads, hd), "fp16")
    dq = X.DevBuf.of(ctx, qb)
    floats = X.kv8_attend_part(s, heads, kv, hd, 40)
    part = X.DevBuf.of(ctx, np.full(floats + 4, np.nan, np.float32))
    outs = []
    for _ in range(3):
        o = X.DevBuf(ctx, (3, heads, hd), np.uint16)
        X.kv8_attend(ctx, d.h, s, heads, dq.h, heads * hd, 0.1, o.h, X.DT_BF16, heads * hd, part.h, floats)
        outs.append(o.get())
    assert (outs[0] == outs[1]).all() and (outs[0] == outs[2]).all()


def filled(ctx, dt, lens, kv, hd, cols, rng, pages=None, table=None):
    """A cache as many steps would leave it: random codes, scales and tails."""
    m, d = cache_of(ctx, dt, len(lens), kv, hd, cols, rng, pages, table)
    m.scales[:] = (rng.uniform(0.5, 2, m.scales.shape) / 64).astype(np.float32)
    for n in ("tk", "tv"):
        getattr(m, n)[:] = normal(rng, getattr(m, n).shape, dt)[0]
    m.lens[:] = lens
    for n in ("scales", "tk", "tv", "lens"):
        d.b[n].upload(getattr(m, n))
    return m, d


def attended(ctx, d, q, new, heads, odt, scale, floats=None):
    """kv8_attend alone, over the cache as it is: its rows' values."""
    m = d.m
    s = X.Seqs(ctx, new)
    dq = X.DevBuf.of(ctx, q)
    o = X.DevBuf.of(ctx, np.full((sum(new) + 1, heads, m.hd), 0x1234, np.uint16))
    n = X.kv8_attend_part(s, heads, m.kv, m.hd, m.cols)
    n = n if floats is None else floats(n)
    part = X.DevBuf.of(ctx, np.full(n + 4, np.nan, np.float32))
    X.kv8_attend(ctx, d.h, s, heads, dq.h, heads * m.hd, scale, o.h, DT[odt], heads * m.hd, part.h if n else None, n)
    got = o.get()
    assert (got[-1] == 0x1234).all()
    assert np.isnan(part.get()[n:]).all()
    return pm.value(got[:-1], odt)


@pytest.mark.parametrize("dt,odt", [("fp16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,top,cols", [(3, 1000, 40), (70, 300, 40), (70, 2500, 40), (5, 2500, 40), (200, 900, 15),
                                        (150, 1100, 18)])
def test_cache_many_sequences(ctx, n, top, cols, dt, odt):
    """Single tokens over lengths from none to TOP, in tables that are larger: shares that begin and
    end within sequences, a workgroup a sequence, more sequences than lanes or workgroups."""
    rng = np.random.default_rng([n, top])
    say("many sequences", n, top, dt)
    lens = rng.integers(0, top, n)
    lens[:3] = [0, top - 1, 63]
    pages = 300                                     # sequences share pages
    kv, hd, heads = 8, 64, 8
    m, d = filled(ctx, dt, lens, kv, hd, cols, rng, pages, rng.integers(0, pages, (n, cols)))
    qb, q = normal(rng, (n, heads, hd), dt)
    want, tol = m.attend(q, [1] * n, 0.125, odt)
    assert off(attended(ctx, d, qb, [1] * n, heads, odt, 0.125), want, tol) <= 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cols", [30, 45])
@pytest.mark.parametrize("new", [[8, 5, 1], [4, 2], [1, 1, 1], [20, 33]], ids=str)
def test_cache_any_scratch(ctx, new, cols, hd):
    """All the scratch asked for, less of it, too little for any split, none; one to 132 rows a
    sequence and head, over tables on both sides of the few-row kernel's bound."""
    rng = np.random.default_rng([sum(new), cols, hd])
    say("any scratch", new, cols, hd)
    lens = rng.integers(cols * 40, cols * 60, len(new))
    kv, heads = 2, 8
    m, d = filled(ctx, "bf16", lens, kv, hd, cols, rng)
    qb, q = normal(rng, (sum(new), heads, hd), "bf16")
    want, tol = m.attend(q, new, 0.125, "fp16")
    for floats in (lambda n: n, lambda n: n // 2, lambda n: n // 7, lambda n: min(n, 100), lambda n: 0):
        assert off(attended(ctx, d, qb, new, heads, "fp16", 0.125, floats), want, tol) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 8, 40])
def test_cache_values_of_very_different_sizes(ctx, new, dt):
    """A block whose values are 2^17 times the others' and whose keys weigh nothing (scores of
    -100, over 100 under each row's largest: e^-100 2^17 is 2^-127 of a value) is as if it were not there."""
    rng = np.random.default_rng(new)
    say("very different sizes", new, dt)
    lens, kv, hd, heads, cols = [1500, 700], 2, 64, 8, 40
    m, d = filled(ctx, dt, lens, kv, hd, cols, rng)
    qb, q = normal(rng, (2 * new, heads, hd), dt)
    qb[:, :, 0], q[:, :, 0] = pm.bits(np.float32(16), dt), 16.0
    for s in range(2):
        for p in m.table[s]:
            m.k[p, :, :, 0] = 0
        p = m.table[s, 5]
        m.k[p] = 0
        m.k[p, :, :, 0] = -100                       # q of 16 x -100 x 1 / 16
        m.scales[p] = [1 / 16, m.scales[p, 0, 1] * 2.0 ** 17]
    m.tk[:, :, :, 0] = 0
    for n in ("k", "scales", "tk"):
        d.b[n].upload(getattr(m, n))
    got = attended(ctx, d, qb, [new, new], heads, dt, 1.0)
    m.table = m.table.copy()
    m.table[:, 5] = -1
    want, tol = m.attend(q, [new, new], 1.0, dt)
    assert off(got, want, tol) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("cols", [12, 40])
@pytest.mark.parametrize("new", [1, 8, 40])
def test_cache_not_finite_in_each_kernel(ctx, new, cols, dt):
    """A block that is not finite makes its sequence's rows NaN and nobody else's; a value of the tail
    its dim only; a page that is none hides a scale of NaN."""
    rng = np.random.default_rng([new, cols])
    say("not finite", new, cols, dt)
    lens, kv, hd, heads = [cols * 32, cols * 50, cols * 40 // 64 * 64 + 5], 1, 128, 4
    m, d = filled(ctx, dt, lens, kv, hd, cols, rng)
    qb, q = normal(rng, (3 * new, heads, hd), dt)
    want, tol = m.attend(q, [new] * 3, 0.1, dt)
    nan = m.table[0, 2]
    m.scales[nan, 0, rng.integers(2)] = np.nan
    m.tv[2, 0, 3, 9] = pm.bits(np.float32(np.inf), dt)[0]
    for n in ("scales", "tv"):
        d.b[n].upload(getattr(m, n))
    got = attended(ctx, d, qb, [new] * 3, heads, dt, 0.1)
    assert np.isnan(got[:new]).all()
    assert (got[2 * new:, :, 9] == np.inf).all()
    same = np.ones(got.shape, bool)
    same[:new] = same[2 * new:, :, 9] = False
    assert (abs(got - want)[same] <= tol[same]).all()
    m.table[0, 2] = -1
    d.b["table"].upload(m.table)
    m.tv[2, 0, 3, 9] = 0
    d.b["tv"].upload(m.tv)
    want, tol = m.attend(q, [new] * 3, 0.1, dt)
    assert off(attended(ctx, d, qb, [new] * 3, heads, dt, 0.1), want, tol) <= 1


@pytest.mark.parametrize("heads,kv", [(1024, 1), (1024, 1024), (96, 6), (17, 1), (1, 1), (1000, 8)])
def test_any_number_of_heads(ctx, heads, kv):
    """As many heads as are taken, groups of 1 to 1024 that do not divide a workgroup's rows: packed
    prompts, and a cache of short and long tables."""
    rng = np.random.default_rng([heads, kv])
    hd, lens = 64, [3, 0, 70]
    say("heads", heads, kv)
    rows = sum(lens)
    qb, q = normal(rng, (rows, heads, hd), "bf16")
    kb, k = normal(rng, (rows, kv, hd), "bf16")
    vb, v = normal(rng, (rows, kv, hd), "bf16")
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (rows, heads, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, lens), X.DT_BF16, heads, kv, hd, dq.h, heads * hd, dk.h, kv * hd, dv.h, kv * hd, 0.125,
                    o.h, X.DT_BF16, heads * hd)
    want, tol = pm.packed(q, k, v, lens, 0.125, "bf16", "bf16")
    assert off(pm.value(o.get(), "bf16"), want, tol) <= 1
    for cols in (3, 33):
        m, d = cache_of(ctx, "bf16", 3, kv, hd, cols, rng)
        for new in ([100, 70, 1], [1, 1, 1], [2, 0, 1], [9, 3, 0]):
            assert step(ctx, m, d, new, heads, "bf16", rng) <= 1


# --- a run of them under a graph, on another stream ---------------------------------------------


def test_captured_steps(ctx):
    """A serving step (append, attend, advance) captured once and replayed token by token, the
    program's own eager work between; the plan and the scratch made before."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng(18)
    kv, hd, heads, n = 2, 128, 8, 4
    say("captured steps")
    c2 = X.Context(0)
    st = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(st), 1) == 0
    X.call("exn_set_stream", c2.h, st)
    m, d = cache_of(c2, "bf16", n, kv, hd, 4, rng)
    step(c2, m, d, [61, 130, 0, 190], heads, "bf16", rng)
    new = [1] * n
    s = X.Seqs(c2, new)
    floats = X.kv8_attend_part(s, heads, kv, hd, 4)
    part = X.DevBuf.of(c2, np.zeros(floats + 4, np.float32))
    dk, dv, dq = (X.DevBuf(c2, (n, w, hd), np.uint16) for w in (kv, kv, heads))
    o = X.DevBuf(c2, (n, heads, hd), np.uint16)

    def once():
        X.kv8_append(c2, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
        X.kv8_attend(c2, d.h, s, heads, dq.h, heads * hd, 0.1, o.h, X.DT_BF16, heads * hd, part.h, floats)
        X.kv8_advance(c2, d.h, s)

    graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
    c2.sync()
    assert hip.hipStreamBeginCapture(st, 2) == 0
    once()
    with pytest.raises(X.ExnError) as e:
        X.Seqs(c2, [1])                                # a plan is not made in a capture
    assert e.value.code == X.ESTATE
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for i in range(6):
        kb, _ = normal(rng, (n, kv, hd), "bf16")
        vb, _ = normal(rng, (n, kv, hd), "bf16")
        qb, q = normal(rng, (n, heads, hd), "bf16")
        for b, a in ((dk, kb), (dv, vb), (dq, qb)):
            b.upload(a)
        if i % 3 == 2:
            once()                                     # the program's own eager step between
        else:
            assert hip.hipGraphLaunch(ex, st) == 0
        c2.sync()
        m.append(kb, vb, new)
        want, tol = m.attend(q, new, 0.1, "bf16")
        m.advance(new)
        d.same()
        assert off(pm.value(o.get(), "bf16"), want, tol) <= 1
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    X.call("exn_set_stream", c2.h, None)
    assert hip.hipStreamDestroy(st) == 0
    for b in (*d.b.values(), part, dk, dv, dq, o):
        b.free()
    c2.close()


@pytest.mark.parametrize("new", [1, 40])
def test_captured_splits(ctx, new):
    """Calls that split keys over workgroups and join them, captured and replayed over lengths that
    change, with eager calls of other sizes on the same scratch between."""
    hip = ctypes.CDLL("libamdhip64.so")
    rng = np.random.default_rng([19, new])
    kv, hd, heads, cols = 2, 128, 8, 60
    say("captured splits", new)
    c2 = X.Context(0)
    st = ctypes.c_void_p()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(st), 1) == 0
    X.call("exn_set_stream", c2.h, st)
    m, d = filled(c2, "fp16", [3000, 10, 900], kv, hd, cols, rng)
    plans = [X.Seqs(c2, [new] * 3), X.Seqs(c2, [2, 0, 17])]
    floats = max(X.kv8_attend_part(s, heads, kv, hd, cols) for s in plans)
    part = X.DevBuf.of(c2, np.zeros(floats + 4, np.float32))
    dq, o = (X.DevBuf(c2, (3 * max(new, 7), heads, hd), np.uint16) for _ in range(2))

    def once(s):
        X.kv8_attend(c2, d.h, s, heads, dq.h, heads * hd, 0.1, o.h, X.DT_BF16, heads * hd, part.h, floats)

    graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
    c2.sync()
    assert hip.hipStreamBeginCapture(st, 2) == 0
    once(plans[0])
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for lens in ([3000, 10, 900], [64, 3700, 0], [1, 2, 3], [3800, 3800, 3800]):
        m.lens[:] = lens
        d.b["lens"].upload(m.lens)
        qb, q = normal(rng, (3 * max(new, 7), heads, hd), "fp16")
        dq.upload(qb)
        for s, lens in ((plans[0], [new] * 3), (plans[1], [2, 0, 17])):
            if s is plans[0]:
                assert hip.hipGraphLaunch(ex, st) == 0
            else:
                once(s)
            c2.sync()
            n = sum(lens)
            want, tol = m.attend(q[:n], lens, 0.1, "bf16")
            assert off(pm.value(o.get()[:n], "bf16"), want, tol) <= 1
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    X.call("exn_set_stream", c2.h, None)
    assert hip.hipStreamDestroy(st) == 0
    for b in (*d.b.values(), part, dq, o):
        b.free()
    c2.close()
