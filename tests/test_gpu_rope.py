"""Rows of heads normed and turned by their positions on the GPU, against a plain form in 64 bits
(prompts_rope.py, which derives the tolerances).  Needs an MI355X."""
import ctypes
import sys

import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
import prompts_rope as pr

pytestmark = pytest.mark.gpu
DT = {"fp16": X.DT_F16, "bf16": X.DT_BF16, "fp32": X.DT_F32}


def say(*a):
    print("[gpu]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx():
    c = X.Context(0)
    yield c
    c.close()


def held(x, t):
    """fp32 values as the type holds them (patterns, or fp32 itself) and as 64-bit values."""
    x = np.asarray(x, np.float32)
    if t == "fp32":
        return x, x.astype(np.float64)
    b = pm.bits(pm.rounded(x, t), t)
    return b, pm.value(b, t)


def value(b, t):
    return b.astype(np.float64) if t == "fp32" else pm.value(b, t)


def padded(b, pad):
    """Rows with PAD unused values after each (NaN)."""
    n = b.shape[0]
    out = np.full((n, b[0].size + pad), np.nan if b.dtype == np.float32 else 0x7FFF, b.dtype)
    out[:, :b[0].size] = b.reshape(n, -1)
    return out


def off(got, want, tol):
    assert np.isfinite(got).all()
    return float((abs(got - want) / tol).max(initial=0))


def run(ctx, lens, heads, kv, hd, freqs, layout, dt, odt, rng, norm=True, axis=None, amp=1.0, pos=None, at=None, eps=1e-6,
        spread=2.0, place=False, given=None):
    """One call, q and k with unused values after their rows; the worst distance over its tolerance."""
    rows = sum(lens)
    qx, kx = given or (spread * rng.standard_normal((rows, h, hd)) for h in (heads, kv))
    qb, q = held(qx, dt)
    kb, k = held(kx, dt)
    w = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    s, r = X.Seqs(ctx, lens), X.Rope(ctx, freqs, layout, axis, amp)
    t = np.float32 if odt == "fp32" else np.uint16
    filled = 7.0 if odt == "fp32" else 0x1234
    dq, dk = X.DevBuf.of(ctx, padded(qb, 24)), X.DevBuf.of(ctx, padded(kb, 0))
    if place:
        oq, ok, pq, pk = dq, dk, 24, 0
    else:
        pq, pk = 8, 16
        oq, ok = (X.DevBuf.of(ctx, np.full((rows + 1, h * hd + p), filled, t)) for h, p in ((heads, pq), (kv, pk)))
    dw = [None if x is None else X.DevBuf.of(ctx, x) for x in w]
    dp = None if pos is None else X.DevBuf.of(ctx, np.ascontiguousarray(pos, np.int32))
    da = None if at is None else X.DevBuf.of(ctx, np.asarray(at, np.int32))
    X.rope_rows(ctx, r, s, hd, DT[dt], DT[odt], (heads, dq.h, heads * hd + 24, dw[0].h if norm else None, oq.h, heads * hd + pq),
                (kv, dk.h, kv * hd, dw[1].h if norm else None, ok.h, kv * hd + pk) if kv else (0, None, 0, None, None, 0),
                eps, dp.h if dp else None, da.h if da else None)
    if pos is None:
        pos = np.concatenate([np.arange(n, dtype=np.int64) + (0 if at is None else at[i]) for i, n in enumerate(lens)] or [[]])
        pos = pos.reshape(-1, 1)
    worst = 0.0
    for o, pad, x, wt, h in ((oq, pq, q, w[0], heads), (ok, pk, k, w[1], kv)):
        if h == 0:
            continue
        got = o.get()
        if not place:
            assert (got[rows:] == filled).all() and (got[:, h * hd:] == filled).all()
        want, tol = pr.rope_rows(x, wt, eps, pos, freqs, axis, layout, amp, odt)
        worst = max(worst, off(value(got[:rows, :h * hd], odt).reshape(want.shape), want, tol))
    return worst


@pytest.mark.parametrize("dt,odt", [("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp16"), ("fp32", "fp32"), ("bf16", "fp16"),
                                    ("fp16", "fp32"), ("fp32", "bf16"), ("fp16", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("hd,pairs", [(128, 64), (64, 32), (128, 32), (64, 9), (8, 1), (8, 4), (72, 36), (80, 40), (96, 20),
                                      (256, 128), (256, 64), (192, 33), (40, 8), (128, 63)])
@pytest.mark.parametrize("layout", [X.ROPE_HALF, X.ROPE_PAIRS], ids=["half", "pairs"])
def test_rows(ctx, hd, pairs, layout, dt, odt):
    rng = np.random.default_rng([hd, pairs, layout])
    say("rope", hd, pairs, layout, dt, odt)
    freqs = X.rope_freqs(2 * pairs, 1e4)
    for lens, heads, kv, norm in (([1], 4, 1, True), ([3, 0, 17], 5, 2, False), ([8, 9, 1, 1], 32, 8, True), ([2] * 20, 1, 1, True)):
        r = run(ctx, lens, heads, kv, hd, freqs, layout, dt, odt, rng, norm, at=rng.integers(0, 5000, len(lens)))
        say(lens, heads, kv, norm, "worst", r)
        assert r <= 1


@pytest.mark.parametrize("layout", [X.ROPE_HALF, X.ROPE_PAIRS], ids=["half", "pairs"])
def test_axes_amplitude_and_heads(ctx, layout):
    """Positions on several axes, of either sign; a factor of all; q alone; many heads."""
    rng = np.random.default_rng(41)
    say("axes", layout)
    freqs = X.rope_freqs(128, 5e6)
    axis = [j % 3 if j < 60 else 0 for j in range(64)]
    pos = rng.integers(-300, 4000, (70, 3))
    assert run(ctx, [40, 30], 32, 8, 128, freqs, layout, "fp16", "fp16", rng, axis=axis, amp=1.14, pos=pos) <= 1
    assert run(ctx, [40, 30], 16, 0, 128, freqs, layout, "bf16", "bf16", rng, axis=[j % 8 for j in range(64)],
               pos=rng.integers(0, 100, (70, 8))) <= 1
    assert run(ctx, [40, 30], 3, 1, 128, freqs, layout, "bf16", "bf16", rng, amp=-0.5, pos=pos[:, :1]) <= 1
    assert run(ctx, [3, 9], 1024, 1024, 64, freqs[:32], layout, "fp16", "bf16", rng) <= 1


def test_more_axes_than_are_named(ctx):
    """Positions may have axes by which no pair turns: their rows are as far apart as the rotary says."""
    rng = np.random.default_rng(47)
    say("axes that no pair names")
    pos = rng.integers(-50, 900, (21, 3)).astype(np.int32)
    freqs = X.rope_freqs(8, 1e4)
    for axis in (None, [1, 0, 1, 0]):
        b, x = held(rng.standard_normal((21, 4, 64)), "fp16")
        s, r = X.Seqs(ctx, [20, 1]), X.Rope(ctx, freqs, X.ROPE_HALF, axis, axes=3)
        d, dp = X.DevBuf.of(ctx, b), X.DevBuf.of(ctx, pos)
        X.rope_rows(ctx, r, s, 64, X.DT_F16, X.DT_F16, (4, d.h, 256, None, d.h, 256), pos=dp.h)
        want, tol = pr.rope_rows(x, None, 0.0, pos, freqs, axis, 0, 1.0, "fp16")
        assert off(pm.value(d.get(), "fp16"), want, tol) <= 1


@pytest.mark.parametrize("far", [131071, 10 ** 6, (1 << 31) - 40, -(1 << 31)])
def test_far_positions(ctx, far):
    """Angles of far positions, to fp32's own rounding."""
    rng = np.random.default_rng(42)
    say("far", far)
    freqs = X.rope_freqs(128, 1e4, X.ROPE_INDEX, 8.0, 8192, 1, 32)
    assert run(ctx, [33, 2], 4, 2, 128, freqs, X.ROPE_HALF, "fp32", "fp32", rng, at=[far, far]) <= 1
    freqs = [1.0, 1024.0, -3.0, 1e-9, 0.0, 6.2831853, 512.25, 0.5]
    assert run(ctx, [33, 2], 4, 2, 64, freqs, X.ROPE_PAIRS, "fp32", "fp32", rng, norm=False, at=[far, 0]) <= 1


@pytest.mark.parametrize("layout,pairs", [(X.ROPE_HALF, 64), (X.ROPE_HALF, 30), (X.ROPE_PAIRS, 64)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_in_place(ctx, dt, layout, pairs):
    rng = np.random.default_rng(43)
    say("in place", dt, layout, pairs)
    assert run(ctx, [100, 1, 0, 33], 12, 4, 128, X.rope_freqs(2 * pairs, 1e4), layout, dt, dt, rng, place=True) <= 1


def test_parts_of_one_row(ctx):
    """q | k | v rows of a fused product, in place, as packed attention takes them: v is left as it was."""
    rng = np.random.default_rng(44)
    heads, kv, hd, lens = 32, 8, 128, [129, 40]
    ld, rows = (heads + 2 * kv) * hd, 169
    b, x = held(2 * rng.standard_normal((rows, heads + 2 * kv, hd)), "fp16")
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    freqs = X.rope_freqs(hd, 5e6)
    s, r = X.Seqs(ctx, lens), X.Rope(ctx, freqs, X.ROPE_PAIRS)
    d, wq, wk = X.DevBuf.of(ctx, b), X.DevBuf.of(ctx, w[0]), X.DevBuf.of(ctx, w[1])
    say("fused rows")
    X.rope_rows(ctx, r, s, hd, X.DT_F16, X.DT_F16, (heads, d.h, ld, wq.h, d.h, ld),
                (kv, d.at(2 * heads * hd), ld, wk.h, d.at(2 * heads * hd), ld), 1e-6)
    got = d.get()
    assert np.array_equal(got[:, heads + kv:], b[:, heads + kv:])
    pos = np.concatenate([np.arange(n) for n in lens])[:, None]
    for a, z, wt in ((0, heads, w[0]), (heads, heads + kv, w[1])):
        want, tol = pr.rope_rows(x[:, a:z], wt, 1e-6, pos, freqs, None, 1, 1.0, "fp16")
        assert off(pm.value(got[:, a:z], "fp16"), want, tol) <= 1
    o = X.DevBuf(ctx, (rows, heads, hd), np.uint16)
    X.attend_packed(ctx, s, X.DT_F16, heads, kv, hd, d.h, ld, d.at(heads * hd * 2), ld, d.at((heads + kv) * hd * 2), ld,
                    hd ** -0.5, o.h, X.DT_BF16, heads * hd)
    y = pm.value(got, "fp16")
    want, tol = pm.packed(y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], lens, hd ** -0.5, "fp16", "bf16")
    assert off(pm.value(o.get(), "bf16"), want, tol) <= 1


def test_sizes_at_the_ends_of_the_range(ctx):
    """Squares past fp32's range or under it; heads of zeros; eps that decides."""
    rng = np.random.default_rng(45)
    say("sizes")
    freqs = X.rope_freqs(128, 1e4)
    for spread, eps in ((1e19, 1e-6), (5e37, 1e-6), (1e-25, 1e-6), (1e-30, 0.0), (1e-36, 0.0), (1e-20, 1e-38), (1e-3, 1e-5)):
        x = [rng.standard_normal((20, h, 128)) for h in (4, 2)]
        # heads of one size each, and one whose values are far apart
        for a in x:
            a *= spread
            a[3, 0, 1:] *= 1e-4
        for dt in ("bf16", "fp32"):
            r = run(ctx, [20], 4, 2, 128, freqs, X.ROPE_HALF, dt, "fp32", rng, eps=eps, given=x)
            say(spread, eps, dt, "worst", r)
            assert r <= 1
    x = [np.zeros((3, 2, 128)), np.zeros((3, 1, 128))]
    assert run(ctx, [3], 2, 1, 128, freqs, X.ROPE_PAIRS, "fp16", "fp16", rng, given=x) <= 1


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_values_that_are_not_finite(ctx, bad):
    """Without a norm: its own pair and nothing else, dims that are not turned as they are.  With one: its head only."""
    rng = np.random.default_rng(46)
    say("not finite", bad)
    freqs = X.rope_freqs(64, 1e4)
    for layout in (X.ROPE_HALF, X.ROPE_PAIRS):
        qb, q = held(rng.standard_normal((9, 4, 128)), "bf16")
        p = pm.bits(np.float32(bad), "bf16")[0]
        qb[2, 1, 3] = p
        qb[5, 2, 100] = p
        o = X.DevBuf(ctx, (9, 4, 128), np.uint16)
        dq, w = X.DevBuf.of(ctx, qb), X.DevBuf.of(ctx, np.ones(128, np.float32))
        for norm in (False, True):
            X.rope_rows(ctx, X.Rope(ctx, freqs, layout), X.Seqs(ctx, [9]), 128, X.DT_BF16, X.DT_BF16,
                        (4, dq.h, 512, w.h if norm else None, o.h, 512))
            got = pm.value(o.get(), "bf16")
            want, tol = pr.rope_rows(q, np.ones(128) if norm else None, 0.0, np.arange(9)[:, None], freqs, None, layout, 1.0, "bf16")
            same = np.ones(got.shape, bool)
            if norm:
                same[2, 1], same[5, 2] = False, False
                assert np.isnan(got[2, 1, 3]) and np.isnan(got[5, 2, 100])
            else:
                pair = [3, 35] if layout == X.ROPE_HALF else [2, 3]
                same[2, 1, pair], same[5, 2, 100] = False, False
                assert not np.isfinite(got[2, 1, pair]).any()
                assert np.isnan(got[5, 2, 100]) if np.isnan(bad) else got[5, 2, 100] == bad
            assert (abs(got - want)[same] <= tol[same]).all()


def test_rows_far_apart(ctx):
    """Strides with which a sequence's rows are over 2^32 bytes apart."""
    rng = np.random.default_rng(47)
    n, hd, ld = 150, 64, 1 << 24
    say("far rows")
    buf = X.DevBuf(ctx, (n * ld,), np.uint16)
    b, x = held(rng.standard_normal((n, 1, hd)), "fp16")
    for i in range(n):
        row = np.ascontiguousarray(b[i, 0])
        X.call("exn_upload", ctx.h, buf.at(2 * i * ld), X.ptr(row), row.nbytes)
    freqs = X.rope_freqs(hd, 1e4)
    s, r = X.Seqs(ctx, [n]), X.Rope(ctx, freqs)
    X.rope_rows(ctx, r, s, hd, X.DT_F16, X.DT_F16, (1, buf.h, ld, None, buf.h, ld))
    got = np.zeros((n, 1, hd), np.uint16)
    for i in range(n):
        X.call("exn_download", ctx.h, X.ptr(got[i, 0]), buf.at(2 * i * ld), 2 * hd)
    buf.free()
    want, tol = pr.rope_rows(x, None, 0.0, np.arange(n)[:, None], freqs, None, 0, 1.0, "fp16")
    assert off(pm.value(got, "fp16"), want, tol) <= 1


def test_no_rows(ctx):
    s, r = X.Seqs(ctx, [0, 0]), X.Rope(ctx, [0.5])
    o = X.DevBuf.of(ctx, np.full((2, 64), 0x1234, np.uint16))
    say("no rows")
    X.rope_rows(ctx, r, s, 64, X.DT_F16, X.DT_F16, (1, o.h, 64, None, o.h, 64))
    assert (o.get() == 0x1234).all()


def test_long_rows(ctx):
    """Thousands of rows: the shares of a tile's heads, and every row's own position."""
    rng = np.random.default_rng(48)
    say("long")
    assert run(ctx, [4097, 1, 1030], 32, 8, 128, X.rope_freqs(128, 5e6), X.ROPE_HALF, "bf16", "bf16", rng, at=[0, 77, 70000]) <= 1


def test_the_encoders_own_rotary(ctx):
    """The frequencies and axes with which the prompt encoder's table is made give its cosines and sines."""
    say("encoder's table")
    rng = np.random.default_rng(49)
    pos = np.ascontiguousarray(rng.integers(0, 1500, (50, 3)), np.int32)
    cs = X.enc_rope_table(50, pos).reshape(50, 64, 2)
    freqs = X.rope_freqs(128, X.ENC_ROPE_BASE)
    axis = [j % 3 if j < 60 else 0 for j in range(64)]
    one = np.zeros((50, 1, 128), np.float32)
    one[..., 0::2] = 1
    d, o, p = X.DevBuf.of(ctx, one), X.DevBuf(ctx, (50, 1, 128), np.float32), X.DevBuf.of(ctx, pos)
    X.rope_rows(ctx, X.Rope(ctx, freqs, X.ROPE_PAIRS, axis), X.Seqs(ctx, [50]), 128, X.DT_F32, X.DT_F32, (1, d.h, 128, None, o.h, 128),
                pos=p.h)
    got = o.get().reshape(50, 64, 2)
    # the table's own entries are fp32 cosines of 64-bit (or fp32) angles: both within their roundings of the same values
    a = pr.angles(pos, freqs, axis)
    want = np.stack([np.cos(a), np.sin(a)], -1).astype(np.float64)
    assert abs(got - want).max() <= 10 * 2.0 ** -24
    assert abs(cs - want).max() <= 1500 * 2.0 ** -24 + 10 * 2.0 ** -24
