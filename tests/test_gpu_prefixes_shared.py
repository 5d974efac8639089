"""Attention over the 8-bit cache for sequences that begin alike, in calls that the plan shares (asserted in each), against
the plain form in 64 bits (prompts_model.py derives the tolerances): groups of more heads than a workgroup's rows, prefixes of
every tiling, pages past 4 GB.  Needs an MI355X."""
import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prefixes import LONG, alike, ctx, say, step
from test_gpu_prompts import normal, off

pytestmark = pytest.mark.gpu


def shares(ctx, of, blocks, new, heads, kv, hd, cols):
    """Whether the plan's calls are shared: their scratch is not kv8_attend's."""
    s = X.Seqs(ctx, new)
    return X.attend_shared_part(s, X.Prefixes(ctx, s, of, blocks), heads, kv, hd, cols) != X.kv8_attend_part(s, heads, kv, hd, cols)


def run(ctx, seed, dt, odt, heads, kv, hd, of, blocks, own, new, steps=2, part=None):
    rng = np.random.default_rng(seed)
    before = [n + 64 * (blocks[g] if g >= 0 else 0) for n, g in zip(own, of)]
    m, d = alike(ctx, dt, kv, hd, of, blocks, before, rng)
    if part:
        part(m)
        d.b["table"].upload(m.table)
    assert shares(ctx, of, blocks, new, heads, kv, hd, m.cols)
    for _ in range(steps):
        r = step(ctx, m, d, of, blocks, new, heads, odt, rng)
        say("worst", r)
        assert r <= 1


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv,hd", [(17, 1, 64), (20, 1, 128), (34, 2, 128), (48, 1, 64), (96, 4, 128)])
def test_groups_of_more_than_sixteen(ctx, heads, kv, hd, dt, odt):
    """More heads a key/value head than a row tile holds: several workgroups take a sequence's own blocks."""
    say("large groups", heads, kv, hd, dt, odt)

    def part(m):
        m.table[3, 9] = m.table[3, -1]
        m.table[5, 0] = m.table[5, -2]

    run(ctx, [71, heads], dt, odt, heads, kv, hd, [0] * 12, [40], [(53 * i) % 190 for i in range(12)], [1] * 12, part=part)


@pytest.mark.parametrize("heads,kv,hd,tokens", [(17, 1, 64, 64000), (40, 2, 64, 64000), (34, 2, 128, 60000), (20, 4, 64, 40000)])
def test_groups_of_more_than_sixteen_after_long_prefixes(ctx, heads, kv, hd, tokens):
    """Two sequences, of as many rows as few_rows takes of a prefix: its rows and its chunks of heads."""
    say("large groups, two sequences", heads, kv, hd, tokens)
    run(ctx, [72, heads], "bf16", "bf16", heads, kv, hd, [0, 0], [tokens // 64], [70, 201], [1, 1], 1)


# as test_gpu_prefixes' SHAPES, with prefixes that the plan shares: of, blocks, tokens of its own before the step, new tokens
SHAPES = {
    "two": ([0, 0], [700], [5, 60], [1, 1]),
    "new blocks": ([0] * 9, [40], [63, 0, 127, 62, 61, 126, 190, 1, 64], [1] * 9),
    "chunks": ([0] * 14, [66], [10 + 9 * i for i in range(14)], [5, 1, 8] * 4 + [7, 3]),
    "mixed": ([1, 0, -1, 0, 1, -1] * 5, [50, 31], [3, 70, 100, 0, 64, 0] * 5, [1, 1, 1, 1, 1, 2] * 5),
    "waiting": ([0] * 24, [33], [0, 5, 9, 70] * 6, [0, 1, 0, 1] * 6),
    "many": ([i % 3 - 1 for i in range(60)], [45, 20], [(7 * i) % 90 for i in range(60)], [1] * 60),
    "one alone": ([0] * 12 + [1], [30, 40], [9] * 13, [1] * 13),
}


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (8, 4, 64), (3, 3, 128), (12, 4, 64)])
@pytest.mark.parametrize("shape", SHAPES)
def test_shared(ctx, shape, heads, kv, hd, dt, odt):
    say("shared", shape, heads, kv, hd, dt, odt)
    of, blocks, own, new = SHAPES[shape]
    run(ctx, [73, len(of), heads], dt, odt, heads, kv, hd, of, blocks, own, new)


@pytest.mark.parametrize("shape", LONG)
def test_long_shapes_are_shared(ctx, shape):
    """Of test_gpu_prefixes' long shapes all but the one of few sequences with rows."""
    of, blocks, own, new = LONG[shape]
    cols = max(n + 64 * (blocks[g] if g >= 0 else 0) for n, g in zip(own, of)) // 64 + 4
    for heads, kv, hd in ((8, 2, 128), (4, 1, 64), (3, 3, 128), (4, 2, 64), (5, 1, 128), (2, 2, 64)):
        assert shares(ctx, of, blocks, new, heads, kv, hd, cols) == (shape != "waiting"), (heads, kv, hd)


@pytest.mark.parametrize("n,new,heads,blocks", [(6, 1, 8, 30), (12, 1, 16, 20), (12, 1, 32, 20), (24, 5, 32, 20)])
def test_pages_past_4_gb(ctx, n, new, heads, blocks):
    """Pages whose codes lie past 2^32 bytes, the prefix's and a sequence's own: in each tiling of a prefix's rows."""
    rng = np.random.default_rng([74, n])
    kv, hd, pages = 8, 128, 66000
    of, new = [0] * n, [new] * n
    say("past 4 GB", n, new[0], heads, blocks)
    m, d = alike(ctx, "fp16", kv, hd, of, [blocks], [64 * blocks + (31 * i) % 150 for i in range(n)], rng, spare=0)
    # only the pages in use go up, to the end of the large arrays
    used = np.unique(m.table)
    move = {int(p): pages - 1 - i for i, p in enumerate(used)}
    assert (pages - len(used)) * kv * 64 * hd > 2 ** 32
    big = {x: X.DevBuf(ctx, (pages, kv, 64, hd), np.int8) for x in ("k", "v")}
    sc = X.DevBuf(ctx, (pages, kv, 2), np.float32)
    for buf, name in ((big["k"], "k"), (big["v"], "v"), (sc, "scales")):
        x = np.ascontiguousarray(getattr(m, name)[used[::-1]])
        X.call("exn_upload", ctx.h, buf.at((pages - len(used)) * x[0].nbytes), X.ptr(x), x.nbytes)
    d.b["table"].upload(np.vectorize(move.get)(m.table).astype(np.int32))
    h = X.Kv8(X.DT_F16, kv, hd, pages, n, m.cols, big["k"].ptr, big["v"].ptr, sc.ptr,
              *(d.b[x].ptr for x in ("tk", "tv", "table", "lens")))
    s = X.Seqs(ctx, new)
    p = X.Prefixes(ctx, s, of, [blocks])
    rows = sum(new)
    kb, vb = (normal(rng, (rows, kv, hd), "fp16")[0] for _ in range(2))
    qb, q = normal(rng, (rows, heads, hd), "fp16")
    dk, dv, dq, o = X.DevBuf.of(ctx, kb), X.DevBuf.of(ctx, vb), X.DevBuf.of(ctx, qb), X.DevBuf(ctx, (rows, heads, hd), np.uint16)
    X.kv8_append(ctx, h, s, dk.h, kv * hd, dv.h, kv * hd)
    floats = X.attend_shared_part(s, p, heads, kv, hd, m.cols)
    assert floats != X.kv8_attend_part(s, heads, kv, hd, m.cols)
    part = X.DevBuf(ctx, (floats,), np.float32)
    X.attend_shared(ctx, h, s, p, heads, dq.h, heads * hd, 0.09, o.h, X.DT_F16, heads * hd, part.h, floats)
    got = pm.value(o.get(), "fp16")
    for b in (*big.values(), sc):
        b.free()
    m.append(kb, vb, new)
    want, tol = m.attend(q, new, 0.09, "fp16")
    assert off(got, want, tol) <= 1


@pytest.mark.parametrize("n,heads,kv,hd,blocks", [(64, 32, 32, 128, 8), (96, 32, 32, 128, 3), (300, 16, 8, 128, 8)])
def test_short_prefixes_of_many_sequences(ctx, n, heads, kv, hd, blocks):
    """A few blocks, which many sequences of many heads read: shared all the same; one table has parted, one sequence is new."""
    say("short prefixes", n, heads, kv, hd, blocks)

    def part(m):
        m.table[7, 1] = m.table[7, -1]
        m.lens[9] = 0

    rng = np.random.default_rng([75, n])
    of, before = [0] * n, [64 * blocks + (11 * i) % 60 for i in range(n)]
    m, d = alike(ctx, "bf16", kv, hd, of, [blocks], before, rng, cols=blocks + 2, spare=0)
    part(m)
    d.b["table"].upload(m.table)
    d.b["lens"].upload(m.lens)
    assert shares(ctx, of, [blocks], [1] * n, heads, kv, hd, m.cols)
    r = step(ctx, m, d, of, [blocks], [1] * n, heads, "bf16", rng)
    say("worst", r)
    assert r <= 1
