"""Steps whose sequences get very different numbers of new tokens, tables much wider than their sequences,
and one long prompt alone: the prompt side's attention against prompts_model.py's plain form in 64 bits,
with its tolerances.  Needs an MI355X."""
import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prompts import DT, attended, cache_of, ctx, filled, normal, off, say, step  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "fp16")])
@pytest.mark.parametrize("hd", [64, 128])
def test_one_long_and_many_single(ctx, hd, dt, odt):  # noqa: F811
    rng = np.random.default_rng(hd)
    say("mixed step", hd, dt)
    lens = rng.integers(0, 2200, 24)
    new = [1] * 24
    new[5], new[11], new[17] = 76, 0, 3
    kv, heads, pages, cols = 2, 8, 200, 60
    m, d = filled(ctx, dt, lens, kv, hd, cols, rng, pages, rng.integers(0, pages, (24, cols)))
    qb, q = normal(rng, (sum(new), heads, hd), dt)
    want, tol = m.attend(q, new, hd ** -0.5, odt)
    for floats in (None, lambda n: 0):
        assert off(attended(ctx, d, qb, new, heads, odt, hd ** -0.5, floats), want, tol) <= 1


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_mixed_steps_into_wide_tables(ctx, dt):  # noqa: F811
    """Appended, read and attended too: tables of 500 blocks over sequences of up to 4."""
    rng = np.random.default_rng(31)
    say("wide tables", dt)
    table = np.full((4, 500), -1)
    table[:, :5] = rng.permutation(20).reshape(4, 5)
    m, d = cache_of(ctx, dt, 4, 2, 128, 500, rng, pages=20, table=table)
    for new in ([100, 1, 63, 0], [1, 70, 1, 1], [1, 1, 1, 1], [9, 1, 0, 2], [1, 1, 40, 130]):
        assert step(ctx, m, d, new, 8, "bf16", rng) <= 1


@pytest.mark.parametrize("dt,odt", [("fp16", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n", [1100, 1501])
def test_one_long_prompt(ctx, n, dt, odt):  # noqa: F811
    rng = np.random.default_rng(n)
    say("one prompt", n, dt)
    heads, kv, hd = 8, 2, 128
    qb, q = normal(rng, (n, heads, hd), dt)
    kb, k = normal(rng, (n, kv, hd), dt, 1.5)
    vb, v = normal(rng, (n, kv, hd), dt)
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (n, heads, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, [n]), DT[dt], heads, kv, hd, dq.h, heads * hd, dk.h, kv * hd, dv.h, kv * hd, hd ** -0.5,
                    o.h, DT[odt], heads * hd)
    want, tol = pm.packed(q, k, v, [n], hd ** -0.5, dt, odt)
    assert off(pm.value(o.get(), odt), want, tol) <= 1
