"""A key that takes nearly all of a row's weight and whose value is nothing (a sink, which trained
models' first tokens are): the result is the sum of many weights far under the largest, so that none
may be lost.  The prompt side's attention against prompts_model.py's plain form in 64 bits.

The bound is that form's, but for fp16 weights' least value: a weight that stands for 2^-32 of a row's
largest and more takes part, so that each of m keys adds an error of at most 2^-32 max |v| where the plain
form's bound has half of fp16's least value at a largest weight of 1, 2^-25.  Needs an MI355X."""
import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prompts import DT, attended, ctx, filled, normal, off, say  # noqa: F401

pytestmark = pytest.mark.gpu
SCALE, S = 0.125, 17.0        # a sink's score: the others' are normal, of 1


def bound(tol, m, vmax, odt):
    """pm.attend's tolerance (1.01 low + a rounding of it) with 2^-32 in place of 2^-25."""
    return tol - (1.01 + pm.HALF[odt]) * m * (2.0 ** -25 - 2.0 ** -32) * vmax


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 8, 40])
@pytest.mark.parametrize("split", [True, False])
def test_cache_sink(ctx, split, new, hd, dt):  # noqa: F811
    """With scratch, the sink is in one split's sums; without, the other keys' weights stand beside it."""
    rng = np.random.default_rng([new, hd])
    say("cache sink", split, new, hd, dt)
    kv, heads, n = 2, 8, 8100
    m, d = filled(ctx, dt, [n], kv, hd, (n + 64) // 64 + 1, rng)
    qb, q = normal(rng, (new, heads, hd), dt, 8 / hd ** 0.5)
    qb[:, :, 0], q[:, :, 0] = pm.bits(np.float32(16), dt), 16.0
    first = m.table[0, 0]
    m.k[:, :, :, 0] = 0
    m.k[first] = rng.integers(-16, 17, m.k[first].shape)
    m.k[first, :, :, 0] = 0
    m.k[first, :, 0] = 0
    m.k[first, :, 0, 0] = 127
    m.scales[first, :, 0] = S / (16 * SCALE) / 127
    m.tk[:, :, :, 0] = 0
    m.v[:] = rng.integers(32, 128, m.v.shape)          # values above 0: their sums are not
    m.tv &= 0x7FFF
    m.v[first, :, :, 0] = 0
    for x in ("k", "v", "scales", "tk", "tv"):
        d.b[x].upload(getattr(m, x))
    want, tol = m.attend(q, [new], SCALE, dt)
    k, v, _ = m.rows(0, new)
    got = attended(ctx, d, qb, [new], heads, dt, SCALE, None if split else lambda n: 0)
    r = off(got, want, bound(tol, len(k), v.max((0, 2)).min(), dt))
    say("worst", r, "rel", np.linalg.norm(got - want) / np.linalg.norm(want))
    assert r <= 1


@pytest.mark.parametrize("odt", ["fp16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_packed_sink(ctx, hd, odt):  # noqa: F811
    rng = np.random.default_rng(hd)
    say("packed sink", hd, odt)
    n, heads = 5000, 2
    qb, q = normal(rng, (n, heads, hd), "fp16", 8 / hd ** 0.5)
    kb, k = normal(rng, (n, 1, hd), "fp16")
    vb = pm.bits(pm.rounded(rng.uniform(0.5, 2, (n, 1, hd)), "fp16"), "fp16")
    qb[:, :, 0] = pm.bits(np.float32(16), "fp16")
    kb[:, :, 0] = kb[0] = 0
    kb[0, 0, 0] = pm.bits(np.float32(S / (16 * SCALE)), "fp16")
    vb[0] = 0
    q, k, v = (pm.value(b, "fp16") for b in (qb, kb, vb))
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (n, heads, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, [n]), X.DT_F16, heads, 1, hd, dq.h, heads * hd, dk.h, hd, dv.h, hd, SCALE, o.h, DT[odt],
                    heads * hd)
    want, tol = pm.packed(q, k, v, [n], SCALE, "fp16", odt)
    got = pm.value(o.get(), odt)
    r = off(got, want, bound(tol, n, v.max(), odt))
    say("worst", r, "rel", np.linalg.norm(got - want) / np.linalg.norm(want))
    assert r <= 1
