"""Values at the end of fp16's range in the prompt side's attention: a block's scale is rounded up to 12
significant bits, so that 127 of its steps may be up to 2^-11 more than the block's largest value, past
where fp16 rounds to infinity.  What is finite is read as finite, and so are means of it.  And values near
the end of fp32's.  Needs an MI355X."""
import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm
from test_gpu_prompts import attended, cache_of, ctx, filled, normal, off, say  # noqa: F401

pytestmark = pytest.mark.gpu
TOP = 65504.0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,part", [(1, True), (1, False), (8, True), (40, True), (40, False)])
def test_cache_of_the_largest_values(ctx, new, part, hd):  # noqa: F811
    """Values of +-65504 in every block, one sign a dim: the results are +-65504 whatever the weights (a
    mean of equal values, off by a weight's rounding: half a step of fp16 or none)."""
    rng = np.random.default_rng([new, hd])
    say("largest values", new, part, hd)
    kv, heads, n = 2, 8, 2200
    m, d = cache_of(ctx, "fp16", 1, kv, hd, 36, rng)
    kb, _ = normal(rng, (n, kv, hd), "fp16")
    sign = np.where(rng.integers(0, 2, (kv, hd)), TOP, -TOP)
    vb = pm.bits(np.broadcast_to(sign, (n, kv, hd)).astype(np.float32), "fp16")
    assert (abs(np.float64(pm.scale_of(sign[0])) * 127) > 65520)          # the case there is
    for rows in (n - new, new):
        s = X.Seqs(ctx, [rows])
        at = 0 if rows == n - new else n - new
        dk, dv = X.DevBuf.of(ctx, kb[at:at + rows]), X.DevBuf.of(ctx, vb[at:at + rows])
        X.kv8_append(ctx, d.h, s, dk.h, kv * hd, dv.h, kv * hd)
        rk, rv = (X.DevBuf(ctx, (rows, kv, hd), np.uint16) for _ in range(2))
        X.kv8_read(ctx, d.h, s, rk.h, kv * hd, rv.h, kv * hd)
        assert (pm.value(rv.get(), "fp16") == sign).all()
        if at == 0:
            X.kv8_advance(ctx, d.h, s)
    qb, _ = normal(rng, (new, heads, hd), "fp16")
    dq, o = X.DevBuf.of(ctx, qb), X.DevBuf(ctx, (new, heads, hd), np.uint16)
    floats = X.kv8_attend_part(s, heads, kv, hd, 36) if part else 0
    scratch = X.DevBuf(ctx, (floats + 4,), np.float32)
    X.kv8_attend(ctx, d.h, s, heads, dq.h, heads * hd, hd ** -0.5, o.h, X.DT_F16, heads * hd, scratch.h if floats else None,
                 floats)
    got = pm.value(o.get(), "fp16")
    assert (abs(got - np.repeat(sign, heads // kv, 0)) <= 32).all()       # a step there


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_largest_values(ctx, hd):  # noqa: F811
    rng = np.random.default_rng(hd)
    say("packed largest values", hd)
    n, heads = 300, 4
    qb, _ = normal(rng, (n, heads, hd), "fp16")
    kb, _ = normal(rng, (n, 1, hd), "fp16")
    sign = np.where(rng.integers(0, 2, (1, hd)), TOP, -TOP)
    vb = pm.bits(np.broadcast_to(sign, (n, 1, hd)).astype(np.float32), "fp16")
    dq, dk, dv = (X.DevBuf.of(ctx, b) for b in (qb, kb, vb))
    o = X.DevBuf(ctx, (n, heads, hd), np.uint16)
    X.attend_packed(ctx, X.Seqs(ctx, [n]), X.DT_F16, heads, 1, hd, dq.h, heads * hd, dk.h, hd, dv.h, hd, hd ** -0.5, o.h,
                    X.DT_F16, heads * hd)
    assert (abs(pm.value(o.get(), "fp16") - sign) <= 32).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 20])
def test_cache_of_very_large_values(ctx, new, hd):  # noqa: F811
    """bf16 values of 2^112 in an unfinished block whose keys' weights are 2^7 of the blocks before it, so
    that a reference lags by 7: the sums of values under weights that are held 2^7 higher still are past
    fp32's largest (2^14 x 4 keys x 2^112), under the weights themselves 2^121."""
    rng = np.random.default_rng([new, hd])
    say("very large values", new, hd)
    kv, heads, n = 2, 2, 256 + 4
    m, d = filled(ctx, "bf16", [n - new], kv, hd, 6, rng)
    qb = np.zeros((new, heads, hd), np.uint16)
    qb[:, :, 0] = pm.bits(np.float32(16), "bf16")
    q = pm.value(qb, "bf16")
    m.k[:, :, :, 0] = 0
    m.tk[:, :, :, 0] = pm.bits(np.float32(2.421875), "bf16")       # 16 x 2.42 x 0.125 = 4.84 = 7 ln 2
    vb, _ = normal(rng, m.tv.shape, "bf16")
    m.tv[:] = pm.bits(pm.rounded((2.0 ** 112 * (1.5 + 0.4 * np.sign(pm.value(vb, "bf16")))).astype(np.float32), "bf16"), "bf16")
    for x in ("k", "tk", "tv"):
        d.b[x].upload(getattr(m, x))
    want, tol = m.attend(q, [new], 0.125, "bf16")
    assert off(attended(ctx, d, qb, [new], heads, "bf16", 0.125), want, tol) <= 1
