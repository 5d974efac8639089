"""Norm weights at the ends of fp32's range, on the GPU, against the plain form in 64 bits (prompts_rope.py derives the
tolerances): what a head comes to is in the range, so it is to come out.  Needs an MI355X."""
import numpy as np
import pytest

import exn_hip as X
import prompts_rope as pr
from test_gpu_rope import DT, ctx, held, off, say, value

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odt", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", [X.ROPE_HALF, X.ROPE_PAIRS])
@pytest.mark.parametrize("spread,weight,eps", [(5e16, 1e-27, 1e-6), (5e-15, 1e25, 0.0), (1e-20, 1e30, 0.0), (1e25, 1e-30, 1e-6),
                                               (1.0, 1e-35, 1e-6), (1.0, 1e35, 1e-6)])
def test_weights_at_the_ends_of_the_range(ctx, spread, weight, eps, layout, odt):
    """Heads of large values and small weights and the other way round: 1 / the root times the weight is past the range,
    or under it, where the head is not."""
    rng = np.random.default_rng(81)
    say("weights", spread, weight, eps, layout, odt)
    rows, heads, hd = 9, 3, 128
    xb, x = held(spread * rng.standard_normal((rows, heads, hd)), "fp32")
    w = (weight * (1 + 0.3 * rng.random(hd))).astype(np.float32)
    freqs = X.rope_freqs(hd, 1e4)
    s, r = X.Seqs(ctx, [rows]), X.Rope(ctx, freqs, layout)
    dx, dw = X.DevBuf.of(ctx, xb), X.DevBuf.of(ctx, w)
    o = X.DevBuf(ctx, (rows, heads, hd), np.float32 if odt == "fp32" else np.uint16)
    X.rope_rows(ctx, r, s, hd, X.DT_F32, DT[odt], (heads, dx.h, heads * hd, dw.h, o.h, heads * hd), eps=eps)
    want, tol = pr.rope_rows(x, w, eps, np.arange(rows)[:, None], freqs, None, layout, 1.0, odt)
    worst = off(value(o.get(), odt), want, tol)
    say("worst", worst)
    assert worst <= 1
