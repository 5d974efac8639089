"""Plain form, in 64 bits, of rows normed and turned by their positions (numpy), for the tests, with how far a
kernel in fp32 may be off."""
import numpy as np

HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8, "fp32": 2.0 ** -24}     # half a step, relative
LEAST = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134, "fp32": 2.0 ** -150}  # half the smallest step


def angles(pos, freqs, axis):
    """[row][pair], from positions [row][axes], in 80 bits."""
    axis = np.zeros(len(freqs), int) if axis is None else np.asarray(axis)
    return np.asarray(pos)[:, axis].astype(np.longdouble) * np.asarray(freqs, np.longdouble)


def rope_rows(x, w, eps, pos, freqs, axis, layout, amp, odt):
    """X [row][head][hd] normed by W (or None), its first 2 len(freqs) dims turned; LAYOUT 0 halves, 1 pairs.  The
    values and how far a kernel may be off them, element by element:
    - a norm: a sum of hd squares, off by at most (hd + 2) 2^-24 of it, whose root halves that; the mean, eps and the root
      itself, 2^-22; two products, 2^-23
    - a cosine or sine: the angle past the nearest quarter turn, at most pi / 4, is off by 3 2^-24 of it, the series by as
      much again and 2^-29; times AMP, 2^-24: 7 2^-24 of AMP in all
    - the two products and their sum, 2 2^-24 of what is added
    - the result is rounded to ODT"""
    x = np.asarray(x, np.float64)
    hd, p = x.shape[-1], len(freqs)
    held = 0.0
    if w is not None:
        with np.errstate(invalid="ignore", divide="ignore"):
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
        held = (hd + 2) * 2.0 ** -25 + 2.0 ** -22 + 2.0 ** -23
    a = angles(pos, freqs, axis)
    c, s = (f(a).astype(np.float64)[:, None] * amp for f in (np.cos, np.sin))
    u, v = (slice(0, p), slice(p, 2 * p)) if layout == 0 else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    y, tol = x.copy(), held * abs(x)
    y[..., u], y[..., v] = x[..., u] * c - x[..., v] * s, x[..., u] * s + x[..., v] * c
    both = (abs(x[..., u]) + abs(x[..., v])) * abs(amp) * (9 * 2.0 ** -24 + held)
    tol[..., u], tol[..., v] = both, both
    return y, tol + HALF[odt] * (abs(y) + tol) + LEAST[odt]
