"""Plain forms, in 64 bits, of the prompt side's attention and of its cache in 8 bits (numpy), for
the tests, with how far a 16-bit kernel may be off."""
import numpy as np

PAGE = 64
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative


def bits(x, t):
    """fp32 values that the type holds, as 16-bit patterns."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    return x.astype(np.float16).view(np.uint16) if t == "fp16" else (x.view(np.uint32) >> 16).astype(np.uint16)


def value(b, t):
    b = np.ascontiguousarray(b, dtype=np.uint16)
    return b.view(np.float16).astype(np.float64) if t == "fp16" else \
        (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, t):
    """x rounded to the type (nearest even), as 64-bit values."""
    x = np.asarray(x, dtype=np.float32)
    if t == "fp16":
        return x.astype(np.float16).astype(np.float64)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    return np.where(np.isnan(x), np.nan, r)


def attend(q, k, v, seen, scale, dt, odt, codes=False):
    """One head: q [n][hd] over k, v [m][hd], row i seeing the keys of seen [n][m]; zeros where it
    sees none.  The values and how far a kernel may be off them, element by element:
    - a weight p (at most 2^8 times the running largest: the sum of p is at least 1) is rounded to
      DT: half a step of p, and 2^-25 where fp16 has no smaller step; and, on the sum's side, the
      same again at most.  For bf16 in and fp16 out it is held as two bf16 parts: 2^-16 (CODES: a
      cache's codes of either type may take fp16 weights)
    - a score is a sum of hd products in fp32, off by at most hd 2^-24 sum |q k|, scaled (and
      SCALE log2(e) rounded: 2^-23 of it); p is off by as much times ln 2, plus 2^-22 of exp2 itself
    - the sums over m keys are off by at most m 2^-24 of the sum of |p v|
    - the result is rounded to ODT"""
    s = scale * (q @ k.T)
    s = np.where(seen, s, -np.inf)
    with np.errstate(invalid="ignore"):
        p = np.exp(s - s.max(1, keepdims=True))
    live = seen.any(1)
    p = np.where(live[:, None], p, 0.0)
    l = np.where(live, p.sum(1), 1.0)[:, None]
    # what is not seen weighs nothing, whatever it holds
    used = seen.any(0)
    k, v = np.where(used[:, None], k, 0.0), np.where(used[:, None], v, 0.0)
    o = p @ v / l
    m, hd = k.shape
    top = np.where(seen, abs(scale) * (abs(q) @ abs(k).T), 0).max(1, keepdims=True, initial=0)
    held = HALF[dt] if dt == odt or odt == "bf16" else HALF["fp16"] if codes else 2.0 ** -16
    c = 2 * held + 2 * m * 2.0 ** -24 + 2 * (top * (hd + 3) * 2.0 ** -24 + 2.0 ** -22)
    size = p @ abs(v) / l
    low = m * 2.0 ** -25 * abs(v).max(initial=0) if dt == "fp16" or codes else 0.0
    tol = 1.01 * (size * c + low) + HALF[odt] * (abs(o) + size * c + low) + (2.0 ** -25 if odt == "fp16" else 1e-38)
    return o, tol


def packed(q, k, v, lens, scale, dt, odt):
    """Causal attention of packed sequences: q [rows][heads][hd], k, v [rows][kv heads][hd]."""
    o, tol, r = np.zeros(q.shape), np.zeros(q.shape), 0
    group = q.shape[1] // k.shape[1]
    for n in lens:
        for h in range(q.shape[1]):
            if n:
                o[r:r + n, h], tol[r:r + n, h] = attend(q[r:r + n, h], k[r:r + n, h // group], v[r:r + n, h // group],
                                                        np.tri(n, dtype=bool), scale, dt, odt)
        r += n
    return o, tol


def scale_of(x):
    """A block's scale: its largest |x| / 127 in fp32, rounded up to 12 significant bits."""
    top = np.float32(np.abs(x).max())
    if not np.isfinite(top):
        return np.float32(np.nan)
    d = np.array(top / np.float32(127), np.float32).view(np.uint32)
    return ((d + np.uint32(0xFFF)) & np.uint32(0xFFFFF000)).view(np.float32)[()]


def codes_of(x, d):
    if not d > 0:
        return np.zeros(x.shape, np.int8)
    return np.rint(x.astype(np.float64) / np.float64(d)).astype(np.int8)


class Cache:
    """The cache in numpy: codes, scales, tails (16-bit patterns), table, lens."""

    def __init__(self, dt, seqs, kv, hd, pages, cols, table, rng):
        self.dt, self.kv, self.hd, self.pages, self.cols = dt, kv, hd, pages, cols
        # what nobody wrote yet is anything at all
        self.k = rng.integers(-127, 128, (pages, kv, PAGE, hd)).astype(np.int8)
        self.v = rng.integers(-127, 128, (pages, kv, hd, PAGE)).astype(np.int8)
        self.scales = np.full((pages, kv, 2), np.nan, np.float32)
        self.tk = np.full((seqs, kv, PAGE, hd), 0x7FFF, np.uint16)
        self.tv = np.full((seqs, kv, PAGE, hd), 0xFFFF, np.uint16)
        self.table = np.asarray(table, np.int32).reshape(seqs, cols)
        self.lens = np.zeros(seqs, np.int32)

    def page(self, s, b):
        p = self.table[s, b]
        return p if 0 <= p < self.pages else -1

    def base(self, s):
        return min(max(int(self.lens[s]), 0), self.cols * PAGE)

    def append(self, k, v, new):
        r = 0
        for s, n in enumerate(new):
            base = self.base(s)
            for i in range(n):
                pos = base + i
                if pos >= self.cols * PAGE:
                    break
                for tail, x in ((self.tk, k), (self.tv, v)):
                    tail[s, :, pos % PAGE] = x[r + i]
                if pos % PAGE == PAGE - 1:
                    p = self.page(s, pos // PAGE)
                    for h in range(self.kv if p >= 0 else 0):
                        for w, tail in enumerate((self.tk, self.tv)):
                            x = value(tail[s, h], self.dt)
                            d = scale_of(x)
                            self.scales[p, h, w] = d
                            c = codes_of(x, d)
                            (self.k if w == 0 else self.v)[p, h] = c if w == 0 else c.T
            r += n

    def total(self, s, n):
        return min(self.base(s) + n, self.cols * PAGE)

    def rows(self, s, n):
        """A sequence's keys and values after N new tokens, [total][kv][hd], and which are there."""
        total = self.total(s, n)
        k, v = np.zeros((total, self.kv, self.hd)), np.zeros((total, self.kv, self.hd))
        there = np.ones(total, bool)
        for b in range((total + PAGE - 1) // PAGE):
            at = slice(b * PAGE, min((b + 1) * PAGE, total))
            if (b + 1) * PAGE <= total:
                p = self.page(s, b)
                if p < 0:
                    there[at] = False
                    continue
                d = self.scales[p].astype(np.float64)
                k[at] = (self.k[p] * d[:, 0, None, None]).transpose(1, 0, 2)
                v[at] = (self.v[p] * d[:, 1, None, None]).transpose(2, 0, 1)
            else:
                m = total - b * PAGE
                k[at] = value(self.tk[s, :, :m], self.dt).transpose(1, 0, 2)
                v[at] = value(self.tv[s, :, :m], self.dt).transpose(1, 0, 2)
        return k, v, there

    def attend(self, q, new, scale, odt):
        o, tol, r = np.zeros(q.shape), np.zeros(q.shape), 0
        group = q.shape[1] // self.kv
        for s, n in enumerate(new):
            if n:
                k, v, there = self.rows(s, n)
                place = np.minimum(self.base(s) + np.arange(n), len(k) - 1)
                seen = (np.arange(len(k)) <= place[:, None]) & there
                for h in range(q.shape[1]):
                    o[r:r + n, h], tol[r:r + n, h] = attend(q[r:r + n, h], k[:, h // group], v[:, h // group], seen,
                                                            scale, self.dt, odt, True)
            r += n
        return o, tol

    def read(self, new):
        """The step's rows as the cache holds them, rounded to its type."""
        ks, vs = [], []
        for s, n in enumerate(new):
            k, v, _ = self.rows(s, n)
            pad = np.zeros((max(0, self.base(s) + n - len(k)), self.kv, self.hd))
            ks.append(np.concatenate([k, pad])[self.base(s):self.base(s) + n])
            vs.append(np.concatenate([v, pad])[self.base(s):self.base(s) + n])
        return rounded(np.concatenate(ks), self.dt), rounded(np.concatenate(vs), self.dt)

    def advance(self, new):
        for s, n in enumerate(new):
            self.lens[s] = self.total(s, n)
