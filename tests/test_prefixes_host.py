"""Plans of prefixes and rotaries without a GPU: what their entry points refuse, the plans they make, and
the frequencies.  tests/host/prefixes_host.cpp stands in for the device and the kernels (linked with this
build's own api_prompts.o, api_prefixes.o and api_rope.o)."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

import exn_hip as X

HERE = os.path.dirname(os.path.abspath(__file__))
OBJS = [os.path.join(HERE, "..", "ex-nihilo_amd", "_build", n) for n in ("api_prompts.o", "api_prefixes.o", "api_rope.o")]
vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not all(os.path.exists(o) for o in OBJS):
        pytest.skip("the library's objects are not here")
    d = tmp_path_factory.mktemp("prefixes_host")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "prefixes_host.cpp"), "-o", o], check=True)
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", "-o", so, o, *OBJS], check=True)
    lib = ctypes.CDLL(so)
    for n in ("ph_error", "ph_log"):
        getattr(lib, n).restype = ctypes.c_char_p
    lib.ph_ctx.restype = vp
    for n, (res, args) in X.SIGNATURES.items():
        if n.startswith(("exn_seqs", "exn_prefixes", "exn_attend_shared", "exn_rope")):
            f = getattr(lib, n)
            f.restype, f.argtypes = res, args
    return lib


MEM = np.zeros(4096, np.uint8)
AT = (MEM.ctypes.data + 63) // 64 * 64


def seqs(L, lens):
    h = vp()
    a = np.asarray(lens, np.int32)
    assert L.exn_seqs_create(L.ph_ctx(), a.ctypes.data_as(vp), len(a), ctypes.byref(h)) == X.OK
    return h


def prefixes(L, s, of, blocks):
    h = vp()
    o, b = np.asarray(of, np.int32), np.asarray(blocks, np.int32)
    r = L.exn_prefixes_create(L.ph_ctx(), s, o.ctypes.data_as(vp), b.ctypes.data_as(vp), len(b), ctypes.byref(h))
    return r, h


def cache(s, **over):
    f = dict(dt=X.DT_F16, kv_heads=2, head_dim=64, pages=4, seqs=s, cols=2, k=AT, v=AT, scales=AT, tk=AT, tv=AT,
             table=AT, lens=AT)
    f.update(over)
    return X.Kv8(*(f[n] for n in ("dt", "kv_heads", "head_dim", "pages", "seqs", "cols", "k", "v", "scales", "tk", "tv",
                                  "table", "lens")))


SHARED = ("ctx", "c", "s", "p", "heads", "q", "ldq", "scale", "out", "odt", "ldo", "part", "cap")


def shared(L, plan, begun, n, **over):
    c = cache(n)
    a = dict(zip(SHARED, (L.ph_ctx(), c.ref, plan, begun, 4, AT, 256, 1.0, AT, X.DT_BF16, 256, None, 0)))
    a.update(over)
    return L.exn_attend_shared(*(a[x] for x in SHARED))


@pytest.mark.parametrize("lens,of,blocks", [
    ([1, 1, 1], [0, 0, 0], [5]),
    ([3, 0, 9, 1, 40], [1, 1, 0, -1, 1], [2, 7]),
    ([4, 4], [0, 1], [3, 3]),                 # one sequence each: nothing to share
    ([4, 4], [0, 0], [0]),                    # no blocks
    ([0, 0, 5], [0, 0, 0], [9]),              # one with rows
    ([2] * 300, [i % 7 - 1 for i in range(300)], [1, 2, 3, 4, 5, 6]),
    ([5, 6], [-1, -1], []),
    ([300, 1, 70], [0, 0, 0], [1 << 20]),
])
def test_plans(L, lens, of, blocks):
    """Each shared prefix's rows, once, by sequences; every list's tiles cover them once."""
    s = seqs(L, lens)
    r, p = prefixes(L, s, of, blocks)
    assert r == X.OK
    assert shared(L, s, p, len(lens)) == X.OK and L.ph_log() == b"shared "
    out = np.zeros(1 << 16, np.int32)
    count, groups = len(lens), len(blocks)
    n = L.ph_shared(out.ctypes.data_as(vp), count)
    rows, most, top = out[:3].tolist()
    who = {g: [i for i in range(count) if of[i] == g and lens[i]] for g in range(groups)}
    live = [g for g in who if len(who[g]) > 1 and blocks[g] > 0]
    size = {g: sum(lens[i] for i in who[g]) for g in live}
    assert rows == sum(size.values()) and most == max(size.values(), default=0)
    assert top == max((blocks[g] for g in live), default=0)
    mine = out[3:3 + 4 * count].reshape(-1, 4).tolist()
    entry = out[3 + 4 * count:3 + 4 * count + 2 * rows].reshape(-1, 2).tolist()
    starts = np.concatenate([[0], np.cumsum(lens)])
    first = dict(zip(live, np.concatenate([[0], np.cumsum([size[g] for g in live])])))
    for i in range(count):
        if of[i] not in live:
            assert mine[i][0] == -1
            continue
        assert mine[i][:2] == [who[of[i]][0], blocks[of[i]]]
        for k in range(lens[i]):
            assert entry[mine[i][2] + k] == [starts[i] + k, i]
    assert sorted(e[0] for e in entry) == sorted(int(starts[i]) + k for g in live for i in who[g] for k in range(lens[i]))
    rest = out[3 + 4 * count + 2 * rows:n].reshape(-1, 5)
    heads = np.flatnonzero(rest[:, 0] == -1)
    assert list(rest[heads, 1]) == [8, 16, 32, 64, 128]
    for a, b in zip(heads, [*heads[1:], len(rest)]):
        tt = int(rest[a, 1])
        want = [(int(first[g]), size[g], t0, who[g][0], blocks[g]) for g in live for t0 in range(0, size[g], tt)]
        assert list(map(tuple, rest[a + 1:b].tolist())) == want
    assert L.exn_prefixes_free(p) == X.OK and L.exn_seqs_free(s) == X.OK


def test_plan_refusals(L):
    s = seqs(L, [5, 6])
    for of, blocks in (([0, 1], [3]), ([0, -2], [3]), ([0, 0], [-1]), ([0, 0], [(1 << 20) + 1]), ([0, 0], [1, 1, 1])):
        r, p = prefixes(L, s, of, blocks)
        assert r == X.EINVAL and not p.value and b"prefix" in L.ph_error(), (of, blocks)
    ctx, a = L.ph_ctx(), np.zeros(2, np.int32).ctypes.data_as(vp)
    assert L.exn_prefixes_create(None, s, a, a, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_prefixes_create(ctx, None, a, a, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_prefixes_create(ctx, s, None, a, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_prefixes_create(ctx, s, a, None, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_prefixes_create(ctx, s, a, a, -1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_prefixes_create(ctx, s, a, a, 1, None) == X.EINVAL
    L.ph_capturing(1)
    assert prefixes(L, s, [0, 0], [1])[0] == X.ESTATE and b"capture" in L.ph_error()
    L.ph_capturing(0)
    L.ph_no_memory(1)
    assert prefixes(L, s, [0, 0], [1])[0] == X.ENOMEM
    L.ph_no_memory(0)
    L.ph_device(1)
    assert prefixes(L, s, [0, 0], [1])[0] == X.EINVAL and b"device" in L.ph_error()
    L.ph_device(0)
    assert L.exn_prefixes_free(None) == X.OK
    L.exn_seqs_free(s)


def test_call_refusals(L):
    s, other = seqs(L, [5, 6]), seqs(L, [5, 6])
    _, p = prefixes(L, s, [0, 0], [1])
    n = ctypes.c_int64()
    assert shared(L, s, p, 2) == X.OK and shared(L, s, p, 2, part=AT, cap=8) == X.OK and L.ph_log()
    bad = [dict(ctx=None), dict(c=None), dict(s=None), dict(p=None), dict(s=other), dict(heads=3), dict(heads=0),
           dict(heads=1026), dict(q=None), dict(q=AT + 4), dict(ldq=248), dict(ldq=257), dict(out=None), dict(out=AT + 8),
           dict(ldo=260), dict(odt=X.DT_F32), dict(cap=4), dict(cap=-1), dict(part=AT + 4, cap=8)]
    for b in bad:
        assert shared(L, s, p, 2, **b) == X.EINVAL, b
        assert L.ph_error() and not L.ph_log(), b
    for k in (1, 3):
        assert shared(L, s, p, k) == X.EINVAL and b"plan" in L.ph_error()
    for over in (dict(dt=X.DT_F32), dict(head_dim=72), dict(pages=0), dict(cols=0), dict(k=None), dict(lens=None)):
        c = cache(2, **over)
        assert shared(L, s, p, 2, c=c.ref) == X.EINVAL, over
    L.ph_device(1)
    assert shared(L, s, p, 2) == X.EINVAL and b"device" in L.ph_error()
    L.ph_device(0)
    assert L.exn_attend_shared_part(s, p, 4, 2, 64, 2, ctypes.byref(n)) == X.OK and n.value == 34
    for a in ((None, p, 4, 2, 64, 2), (s, None, 4, 2, 64, 2), (other, p, 4, 2, 64, 2), (s, p, 3, 2, 64, 2),
              (s, p, 4, 2, 72, 2), (s, p, 4, 2, 64, 0)):
        assert L.exn_attend_shared_part(*a, ctypes.byref(n)) == X.EINVAL, a
    assert L.exn_attend_shared_part(s, p, 4, 2, 64, 2, None) == X.EINVAL
    empty = seqs(L, [0, 0])
    _, q = prefixes(L, empty, [0, 0], [4])
    assert L.exn_attend_shared_part(empty, q, 4, 2, 64, 2, ctypes.byref(n)) == X.OK and n.value == 0
    for h in (p, q):
        L.exn_prefixes_free(h)
    for h in (s, other, empty):
        L.exn_seqs_free(h)


# --- rotaries -----------------------------------------------------------------------------------


def plain(dims, base):
    return [float(base) ** (-2 * j / dims) for j in range(dims // 2)]


@pytest.mark.parametrize("dims,base", [(2, 1e4), (32, 1e4), (128, 5e6), (256, 1e6), (10, 0.5)])
def test_frequencies(dims, base):
    f = plain(dims, base)
    # each value is a power and at most three more operations in 64 bits: some units in the last place
    assert np.allclose(X.rope_freqs(dims, base), f, rtol=1e-14, atol=0)
    assert np.allclose(X.rope_freqs(dims, base, X.ROPE_LINEAR, 4.0), [x / 4 for x in f], rtol=1e-14, atol=0)
    if dims > 2:
        assert np.allclose(X.rope_freqs(dims, base, X.ROPE_BASE, 4.0), plain(dims, base * 4.0 ** (dims / (dims - 2))),
                           rtol=1e-13, atol=0)
        # the slowest pair is slowed by the factor, the fastest is not
        g = X.rope_freqs(dims, base, X.ROPE_BASE, 4.0)
        assert g[0] == 1 and np.isclose(g[-1], f[-1] / 4, rtol=1e-13)


@pytest.mark.parametrize("kept,low,high", [(8192, 1, 4), (32768, 1, 32), (100, 0.5, 2)])
def test_blended_frequencies(kept, low, high):
    dims, base, factor = 128, 5e5, 8.0
    f = plain(dims, base)
    got = X.rope_freqs(dims, base, X.ROPE_TURNS, factor, kept, low, high)
    for x, y in zip(f, got):
        turns = kept * x / math.tau
        r = 0 if turns < low else 1 if turns > high else (turns - low) / (high - low)
        assert math.isclose(y, r * x + (1 - r) * x / factor, rel_tol=1e-13)
    got = X.rope_freqs(dims, base, X.ROPE_INDEX, factor, kept, low, high)
    # the pair that turns n times: base^(-2 i / dims) kept = 2 pi n
    at = [dims / 2 * math.log(kept / (math.tau * n), base) for n in (high, low)]
    a, b = max(0, math.floor(at[0])), min(dims - 1, math.ceil(at[1]))
    for j, (x, y) in enumerate(zip(f, got)):
        g = min(1, max(0, (j - a) / (b - a)))
        assert math.isclose(y, (1 - g) * x + g * x / factor, rel_tol=1e-13)
    assert (np.diff(got) < 0).all()


def test_frequencies_of_a_step(L):
    """Both ends of the ramp at the same pair: all divided but the first."""
    f = plain(8, 1e4)
    got = X.rope_freqs(8, 1e4, X.ROPE_INDEX, 2.0, 1.0, 0.5, 0.6)
    assert np.allclose(got, [f[0], *(x / 2 for x in f[1:])], rtol=1e-13)


def test_frequencies_with_the_ramp_past_an_end(L):
    """Every pair turns more than HIGH times, or fewer than LOW: all as they are, or all but the first divided."""
    f = plain(64, 10.0)
    assert np.allclose(X.rope_freqs(64, 10.0, X.ROPE_INDEX, 4.0, 1e6, 1.0, 32.0), f, rtol=1e-13)
    assert np.allclose(X.rope_freqs(64, 10.0, X.ROPE_INDEX, 4.0, 1e-3, 1.0, 32.0), [f[0], *(x / 4 for x in f[1:])], rtol=1e-13)


def test_frequency_refusals(L):
    f = np.zeros(128)
    p = f.ctypes.data_as(vp)
    good = (128, 1e4, X.ROPE_INDEX, 4.0, 8192.0, 1.0, 32.0)
    assert L.exn_rope_freqs(*good, p) == X.OK
    for i, v in ((0, 0), (0, 3), (0, 258), (0, -2), (1, 0.0), (1, -1.0), (1, math.inf), (1, math.nan), (1, 1.0), (2, -1),
                 (2, 5), (3, 0.0), (3, math.nan), (4, 0.0), (4, math.inf), (5, 0.0), (5, math.nan), (6, 1.0), (6, 0.5)):
        a = list(good)
        a[i] = v
        assert L.exn_rope_freqs(*a, p) == X.EINVAL, (i, v)
    assert L.exn_rope_freqs(2, 1e4, X.ROPE_BASE, 4.0, 1.0, 0.0, 1.0, p) == X.EINVAL
    assert L.exn_rope_freqs(*good, None) == X.EINVAL
    # what a scaling does not use is not looked at
    assert L.exn_rope_freqs(128, 1e4, X.ROPE_PLAIN, math.nan, math.nan, math.nan, math.nan, p) == X.OK
    assert L.exn_rope_freqs(128, 1e4, X.ROPE_LINEAR, 2.0, math.nan, math.nan, math.nan, p) == X.OK


def rope(L, freq, layout=0, axis=None, axes=1, amp=1.0):
    f = np.asarray(freq, np.float64)
    a = None if axis is None else np.asarray(axis, np.int32).ctypes.data_as(vp)
    h = vp()
    return L.exn_rope_create(L.ph_ctx(), f.ctypes.data_as(vp), len(f), layout, a, axes, amp, ctypes.byref(h)), h


ROWS = ("ctx", "r", "s", "pos", "lens", "hd", "dt", "odt", "eps", "heads", "q", "ldq", "wq", "qo", "ldqo", "kv", "k", "ldk",
        "wk", "ko", "ldko")


def rows(L, r, s, **over):
    a = dict(zip(ROWS, (L.ph_ctx(), r, s, None, AT, 64, X.DT_F16, X.DT_F16, 1e-6, 4, AT, 256, AT, AT + 1024, 256, 2, AT, 128,
                        AT, AT + 1024, 128)))
    a.update(over)
    return L.exn_rope_rows(*(a[x] for x in ROWS))


def test_turns(L):
    """A frequency is held as its exact fraction of a turn, to a unit of 2^-64."""
    s = seqs(L, [5])
    freq = [1.0, 0.1, 2.0 ** -30, 1e-7, 0.0, -0.25, 6.5, 1024.0, 6.283185307179586, 5e-324]
    r, h = rope(L, freq, X.ROPE_PAIRS, [0, 1, 2, 0, 1, 2, 0, 1, 2, 0], 3)
    assert r == X.OK and rows(L, h, s, lens=None, pos=AT) == X.OK and L.ph_log() == b"rope "
    turns, axis = np.zeros(16, np.uint64), np.zeros(16, np.int32)
    n = L.ph_rope(turns.ctypes.data_as(vp), axis.ctypes.data_as(vp))
    assert n == 10 and axis[:10].tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 2, 0]
    # 2 pi to 35 places
    tau = Fraction(628318530717958647692528676655900576, 10 ** 35)
    for f, t in zip(freq, turns.tolist()):
        want = Fraction(f) / tau
        want -= math.floor(want)
        miss = abs(Fraction(t, 2 ** 64) - want)
        # an 80-bit quotient of an 80-bit 2 pi: 2^-63 of the whole value, and half a unit
        assert min(miss, 1 - miss) <= Fraction(1, 2 ** 64) + abs(Fraction(f)) / tau / 2 ** 62, f
    L.exn_rope_free(h)
    L.exn_seqs_free(s)


def test_rotary_refusals(L):
    for kw in (dict(freq=[]), dict(freq=[0.1] * 129), dict(freq=[math.nan]), dict(freq=[math.inf]), dict(freq=[1025.0]),
               dict(layout=2), dict(layout=-1), dict(axes=0), dict(axes=9), dict(axis=[1]), dict(axis=[-1]),
               dict(axis=[3], axes=3), dict(amp=math.nan), dict(amp=math.inf)):
        r, h = rope(L, **dict(dict(freq=[0.5]), **kw))
        assert r == X.EINVAL and not h.value and b"rotary" in L.ph_error(), kw
    f = np.ones(2).ctypes.data_as(vp)
    assert L.exn_rope_create(None, f, 2, 0, None, 1, 1.0, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_rope_create(L.ph_ctx(), None, 2, 0, None, 1, 1.0, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_rope_create(L.ph_ctx(), f, 2, 0, None, 1, 1.0, None) == X.EINVAL
    L.ph_capturing(1)
    assert rope(L, [0.5])[0] == X.ESTATE
    L.ph_capturing(0)
    L.ph_no_memory(1)
    assert rope(L, [0.5])[0] == X.ENOMEM
    L.ph_no_memory(0)
    assert L.exn_rope_free(None) == X.OK


def test_row_refusals(L):
    s = seqs(L, [5, 6])
    _, r = rope(L, [0.5] * 32)
    _, three = rope(L, [0.5] * 3, axis=[0, 1, 2], axes=3)
    assert rows(L, r, s) == X.OK and rows(L, r, s, lens=None) == X.OK and rows(L, r, s, lens=None, pos=AT) == X.OK
    assert rows(L, r, s, wq=None, wk=None) == X.OK
    assert rows(L, r, s, kv=0, k=None, ldk=0, ko=None, ldko=0) == X.OK
    assert rows(L, r, s, qo=AT, ko=AT) == X.OK                       # in place
    assert rows(L, r, s, dt=X.DT_F32, odt=X.DT_BF16) == X.OK
    assert rows(L, three, s, lens=None, pos=AT) == X.OK
    assert L.ph_log() == b"rope " * 8
    bad = [dict(ctx=None), dict(r=None), dict(s=None), dict(pos=AT), dict(hd=60), dict(hd=56), dict(hd=264), dict(hd=0),
           dict(dt=3), dict(odt=-1), dict(eps=-1e-6), dict(eps=math.nan), dict(eps=math.inf), dict(heads=0), dict(heads=1025),
           dict(kv=-1), dict(kv=1025), dict(q=None), dict(q=AT + 8), dict(ldq=248), dict(ldq=260), dict(ldq=1 << 25),
           dict(wq=AT + 4), dict(qo=None), dict(qo=AT + 8), dict(ldqo=128), dict(k=None), dict(k=AT + 2), dict(ldk=120),
           dict(wk=AT + 8), dict(ko=None), dict(ldko=129), dict(qo=AT, odt=X.DT_BF16), dict(qo=AT, ldqo=264),
           dict(ko=AT, ldko=136), dict(lens=AT + 2), dict(lens=None, pos=AT + 1), dict(r=three, lens=None), dict(r=three)]
    for b in bad:
        a = dict(r=r, s=s)
        a.update(b)
        r2, s2 = a.pop("r"), a.pop("s")
        assert rows(L, r2, s2, **a) == X.EINVAL, b
        assert L.ph_error() and not L.ph_log(), b
    L.ph_device(1)
    assert rows(L, r, s) == X.EINVAL and b"device" in L.ph_error()
    L.ph_device(0)
    for h in (r, three):
        L.exn_rope_free(h)
    L.exn_seqs_free(s)
