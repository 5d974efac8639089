"""The prompt side's attention without a GPU: what its entry points refuse, the plans they make, and
the cache's rules for places, pages, scales and codes.  tests/host/prompts_host.cpp stands in for
the device and the kernels (linked with this build's own api_prompts.o)."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

import exn_hip as X
import prompts_model as pm

HERE = os.path.dirname(os.path.abspath(__file__))
OBJ = os.path.join(HERE, "..", "ex-nihilo_amd", "_build", "api_prompts.o")
vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not os.path.exists(OBJ):
        pytest.skip("the library's objects are not here")
    d = tmp_path_factory.mktemp("prompts_host")
    o, so = str(d / "prompts_host.o"), str(d / "prompts_host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "prompts_host.cpp"), "-o", o], check=True)
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", "-o", so, o, OBJ], check=True)
    lib = ctypes.CDLL(so)
    for n in ("ph_error", "ph_log"):
        getattr(lib, n).restype = ctypes.c_char_p
    lib.ph_ctx.restype = vp
    lib.ph_block.restype = ctypes.c_float
    for n, (res, args) in X.SIGNATURES.items():
        if n.startswith(("exn_seqs", "exn_attend_packed", "exn_kv8")):
            f = getattr(lib, n)
            f.restype, f.argtypes = res, args
    return lib


def seqs(L, lens):
    h = vp()
    a = np.asarray(lens, np.int32)
    r = L.exn_seqs_create(L.ph_ctx(), a.ctypes.data_as(vp), len(a), ctypes.byref(h))
    return r, h


MEM = np.zeros(4096, np.uint8)
AT = (MEM.ctypes.data + 63) // 64 * 64


def cache(s, **over):
    f = dict(dt=X.DT_F16, kv_heads=2, head_dim=64, pages=4, seqs=s, cols=2, k=AT, v=AT, scales=AT, tk=AT, tv=AT,
             table=AT, lens=AT)
    f.update(over)
    return X.Kv8(*(f[n] for n in ("dt", "kv_heads", "head_dim", "pages", "seqs", "cols", "k", "v", "scales", "tk", "tv",
                                  "table", "lens")))


def test_plans(L):
    """Every list covers each sequence's tokens once, the latest (costliest) tiles first."""
    for lens in ([1], [0], [0, 300, 7, 0, 64], [129, 1000, 5, 5], [8] * 70):
        r, h = seqs(L, lens)
        assert r == X.OK
        assert L.exn_attend_packed(L.ph_ctx(), h, X.DT_F16, 4, 2, 64, AT, 256, AT, 128, AT, 128, 1.0, AT, X.DT_BF16,
                                   256) == X.OK
        assert L.ph_log() == b"packed "
        out = np.zeros((4096, 4), np.int32)
        n = L.ph_tiles(out.ctypes.data_as(vp), 4096)
        out = out[:n]
        starts = np.concatenate([[0], np.cumsum(lens)])
        heads = np.flatnonzero(out[:, 0] == -1)
        assert list(out[heads, 1]) == [8, 16, 32, 64, 128]
        for a, b in zip(heads, [*heads[1:], n]):
            tt, t = out[a, 1], out[a + 1:b]
            want = sorted((int(starts[i]), m, t0, i) for i, m in enumerate(lens) for t0 in range(0, m, tt))
            assert sorted(map(tuple, t.tolist())) == want
            assert (np.diff(t[:, 2]) <= 0).all()
        a, b, c = ctypes.c_int(), ctypes.c_int64(), ctypes.c_int()
        assert L.exn_seqs_info(h, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c)) == X.OK
        assert (a.value, b.value, c.value) == (len(lens), sum(lens), max(lens))
        assert L.exn_seqs_free(h) == X.OK


def test_plan_refusals(L):
    for lens in ([-1], [3, -2], [1 << 22, 1], [1] * 65537, []):
        r, h = seqs(L, lens)
        assert r == X.EINVAL and not h.value, len(lens)
        assert b"sequences" in L.ph_error()
    assert L.exn_seqs_create(L.ph_ctx(), None, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_seqs_create(L.ph_ctx(), AT, 1, None) == X.EINVAL
    assert L.exn_seqs_create(None, AT, 1, ctypes.byref(vp())) == X.EINVAL
    assert L.exn_seqs_info(None, None, None, None) == X.EINVAL
    assert L.exn_seqs_free(None) == X.OK
    L.ph_capturing(1)
    r, h = seqs(L, [1])
    L.ph_capturing(0)
    assert r == X.ESTATE and b"capture" in L.ph_error()


PACKED = ("ctx", "s", "dt", "heads", "kv", "hd", "q", "ldq", "k", "ldk", "v", "ldv", "scale", "out", "odt", "ldo")


def test_packed_refusals(L):
    r, h = seqs(L, [5, 6])
    good = dict(zip(PACKED, (L.ph_ctx(), h, X.DT_F16, 4, 2, 64, AT, 256, AT, 128, AT, 128, 1.0, AT, X.DT_BF16, 256)))

    def call(**over):
        a = dict(good, **over)
        return L.exn_attend_packed(*(a[n] for n in PACKED))

    assert call() == X.OK and L.ph_log() == b"packed "
    bad = [dict(ctx=None), dict(s=None), dict(dt=X.DT_F32), dict(odt=X.DT_F32), dict(heads=5), dict(heads=0), dict(kv=0),
           dict(heads=1, kv=2), dict(heads=1026), dict(hd=72), dict(hd=256), dict(q=None), dict(k=None), dict(v=None),
           dict(out=None), dict(q=AT + 2), dict(v=AT + 8), dict(out=AT + 8), dict(ldq=248), dict(ldk=132), dict(ldv=120),
           dict(ldo=260), dict(ldk=1 << 25)]
    for b in bad:
        assert call(**b) == X.EINVAL, b
        assert L.ph_error() and not L.ph_log(), b
    L.ph_device(1)
    assert call() == X.EINVAL and b"device" in L.ph_error()
    L.ph_device(0)
    L.exn_seqs_free(h)


def test_cache_refusals(L):
    r, h = seqs(L, [5, 6])
    ctx = L.ph_ctx()

    def calls(c, ctx=ctx, h=h, k=AT, ld=128, heads=4, q=AT, part=None, cap=0, odt=X.DT_BF16):
        p = c.ref if c is not None else None
        return [L.exn_kv8_append(ctx, p, h, k, ld, AT, 128), L.exn_kv8_read(ctx, p, h, AT, 128, k, ld),
                L.exn_kv8_advance(ctx, p, h),
                L.exn_kv8_attend(ctx, p, h, heads, q, 256, 1.0, AT, odt, 256, part, cap)]

    assert calls(cache(2)) == [X.OK] * 4 and L.ph_log() == b"append read advance attend "
    for over in (dict(dt=X.DT_F32), dict(kv_heads=0), dict(head_dim=72), dict(pages=0), dict(cols=0),
                 dict(cols=(1 << 20) + 1), dict(pages=1 << 31), dict(k=None), dict(v=None), dict(scales=None), dict(tk=None),
                 dict(tv=None), dict(table=None), dict(lens=None), dict(k=AT + 4), dict(v=AT + 8), dict(tk=AT + 2),
                 dict(scales=AT + 4), dict(table=AT + 1), dict(lens=AT + 2)):
        assert calls(cache(2, **over)) == [X.EINVAL] * 4, over
    for s in (1, 3):
        assert calls(cache(s)) == [X.EINVAL] * 4 and b"plan" in L.ph_error()
    assert calls(None) == [X.EINVAL] * 4
    assert calls(cache(2), ctx=None) == [X.EINVAL] * 4 and b"context" in L.ph_error()
    assert calls(cache(2), h=None) == [X.EINVAL] * 4
    L.ph_device(1)
    assert calls(cache(2)) == [X.EINVAL] * 4 and b"device" in L.ph_error()
    L.ph_device(0)
    assert not L.ph_log()
    for over in (dict(k=None), dict(k=AT + 2), dict(ld=120), dict(ld=129)):
        assert calls(cache(2), **over)[:2] == [X.EINVAL] * 2, over
    for over in (dict(heads=3), dict(heads=0), dict(q=None), dict(q=AT + 4), dict(odt=X.DT_F32), dict(cap=4),
                 dict(cap=-1), dict(part=AT + 4, cap=8)):
        assert calls(cache(2), **over)[3] == X.EINVAL, over
    n = ctypes.c_int64()
    assert L.exn_kv8_attend_part(h, 4, 2, 64, 2, ctypes.byref(n)) == X.OK and n.value == 12
    for a in ((None, 4, 2, 64, 2), (h, 3, 2, 64, 2), (h, 4, 2, 72, 2), (h, 4, 2, 64, 0)):
        assert L.exn_kv8_attend_part(*a, ctypes.byref(n)) == X.EINVAL
    assert L.exn_kv8_attend_part(h, 4, 2, 64, 2, None) == X.EINVAL
    L.exn_seqs_free(h)


def test_places_and_pages(L):
    """Lengths and pages that are none: never past the table, never outside the pages."""
    table = np.array([[0, 6, -1], [7, 1 << 30, -(1 << 31)]], np.int32)
    for lens, base in ((-5, 0), (-(1 << 31), 0), (0, 0), (100, 100), (192, 192), (193, 192), ((1 << 31) - 1, 192)):
        ln = np.array([1, lens], np.int32)
        for n in (0, 1, 91, 92, 93, 1 << 22):
            for block, page in ((0, -1), (1, -1), (2, -1)):
                b, t, p = ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()
                L.ph_place(table.ctypes.data_as(vp), ln.ctypes.data_as(vp), 3, ctypes.c_int64(7), 1, n, block,
                           ctypes.byref(b), ctypes.byref(t), ctypes.byref(p))
                assert (b.value, t.value, p.value) == (base, min(base + n, 192), page)
    b, t, p = ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()
    L.ph_place(table.ctypes.data_as(vp), np.array([1, 1], np.int32).ctypes.data_as(vp), 3, ctypes.c_int64(7), 0, 1, 1,
               ctypes.byref(b), ctypes.byref(t), ctypes.byref(p))
    assert p.value == 6


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_scales_and_codes(L, dt):
    """Codes are x / scale rounded to nearest even of the exact quotient, none over 127; the scale
    has 12 significant bits; code x scale is exact in fp32."""
    rng = np.random.default_rng(3)
    for i in range(300):
        spread = 2.0 ** rng.integers(-20, 12)
        x = pm.rounded((spread * rng.standard_normal(64)).astype(np.float32), dt).astype(np.float32)
        if i % 3 == 0:        # values on and next to a tie
            d = pm.scale_of(x)
            x[1:] = pm.rounded(((rng.integers(-126, 126, 63) + 0.5) * np.float64(d)).astype(np.float32), dt)
        codes = np.zeros(64, np.int8)
        d = L.ph_block(x.ctypes.data_as(vp), 64, codes.ctypes.data_as(vp))
        assert np.float32(d) == pm.scale_of(x)
        assert Fraction(d).numerator.bit_length() <= 12 and abs(x).max() / d <= 127
        want = [round(Fraction(float(v)) / Fraction(d)) for v in x]       # round(): to even
        assert list(codes) == want and max(map(abs, want)) <= 127
        assert (np.float64(d) * codes == (np.float32(d) * codes.astype(np.float32)).astype(np.float64)).all()
    for x, codes in ((np.zeros(4), [0] * 4), ([np.nan, 1, 2, 3], None), ([1, -np.inf, 2, 3], None)):
        x, c = np.asarray(x, np.float32), np.ones(4, np.int8)
        d = L.ph_block(x.ctypes.data_as(vp), 4, c.ctypes.data_as(vp))
        assert (math.isnan(d) if codes is None else d == 0) and not c.any()
    # the smallest and the largest values
    for top in (2.0 ** -24, 6e-8, 65504.0) if dt == "fp16" else (2.0 ** -133, 1e-38, 3.38e38):
        x = pm.rounded(np.array([top, -top, top / 2, 0], np.float32), dt).astype(np.float32)
        c = np.zeros(4, np.int8)
        d = L.ph_block(x.ctypes.data_as(vp), 4, c.ctypes.data_as(vp))
        assert np.isfinite(d) and abs(c[0]) <= 127
        assert abs(float(x[0]) - float(d) * c[0]) <= max(abs(float(x[0])) * 2.0 ** -8, 2.0 ** -138)


def test_steps_of_too_many_tokens_are_refused(L):
    for n, ok in ((1 << 21, True), ((1 << 21) + 1, False)):
        r, h = seqs(L, [5, n])
        assert r == X.OK
        c = cache(2)
        for f in (L.exn_kv8_append, L.exn_kv8_read):
            assert f(L.ph_ctx(), ctypes.byref(c), h, AT, 128, AT, 128) == (X.OK if ok else X.EINVAL)
        L.exn_seqs_free(h)
