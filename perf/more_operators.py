"""Further operators of the prompt side in exn_hip, as cases that can be timed and compared.

rope_rows: rows of queries and keys as an attention takes them, each head RMS-normed (or not) and turned
by its position, in one pass: both layouts of the pairs, all of a head or its first dims, positions on one
or several axes or counted on from a cache's lengths, frequencies as they are or scaled for long contexts.

attend_shared: attention over the cache in 8 bits of sequences that begin alike, on the same pages:
what kv8_attend answers, with the keys and values of a common beginning read once for all of them.

The cache, as the library lays it out: a page is a block of 64 tokens; codes of keys
[page][kv head][64][dim] and of values [page][kv head][dim][64], scales [page][kv head][2] (key,
value); a sequence's last block, while it is not full, in 16 bits, tails [sequence][kv head][64][dim];
table [sequence][column] names the pages, lens the tokens before the step.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE = 64
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the next token of a few short texts, positions from the cache's lengths: latency alone
        {"name": "rope 4 tokens over 300", "kind": "rope", "seqs": 4, "longest": 1, "shortest": 1, "far": 333, "heads": 32,
         "kv_heads": 8, "dim": 128, "pairs": 64, "layout": "half", "axes": 1, "norm": True, "scaling": "plain",
         "dt": "fp16", "odt": "fp16"},
        # a server's batch of prompts, some with a picture's rows: positions (frame, row, column)
        {"name": "rope 16 prompts 21..257", "kind": "rope", "seqs": 16, "longest": 257, "shortest": 21, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64, "layout": "pairs", "axes": 3, "norm": True,
         "scaling": "plain", "dt": "fp16", "odt": "fp16"},
        # edit prompts from a product's fp32 rows
        {"name": "rope 4 edit prompts 1100..1180, fp32", "kind": "rope", "seqs": 4, "longest": 1180, "shortest": 1100,
         "far": 0, "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64, "layout": "half", "axes": 3, "norm": True,
         "scaling": "plain", "dt": "fp32", "odt": "fp16"},
        # chunks of long texts of a smaller model, far on in them: narrow heads, half of each turned, scaled
        {"name": "rope chunks 512 at 131071, 64-wide", "kind": "rope", "seqs": 4, "longest": 512, "shortest": 301,
         "far": 131071, "heads": 16, "kv_heads": 2, "dim": 64, "pairs": 16, "layout": "half", "axes": 1, "norm": False,
         "scaling": "turns", "dt": "bf16", "odt": "bf16"},
        # long documents: the memory's rate
        {"name": "rope 2 documents 8192", "kind": "rope", "seqs": 2, "longest": 8192, "shortest": 8192, "far": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "pairs": 64, "layout": "half", "axes": 1, "norm": True,
         "scaling": "index", "dt": "bf16", "odt": "bf16"},
        # the next token of a few texts after one short template: latency
        {"name": "shared 4 tokens after 320", "kind": "shared", "seqs": 4, "alone": 0, "prefixes": 1, "shared": 320,
         "shared_least": 320, "longest": 60, "shortest": 5, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128, "dt": "fp16",
         "odt": "bf16"},
        # the next token of descriptions after a template and a picture
        {"name": "shared 16 tokens after 1088", "kind": "shared", "seqs": 16, "alone": 0, "prefixes": 1, "shared": 1088,
         "shared_least": 1088, "longest": 200, "shortest": 12, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dt": "fp16", "odt": "bf16"},
        # a full batch's next tokens after one long document: the document's products, the rest's bytes
        {"name": "shared 64 tokens after 8192", "kind": "shared", "seqs": 64, "alone": 0, "prefixes": 1, "shared": 8192,
         "shared_least": 8192, "longest": 2000, "shortest": 60, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dt": "bf16", "odt": "bf16"},
        # several instructions for one picture
        {"name": "shared 8 instructions 76 after 1088", "kind": "shared", "seqs": 8, "alone": 0, "prefixes": 1,
         "shared": 1088, "shared_least": 1088, "longest": 76, "shortest": 76, "new": 76, "heads": 32, "kv_heads": 8,
         "dim": 128, "dt": "fp16", "odt": "bf16"},
        # three documents' readers and some texts of their own, a smaller model's narrow heads
        {"name": "shared 30 tokens, 3 prefixes 4032, 64-wide", "kind": "shared", "seqs": 30, "alone": 6, "prefixes": 3,
         "shared": 4032, "shared_least": 1024, "longest": 901, "shortest": 33, "new": 1, "heads": 16, "kv_heads": 2,
         "dim": 64, "dt": "bf16", "odt": "bf16"},
        # a few questions about one very long text
        {"name": "shared 8 tokens after 131008", "kind": "shared", "seqs": 8, "alone": 0, "prefixes": 1, "shared": 131008,
         "shared_least": 131008, "longest": 900, "shortest": 100, "new": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "dt": "fp16", "odt": "fp16"},
        # chunks of many texts after one beginning, narrow heads: the products' rate
        {"name": "shared 16 chunks 256 after 4096, 64-wide", "kind": "shared", "seqs": 16, "alone": 0, "prefixes": 1,
         "shared": 4096, "shared_least": 4096, "longest": 500, "shortest": 256, "new": 256, "heads": 16, "kv_heads": 2,
         "dim": 64, "dt": "bf16", "odt": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rope", "shared"))
    kv, group = rng.choice(((8, 4), (8, 4), (2, 8), (8, 1), (4, 3), (1, 16), (4, 2)))
    c = {"kind": kind, "seqs": _log(rng, 1, 64), "heads": kv * group, "kv_heads": kv, "dim": rng.choice((64, 128, 128))}
    if kind == "rope":
        if rng.random() < 0.3:
            c["dim"] = rng.choice((32, 72, 80, 96, 192, 256))
        c["pairs"] = c["dim"] // 2 if rng.random() < 0.5 else rng.randint(1, c["dim"] // 2)
        c["layout"], c["norm"] = rng.choice(("half", "pairs")), rng.random() < 0.6
        c["axes"] = rng.choice((1, 1, 3))
        c["scaling"] = rng.choice(("plain", "linear", "base", "turns", "index")) if c["pairs"] > 1 else "plain"
        c["dt"], c["odt"] = rng.choice(("fp16", "bf16", "fp32")), rng.choice(("fp16", "bf16", "fp16", "bf16", "fp32"))
        c["longest"] = 1 if rng.random() < 0.3 else _log(rng, 1, 8192)
        c["shortest"] = _log(rng, 1, c["longest"])
        # positions counted on from a cache's lengths up to this one, or (0) given
        c["far"] = 0 if c["axes"] > 1 or rng.random() < 0.3 else _log(rng, 1, 131072)
        while sum(_lens(c)) * (c["heads"] + kv) * c["dim"] * (_size(c["dt"]) + _size(c["odt"])) > 16384 * 40 * 128 * 4:
            c["longest"] = max(1, c["longest"] * 3 // 4)
            c["shortest"] = min(c["shortest"], c["longest"])
        return c
    c["dt"], c["odt"] = rng.choice(("fp16", "bf16")), rng.choice(("fp16", "bf16"))
    c["seqs"] = _log(rng, 2, 64)
    c["prefixes"] = rng.choice((1, 1, 1, 2, 3)) if c["seqs"] > 6 else 1
    c["alone"] = rng.randint(0, c["seqs"] // 4) if rng.random() < 0.3 else 0
    c["new"] = 1 if rng.random() < 0.6 else _log(rng, 1, 256)
    c["shared"] = PAGE * _log(rng, 1, 2048)
    c["shared_least"] = c["shared"] if rng.random() < 0.5 else PAGE * _log(rng, 1, c["shared"] // PAGE)
    c["longest"] = max(c["new"], _log(rng, 1, 4096))
    c["shortest"] = max(c["new"], _log(rng, max(1, c["longest"] // 16), c["longest"]))
    # no more pairs than the listed chunks have, in the plain form's padded scores, and no more bytes than the longest text
    while _padded(c) > 16 * 256 * 16 * (4096 + 256) * 64:
        if c["shared"] > 4096 and c["shared"] > 4 * c["longest"]:
            c["shared"] = PAGE * (c["shared"] // PAGE // 2)
        elif c["new"] > 1 and c["new"] >= c["seqs"]:
            c["new"] //= 2
        else:
            c["seqs"] = max(2, c["seqs"] // 2)
            c["longest"] = max(c["new"], c["longest"] // 2)
            c["alone"], c["prefixes"] = min(c["alone"], c["seqs"] // 4), 1
        c["shared_least"] = min(c["shared"], c["shared_least"])
        c["shortest"] = max(c["new"], min(c["shortest"], c["longest"]))
    while c["kv_heads"] * c["dim"] * (c["prefixes"] * c["shared"] + c["seqs"] * c["longest"]) > 8 * 128 * 131072:
        c["shared"] = max(PAGE, PAGE * (c["shared"] // PAGE // 2))
        c["shared_least"] = min(c["shared"], c["shared_least"])
        c["longest"] = max(c["new"], c["longest"] // 2)
        c["shortest"] = max(c["new"], min(c["shortest"], c["longest"]))
    return c


def _size(t):
    return 4 if t == "fp32" else 2


def _padded(c):
    return c["seqs"] * c["new"] * c["heads"] * (c["shared"] + c["longest"] + 2 * PAGE) * c["dim"]


def _run(n, a, b):
    """A geometric run of n whole numbers from a to b, in a mixed order."""
    run = [int(round(a * (b / a) ** (i / (n - 1)))) if n > 1 and a else a for i in range(n)]
    return [run[i * 7919 % n] for i in range(n)]


def _lens(c):
    """The sequences' tokens; "shared": those of their own, the step's among them."""
    return _run(c["seqs"], c["longest"], c["shortest"])


def _prefixes(c):
    """Each prefix's tokens, and the prefix of each sequence (-1: none), dealt in turn."""
    tokens = [max(PAGE, n // PAGE * PAGE) for n in _run(c["prefixes"], c["shared"], c["shared_least"])]
    return tokens, [i % c["prefixes"] if i < c["seqs"] - c["alone"] else -1 for i in range(c["seqs"])]


def _before(c):
    """Tokens in each cache before the step."""
    tokens, of = _prefixes(c)
    return [n - c["new"] + (tokens[p] if p >= 0 else 0) for n, p in zip(_lens(c), of)]


# --- rotary frequencies: a base of 5e6 over 32768 tokens, four times as many wanted -------------

BASE, KEPT, FACTOR, LOW, HIGH = 5e6, 32768.0, 4.0, 1.0, 32.0


def _frequencies(c):
    """In 64 bits, radians a token: as they are, divided, from a larger base, or between the divided (pairs of few turns over
    KEPT tokens) and the plain ones (of many), by their turns or by their index between the pairs of HIGH and LOW turns."""
    p, mode = c["pairs"], c["scaling"]
    j = torch.arange(p, dtype=torch.float64)
    base = BASE * FACTOR ** (p / (p - 1)) if mode == "base" else BASE
    f = base ** (-j / p)
    if mode == "linear":
        return f / FACTOR
    if mode == "turns":
        kept = ((KEPT * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        return f * kept + f / FACTOR * (1 - kept)
    if mode == "index":
        first, last = (p * math.log(KEPT / (2 * math.pi * n)) / math.log(BASE) for n in (HIGH, LOW))
        first, last = max(math.floor(first), 0), min(math.ceil(last), 2 * p - 1)
        gone = ((j - first) / (last - first if last != first else 1e-3)).clamp(0, 1)
        return f * (1 - gone) + f / FACTOR * gone
    return f


def _amp(c):
    return 1.0 + 0.1 * math.log(FACTOR) if c["scaling"] == "index" else 1.0


def _axis(c):
    """Each pair's axis: frame, row and column in turn in the first 15 of 16 pairs, then the frame."""
    return [j % 3 if c["axes"] == 3 and j < c["pairs"] * 15 // 16 else 0 for j in range(c["pairs"])]


def _quantised(x):
    """Blocks of rows [..., 64, dim] as codes and scales: a block's largest |x| / 127 in fp32, rounded up to 12
    significant bits, and x / scale to nearest even, in 64 bits (the quotient's ties are exact there)."""
    d = (x.abs().amax((-2, -1)).float() / 127).view(torch.int32)
    d = ((d + 0xFFF) & -0x1000).view(torch.float32)
    q = x.double() / d.double().clamp(min=1e-300)[..., None, None]
    return q.round().to(torch.int8), d


def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(int(seed) % (1 << 62))
    kv, hd, n = c["kv_heads"], c["dim"], c["seqs"]
    t = TYPES[c["dt"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # keys: a few channels carry an offset, as trained models' keys do
    lean = 3.0 * (torch.arange(hd, device=DEV) % 37 == 5)
    if c["kind"] == "rope":
        lens, rows = _lens(c), sum(_lens(c))
        st = {"c": c, "lens": lens, "q": (4 * normal(rows, c["heads"], hd)).to(t), "k": (2 * normal(rows, kv, hd) + lean).to(t)}
        if c["norm"]:
            st.update(wq=1 + 0.2 * normal(hd), wk=1 + 0.2 * normal(hd))
        if c["far"]:
            st["at"] = torch.tensor([max(0, x - 1) for x in _run(n, c["far"], max(1, c["far"] // 2))], device=DEV,
                                    dtype=torch.int32)
        else:
            # text from 0 on each; with axes, a picture's rows and columns from a third of the way on
            i = torch.cat([torch.arange(x, device=DEV) for x in lens])
            whole = torch.cat([torch.full((x,), x, device=DEV) for x in lens])
            first, side = whole // 3, (whole.double() / 2).sqrt().ceil().long()
            inside = (i >= first) & (i < first + side * side)
            f = torch.where(inside, first, torch.where(i >= first + side * side, i - side * side + side, i))
            y, x = (torch.where(inside, first + z, f) for z in ((i - first) // side, (i - first) % side))
            st["pos"] = torch.stack([f, y, x][:c["axes"]], -1).int().contiguous() if c["axes"] > 1 else i.int()[:, None].contiguous()
        st.update(qo=torch.empty(st["q"].shape, dtype=TYPES[c["odt"]], device=DEV),
                  ko=torch.empty(st["k"].shape, dtype=TYPES[c["odt"]], device=DEV))
        if own:
            X = _x()
            freqs = X.rope_freqs(2 * c["pairs"], BASE, getattr(X, "ROPE_" + c["scaling"].upper()), FACTOR, KEPT, LOW, HIGH)
            st["seqs"] = X.Seqs(_ctx(), lens)
            st["rope"] = X.Rope(_ctx(), freqs, X.ROPE_PAIRS if c["layout"] == "pairs" else X.ROPE_HALF,
                                _axis(c) if c["axes"] > 1 else None, _amp(c), c["axes"])
        return st
    new = c["new"]
    before, (tokens, of) = _before(c), _prefixes(c)
    total = [b + new for b in before]
    cols = max(total) // PAGE + 1
    blocks = [x // PAGE for x in tokens]
    pages = sum(blocks) + sum(-(-x // PAGE) for x in total) + 3
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.full((n, cols), -1, dtype=torch.int64, device=DEV)
    at = sum(blocks)
    for s in range(n):
        b = blocks[of[s]] if of[s] >= 0 else 0
        if b:
            r = sum(blocks[:of[s]])
            table[s, :b] = order[r:r + b]
        m = -(-total[s] // PAGE) - b
        table[s, b:b + m] = order[at:at + m]
        at += m
    st = {"c": c, "scale": hd ** -0.5, "before": before, "cols": cols, "table": table.int(),
          "lens": torch.tensor(before, device=DEV, dtype=torch.int32)}
    k, ks = _quantised((normal(pages, kv, PAGE, hd) + lean).to(t))
    v, vs = _quantised(normal(pages, kv, PAGE, hd).to(t))
    st.update(k8=k, v8=v.transpose(-1, -2).contiguous(), scales=torch.stack([ks, vs], -1).contiguous(),
              tk=(normal(n, kv, PAGE, hd) + lean).to(t), tv=normal(n, kv, PAGE, hd).to(t),
              q=normal(n * new, c["heads"], hd).to(t))
    st["out"] = torch.empty(st["q"].shape, dtype=TYPES[c["odt"]], device=DEV)
    if own:
        X = _x()
        st["seqs"] = X.Seqs(_ctx(), [new] * n)
        st["prefixes"] = X.Prefixes(_ctx(), st["seqs"], of, blocks)
        st["cache"] = X.Kv8(DT[c["dt"]](X), kv, hd, pages, n, cols, st["k8"].data_ptr(), st["v8"].data_ptr(),
                            st["scales"].data_ptr(), st["tk"].data_ptr(), st["tv"].data_ptr(), st["table"].data_ptr(),
                            st["lens"].data_ptr())
        floats = X.attend_shared_part(st["seqs"], st["prefixes"], c["heads"], kv, hd, cols)
        st["part"] = torch.empty(max(floats, 4), device=DEV)
    return st


# --- the framework's calls -------------------------------------------------------------------

DT = {"fp16": lambda X: X.DT_F16, "bf16": lambda X: X.DT_BF16, "fp32": lambda X: X.DT_F32}
_context = None


def _x():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ex-nihilo_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import exn_hip
    return exn_hip


def _ctx():
    global _context
    if _context is None:
        _context = _x().Context(0)
    return _context


def _own(st):
    X, ctx, c = _x(), _ctx(), st["c"]
    h, kv, hd = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "shared":
        X.attend_shared(ctx, st["cache"], st["seqs"], st["prefixes"], h, st["q"].data_ptr(), h * hd, st["scale"],
                            st["out"].data_ptr(), DT[c["odt"]](X), h * hd, st["part"].data_ptr(), st["part"].numel())
        return st["out"]
    wq, wk = (st[x].data_ptr() if c["norm"] else None for x in ("wq", "wk"))
    X.rope_rows(ctx, st["rope"], st["seqs"], hd, DT[c["dt"]](X), DT[c["odt"]](X),
                (h, st["q"].data_ptr(), h * hd, wq, st["qo"].data_ptr(), h * hd),
                (kv, st["k"].data_ptr(), kv * hd, wk, st["ko"].data_ptr(), kv * hd), eps=1e-6,
                pos=st["pos"].data_ptr() if "pos" in st else None, lens=st["at"].data_ptr() if "at" in st else None)
    return {"q": st["qo"], "k": st["ko"]}


# --- the plain forms -------------------------------------------------------------------------


def _plain_rope(st):
    c, p, d = st["c"], st["c"]["pairs"], torch.float64
    if "pos" in st:
        pos = st["pos"]
    else:
        pos = torch.cat([st["at"][s] + torch.arange(n, device=DEV) for s, n in enumerate(st["lens"])])[:, None]
    f = _frequencies(c).to(DEV)
    a = pos.to(d)[:, torch.tensor(_axis(c), device=DEV)] * f                           # (rows, pairs)
    cos, sin = ((_amp(c) * z).float()[:, None] for z in (a.cos(), a.sin()))
    got = {}
    for name, w in (("q", "wq"), ("k", "wk")):
        x = st[name].float()
        if c["norm"]:
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * st[w]
        u, v, rest = (x[..., :p], x[..., p:2 * p], x[..., 2 * p:]) if c["layout"] == "half" else \
            (x[..., 0:2 * p:2], x[..., 1:2 * p:2], x[..., 2 * p:])
        u, v = u * cos - v * sin, u * sin + v * cos
        turned = torch.cat([u, v], -1) if c["layout"] == "half" else torch.stack([u, v], -1).flatten(-2)
        got[name] = torch.cat([turned, rest], -1).to(TYPES[c["odt"]])
    return got


def _plain_shared(st):
    """Each prefix's keys and values once, for the rows of all its sequences; beside them, padded, each sequence's own."""
    c, new, kv, hd, cols = st["c"], st["c"]["new"], st["c"]["kv_heads"], st["c"]["dim"], st["cols"]
    group, (tokens, of) = c["heads"] // kv, _prefixes(c)
    out = torch.empty(c["seqs"], new, kv, group, hd, device=DEV)
    table, lens, q = st["table"].long(), st["lens"].long(), st["q"].float().view(c["seqs"], new, kv, group, hd)
    for p in range(-1, c["prefixes"]):
        who = [s for s in range(c["seqs"]) if of[s] == p]
        if not who:
            continue
        n, b = len(who), tokens[p] // PAGE if p >= 0 else 0
        ids = torch.tensor(who, device=DEV)
        last = max((st["before"][s] + new) // PAGE for s in who) + 1
        at, total = table[ids, b:last].clamp(min=0), lens[ids] + new
        keys, vals = [], []
        for codes, tail, w, got in ((st["k8"], st["tk"], 0, keys), (st["v8"].transpose(-1, -2), st["tv"], 1, vals)):
            x = codes[at].float() * st["scales"][at][..., w, None, None]               # (n, own blocks, kv, 64, hd)
            x[torch.arange(n, device=DEV), total // PAGE - b] = tail[ids].float()
            got.append(x.transpose(1, 2).reshape(n, kv, (last - b) * PAGE, hd))
            if b:
                x = codes[table[who[0], :b]].float() * st["scales"][table[who[0], :b]][..., w, None, None]
                got.append(x.transpose(0, 1).reshape(kv, b * PAGE, hd))
        mine = q[ids].permute(0, 2, 1, 3, 4).reshape(n, kv, new * group, hd)
        s = (mine @ keys[0].transpose(-1, -2).contiguous()).mul_(st["scale"]).view(n, kv, new, group, -1)
        place = lens[ids, None] + torch.arange(new, device=DEV)
        hidden = torch.arange(b * PAGE, last * PAGE, device=DEV) > place[..., None]    # (n, new, own keys)
        s = s.masked_fill_(hidden[:, None, :, None], -math.inf).view(n, kv, new * group, -1)
        top = s.amax(-1, keepdim=True)
        if b:
            all_rows = mine.transpose(0, 1).reshape(kv, n * new * group, hd)
            sp = (all_rows @ keys[1].transpose(-1, -2).contiguous()).mul_(st["scale"])
            top = torch.maximum(top, sp.amax(-1, keepdim=True).view(kv, n, -1, 1).transpose(0, 1))
        s = (s - top).exp_()
        total_w, o = s.sum(-1, keepdim=True), s @ vals[0]
        if b:
            sp = (sp - top.transpose(0, 1).reshape(kv, -1, 1)).exp_()
            total_w = total_w + sp.sum(-1, keepdim=True).view(kv, n, -1, 1).transpose(0, 1)
            o = o + (sp @ vals[1]).view(kv, n, -1, hd).transpose(0, 1)
        out[ids] = (o / total_w).view(n, kv, new, group, hd).permute(0, 2, 1, 3, 4)
    return out.view(-1, c["heads"], hd).to(st["out"].dtype)


PLAIN = {"rope": _plain_rope, "shared": _plain_shared}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["c"]["kind"]](state)


# --- what a pass cannot do without -----------------------------------------------------------


def work(case):
    c, kv, hd = case, case["kv_heads"], case["dim"]
    if c["kind"] == "rope":
        rows = sum(_lens(c))
        values = rows * (c["heads"] + kv) * hd
        at = 4 * c["seqs"] if c["far"] else 4 * c["axes"] * rows
        return {"bytes": values * (_size(c["dt"]) + _size(c["odt"])) + at + (8 * hd if c["norm"] else 0) + 8 * c["pairs"],
                "flops": values * (4 if c["norm"] else 0) + rows * (c["heads"] + kv) * 6 * c["pairs"]}
    new, (tokens, of) = c["new"], _prefixes(c)
    held = 2 * kv * hd
    b = sum(held * n + 8 * kv * (n // PAGE) for p, n in enumerate(tokens) if p in of)
    f = 0
    for n, p in zip(_before(c), of):
        tail, mine = (n + new) % PAGE, n + new - (tokens[p] if p >= 0 else 0)
        b += held * (mine + tail) + 8 * kv * (mine // PAGE) + new * c["heads"] * hd * 4
        f += 4 * hd * c["heads"] * (new * n + new * (new + 1) // 2)
    return {"bytes": b, "flops": f}


# --- the operators' definitions in 64 bits -----------------------------------------------------


def _exact_rope(case, seed):
    st, c = prepare(case, seed), case
    p, amp = c["pairs"], _amp(c)
    # each row's positions as whole numbers, and each pair's frequency by its own formula
    if "pos" in st:
        pos = st["pos"].tolist()
    else:
        pos = [[int(a) + i] for a, n in zip(st["at"].tolist(), st["lens"]) for i in range(n)]
    freqs = []
    for j in range(p):
        base = BASE * math.exp(math.log(FACTOR) * 2 * p / (2 * p - 2)) if c["scaling"] == "base" else BASE
        f = math.exp(-math.log(base) * 2 * j / (2 * p))
        if c["scaling"] == "linear":
            f /= FACTOR
        elif c["scaling"] == "turns":
            r = min(1.0, max(0.0, (f * KEPT / math.tau - LOW) / (HIGH - LOW)))
            f *= r + (1 - r) / FACTOR
        elif c["scaling"] == "index":
            ends = [2 * p * math.log(KEPT / (math.tau * turns)) / (2 * math.log(BASE)) for turns in (HIGH, LOW)]
            lo, hi = max(0, math.floor(ends[0])), min(2 * p - 1, math.ceil(ends[1]))
            r = min(1.0, max(0.0, (j - lo) / ((hi - lo) or 1e-3)))
            f *= (1 - r) + r / FACTOR
        freqs.append(f)
    axis = torch.tensor(_axis(c))
    a = torch.tensor(pos, dtype=torch.float64)[:, axis] * torch.tensor(freqs, dtype=torch.float64)
    turn = torch.polar(torch.full_like(a, amp), a).to(DEV)[:, None]
    got = {}
    for name, w in (("q", "wq"), ("k", "wk")):
        x = st[name].double()
        if c["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * st[w].double()
        y = x.clone()
        first, second = (slice(0, p), slice(p, 2 * p)) if c["layout"] == "half" else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        got[name] = y
    return got


def exact(case, seed):
    if case["kind"] == "rope":
        return _exact_rope(case, seed)
    st, c, kv, hd, new = prepare(case, seed), case, case["kv_heads"], case["dim"], case["new"]
    group, table = c["heads"] // kv, st["table"].tolist()
    q = st["q"].double().view(c["seqs"], new, kv, group, hd)
    out = torch.empty_like(q)
    for s, n in enumerate(st["before"]):
        total = n + new
        ids = table[s][:total // PAGE]
        left = total - len(ids) * PAGE
        seen = torch.arange(total, device=DEV) <= (n + torch.arange(new, device=DEV))[:, None, None]
        for h in range(kv):
            d = st["scales"][ids, h].double()
            k = (st["k8"][ids, h].double() * d[:, 0, None, None]).reshape(-1, hd)
            v = (st["v8"][ids, h].double() * d[:, 1, None, None]).transpose(1, 2).reshape(-1, hd)
            k = torch.cat([k, st["tk"][s, h, :left].double()])
            v = torch.cat([v, st["tv"][s, h, :left].double()])
            x = torch.mm(q[s, :, h].reshape(-1, hd) * hd ** -0.5, k.t().contiguous()).view(new, group, total)
            w = torch.softmax(x.masked_fill_(~seen, -math.inf), -1)
            out[s, :, h] = torch.mm(w.view(-1, total), v).view(new, group, hd)
    return out.view(-1, c["heads"], hd)
