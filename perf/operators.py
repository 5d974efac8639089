"""The prompt side's attention operators of exn_hip, as cases that can be timed and compared.

Three operators that a host serving pictures calls when it encodes prompts: causal attention over
several prompts packed one after the other (attend_packed); rows of keys and values into a cache
held in 8 bits, a scale for each block of 64 tokens and head (kv8_append, read back with kv8_read);
and the attention of new tokens over that cache (kv8_attend), from one token to a chunk.

The cache, as the library lays it out: a page is a block of 64 tokens; codes of keys
[page][kv head][64][dim] and of values [page][kv head][dim][64], scales [page][kv head][2] (key,
value); a sequence's last block, while it is not full, in 16 bits, tails [sequence][kv head][64][dim];
table [sequence][column] names the pages, lens the tokens before the step.  A block's scale is its
largest |x| / 127 in fp32, rounded up to 12 significant bits, and a code is x / scale rounded to
nearest even, so that codes are the same under any correctly rounded quotient.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE = 64
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one short prompt, the most usual call: latency alone
        {"name": "prompt 24", "kind": "prompts", "seqs": 1, "longest": 24, "shortest": 24, "heads": 32, "kv_heads": 8,
         "dim": 128, "dt": "fp16", "odt": "bf16"},
        # a server's batch of prompts, a line to a long description, ragged
        {"name": "16 prompts 21..257", "kind": "prompts", "seqs": 16, "longest": 257, "shortest": 21, "heads": 32,
         "kv_heads": 8, "dim": 128, "dt": "fp16", "odt": "bf16"},
        # edit prompts, a picture's 1024 rows amid text in each
        {"name": "4 edit prompts 1100..1180", "kind": "prompts", "seqs": 4, "longest": 1180, "shortest": 1100,
         "heads": 32, "kv_heads": 8, "dim": 128, "dt": "fp16", "odt": "bf16"},
        # a skewed batch for a smaller text model: narrow heads, eight to a key/value head
        {"name": "24 texts 5..4001, 64-wide", "kind": "prompts", "seqs": 24, "longest": 4001, "shortest": 5,
         "heads": 16, "kv_heads": 2, "dim": 64, "dt": "bf16", "odt": "bf16"},
        # long documents: the products' rate
        {"name": "2 documents 8192", "kind": "prompts", "seqs": 2, "longest": 8192, "shortest": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "dt": "bf16", "odt": "bf16"},
        # a serving step's new tokens into their caches, one in 64 filling its block
        {"name": "append 64 tokens", "kind": "append", "seqs": 64, "longest": 4000, "shortest": 63, "new": 1,
         "kv_heads": 8, "dim": 128, "dt": "fp16"},
        # whole prompts into empty caches
        {"name": "append 8 prompts 1100", "kind": "append", "seqs": 8, "longest": 0, "shortest": 0, "new": 1100,
         "kv_heads": 8, "dim": 128, "dt": "bf16"},
        # the next token of a few short texts: latency
        {"name": "4 tokens over 300", "kind": "cached", "seqs": 4, "longest": 333, "shortest": 270, "new": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "dt": "fp16", "odt": "bf16"},
        # a full batch's next tokens: the cache's bytes
        {"name": "64 tokens over 700..8191", "kind": "cached", "seqs": 64, "longest": 8191, "shortest": 700, "new": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "dt": "bf16", "odt": "bf16"},
        # one long text's next token: the keys' axis split over the chip
        {"name": "1 token over 131071", "kind": "cached", "seqs": 1, "longest": 131071, "shortest": 131071, "new": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "dt": "fp16", "odt": "fp16"},
        # an instruction after a kept template and picture
        {"name": "instruction 76 over 1100", "kind": "cached", "seqs": 1, "longest": 1100, "shortest": 1100, "new": 76,
         "heads": 32, "kv_heads": 8, "dim": 128, "dt": "fp16", "odt": "bf16"},
        # long texts continued chunk by chunk, a smaller model's narrow heads
        {"name": "chunks 512 over 4001, 64-wide", "kind": "cached", "seqs": 4, "longest": 4001, "shortest": 2500,
         "new": 512, "heads": 16, "kv_heads": 2, "dim": 64, "dt": "bf16", "odt": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("prompts", "prompts", "append", "cached", "cached", "cached"))
    kv, group = rng.choice(((8, 4), (8, 4), (2, 8), (8, 1), (4, 3), (1, 16), (4, 2)))
    c = {"kind": kind, "seqs": _log(rng, 1, 64), "heads": kv * group, "kv_heads": kv, "dim": rng.choice((64, 128, 128)),
         "dt": rng.choice(("fp16", "bf16")), "odt": rng.choice(("fp16", "bf16"))}
    if kind == "prompts":
        c["longest"] = _log(rng, 1, 8192)
        c["shortest"] = _log(rng, 1, c["longest"])
        while sum(n * n for n in _lens(c)) * c["heads"] > 2 * 8192 ** 2 * 32 or sum(_lens(c)) > 32768:
            c["seqs"] = (c["seqs"] + 1) // 2
            c["longest"] = max(1, c["longest"] * 3 // 4)
            c["shortest"] = min(c["shortest"], c["longest"])
        return c
    c["new"] = 1 if kind == "cached" and rng.random() < 0.5 else _log(rng, 1, 1100 if kind == "append" else 512)
    c["longest"] = max(c["new"], _log(rng, 16, 131072))
    c["shortest"] = max(c["new"], _log(rng, max(1, c["longest"] // 16), c["longest"]))
    if kind == "append":
        del c["heads"], c["odt"]
        c["longest"], c["shortest"] = min(c["longest"], 8192), min(c["shortest"], 8192)
        while c["seqs"] * c["new"] > 8800:
            c["seqs"] //= 2
        return c
    # the padded plain form's scores and the cache's bytes stay those of the listed cases
    while c["seqs"] * c["longest"] > 64 * 8192 or c["seqs"] * c["longest"] * c["new"] * c["heads"] > 4 * 4096 * 512 * 64:
        if c["seqs"] > 1:
            c["seqs"] //= 2
        else:
            c["new"] = max(1, c["new"] // 2)
    return c


def _lens(c):
    """The sequences' tokens: a geometric run from the longest to the shortest, in a mixed order."""
    n, a, b = c["seqs"], c["longest"], c["shortest"]
    run = [int(round(a * (b / a) ** (i / (n - 1)))) if n > 1 and a else a for i in range(n)]
    return [run[i * 7919 % n] for i in range(n)]


def _before(c):
    """Tokens in each cache before the step: "cached" counts the new ones in its lengths; "append" starts at a block's
    first token where the new ones would fill a block and go on in the next (a pass can then be made again)."""
    if c["kind"] == "cached":
        return [n - c["new"] for n in _lens(c)]
    return [n - n % PAGE if n % PAGE + c["new"] > PAGE else n for n in _lens(c)]


def _quantised(x):
    """Blocks of rows [..., 64, dim] as codes and scales, in 64 bits (the quotient's ties are exact there)."""
    d = (x.abs().amax((-2, -1)).float() / 127).view(torch.int32)
    d = ((d + 0xFFF) & -0x1000).view(torch.float32)
    q = x.double() / d.double().clamp(min=1e-300)[..., None, None]
    return q.round().to(torch.int8), d


def prepare(case, seed):
    c = case
    g = torch.Generator(DEV).manual_seed(int(seed) % (1 << 62))
    t, kv, hd = TYPES[c["dt"]], c["kv_heads"], c["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # keys after their norm: a few channels carry an offset, as trained models' keys do
    lean = 3.0 * (torch.arange(hd, device=DEV) % 37 == 5)
    st = {"c": c, "scale": hd ** -0.5}
    if c["kind"] == "prompts":
        rows = sum(_lens(c))
        st.update(lens=_lens(c), q=normal(rows, c["heads"], hd).to(t), k=(normal(rows, kv, hd) + lean).to(t),
                  v=normal(rows, kv, hd).to(t))
        if own:
            st["seqs"] = _x().Seqs(_ctx(), st["lens"])
    else:
        before, new, n = _before(c), c["new"], c["seqs"]
        total = [b + new for b in before]
        cols = max(total) // PAGE + 1
        used = [-(-x // PAGE) for x in total]
        pages = sum(used) + 3
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.tensor([sum(used[:i]) for i in range(n)], device=DEV)[:, None] + torch.arange(cols, device=DEV)
        live = torch.arange(cols, device=DEV) < torch.tensor(used, device=DEV)[:, None]
        st.update(before=before, cols=cols, pages=pages,
                  table=torch.where(live, order[at.clamp(max=pages - 1)], -1).int(),
                  lens=torch.tensor(before, device=DEV, dtype=torch.int32))
        k, ks = _quantised((normal(pages, kv, PAGE, hd) + lean).to(t))
        v, vs = _quantised(normal(pages, kv, PAGE, hd).to(t))
        st.update(k8=k, v8=v.transpose(-1, -2).contiguous(), scales=torch.stack([ks, vs], -1).contiguous(),
                  tk=(normal(n, kv, PAGE, hd) + lean).to(t), tv=normal(n, kv, PAGE, hd).to(t))
        if c["kind"] == "append":
            st.update(k=(normal(n * new, kv, hd) + lean).to(t), v=normal(n * new, kv, hd).to(t))
        else:
            st["q"] = normal(n * new, c["heads"], hd).to(t)
        if own:
            X = _x()
            st["seqs"] = X.Seqs(_ctx(), [new] * n)
            st["cache"] = X.Kv8(DT[c["dt"]](X), kv, hd, pages, n, cols, st["k8"].data_ptr(), st["v8"].data_ptr(),
                                st["scales"].data_ptr(), st["tk"].data_ptr(), st["tv"].data_ptr(),
                                st["table"].data_ptr(), st["lens"].data_ptr())
    if c["kind"] == "append":
        st.update(kr=torch.empty_like(st["k"]), vr=torch.empty_like(st["v"]))
    else:
        st["out"] = torch.empty(st["q"].shape, dtype=TYPES[c["odt"]], device=DEV)
    if own and c["kind"] == "cached":
        floats = _x().kv8_attend_part(st["seqs"], c["heads"], kv, hd, st["cols"])
        st["part"] = torch.empty(max(floats, 4), device=DEV)
    return st


# --- the framework's calls -------------------------------------------------------------------

DT = {"fp16": lambda X: X.DT_F16, "bf16": lambda X: X.DT_BF16}
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
    kv, hd = c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        k, v = st["k"], st["v"]
        X.kv8_append(ctx, st["cache"], st["seqs"], k.data_ptr(), kv * hd, v.data_ptr(), kv * hd)
        X.kv8_read(ctx, st["cache"], st["seqs"], st["kr"].data_ptr(), kv * hd, st["vr"].data_ptr(), kv * hd)
        return {"k": st["kr"], "v": st["vr"]}
    h, q, out = c["heads"], st["q"], st["out"]
    if c["kind"] == "prompts":
        X.attend_packed(ctx, st["seqs"], DT[c["dt"]](X), h, kv, hd, q.data_ptr(), h * hd, st["k"].data_ptr(), kv * hd,
                        st["v"].data_ptr(), kv * hd, st["scale"], out.data_ptr(), DT[c["odt"]](X), h * hd)
    else:
        X.kv8_attend(ctx, st["cache"], st["seqs"], h, q.data_ptr(), h * hd, st["scale"], out.data_ptr(),
                     DT[c["odt"]](X), h * hd, st["part"].data_ptr(), st["part"].numel())
    return out


# --- the plain forms -------------------------------------------------------------------------


def _plain_prompts(st):
    c, outs, r = st["c"], [], 0
    kv, hd = c["kv_heads"], c["dim"]
    for n in st["lens"]:
        q, k, v = (st[x][r:r + n].float().transpose(0, 1) for x in "qkv")
        s = q.reshape(kv, -1, hd) @ k.transpose(-1, -2).contiguous() * st["scale"]      # (kv, group n, n)
        s = s.view(kv, -1, n, n).masked_fill_(torch.ones(n, n, dtype=torch.bool, device=DEV).triu_(1), -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        outs.append((p.view(kv, -1, n) @ v.contiguous()).view(-1, n, hd).transpose(0, 1))
        r += n
    return torch.cat(outs).to(st["out"].dtype)


def _rows(st, tail_at):
    """The cache's keys and values as 32-bit rows [sequence][kv head][column x 64][dim]; from each sequence's place
    tail_at on, a multiple of 64, its tail's."""
    c, cols = st["c"], st["cols"]
    at = st["table"].long().clamp(min=0)
    got = []
    for codes, tail, w in ((st["k8"], st["tk"], 0), (st["v8"].transpose(-1, -2), st["tv"], 1)):
        x = codes[at].float() * st["scales"][at][..., w, None, None]                    # (n, cols, kv, 64, hd)
        x[torch.arange(c["seqs"], device=DEV), tail_at // PAGE] = tail.float()
        got.append(x.transpose(1, 2).reshape(c["seqs"], c["kv_heads"], cols * PAGE, c["dim"]))
    return got


def _plain_append(st):
    c, n, new, kv, hd = st["c"], st["c"]["seqs"], st["c"]["new"], st["c"]["kv_heads"], st["c"]["dim"]
    lens, cols = st["lens"].long(), st["cols"]
    first = lens // PAGE                                                               # the block the step begins in
    nb = (PAGE - 1 + new - 1) // PAGE + 1                                              # blocks that a step can touch
    i = torch.arange(n, device=DEV)
    block = first[:, None] + torch.arange(nb, device=DEV)                              # (n, nb)
    full = (block + 1) * PAGE <= (lens + new)[:, None]
    page = st["table"].long()[i[:, None], block.clamp(max=cols - 1)]
    there = ((lens + new) // PAGE < block[:, :1] + nb)
    last = ((lens + new) // PAGE - first).clamp(max=nb - 1)
    spot = (lens % PAGE)[:, None] + torch.arange(new, device=DEV)                      # the new rows among those blocks
    got = {}
    for x, codes, tail, w, back in (("k", "k8", "tk", 0, False), ("v", "v8", "tv", 1, True)):
        rows = torch.zeros(n, nb * PAGE, kv, hd, device=DEV, dtype=st[x].dtype)
        rows[:, :PAGE] = st[tail].transpose(1, 2)
        rows[i[:, None], spot] = st[x].view(n, new, kv, hd)
        blocks = rows.view(n, nb, PAGE, kv, hd).transpose(2, 3)                        # (n, nb, kv, 64, hd)
        q, d = _quantised(blocks)
        st[codes][page[full]] = (q.transpose(-1, -2) if back else q)[full]
        st["scales"][page[full], :, w] = d[full]
        begun = ((lens + new) % PAGE > 0) & there[:, 0]
        kept = torch.arange(PAGE, device=DEV) < ((lens + new) % PAGE)[:, None]         # the rows the last block has
        kept = (kept & begun[:, None])[:, None, :, None]
        st[tail].copy_(torch.where(kept, blocks[i, last], st[tail]))
        seen = torch.where(full[..., None, None, None], q.float() * d[..., None, None], blocks.float())
        seen = seen.transpose(2, 3).reshape(n, nb * PAGE, kv, hd)
        got[x] = seen[i[:, None], spot].view(n * new, kv, hd).to(st[x].dtype)
    return got


def _plain_cached(st):
    c, n, new, kv, hd = st["c"], st["c"]["seqs"], st["c"]["new"], st["c"]["kv_heads"], st["c"]["dim"]
    total = st["lens"].long() + new
    k, v = _rows(st, total - total % PAGE)
    q = st["q"].float().view(n, new, kv, -1, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, hd)
    s = (q @ k.transpose(-1, -2).contiguous()).mul_(st["scale"]).view(n, kv, -1, new, st["cols"] * PAGE)
    place = st["lens"].long()[:, None] + torch.arange(new, device=DEV)
    hidden = torch.arange(st["cols"] * PAGE, device=DEV) > place[..., None]            # (n, new, keys)
    s.masked_fill_(hidden[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = p.view(n, kv, -1, st["cols"] * PAGE) @ v
    return o.view(n, kv, -1, new, hd).permute(0, 3, 1, 2, 4).reshape(n * new, -1, hd).to(st["out"].dtype)


PLAIN = {"prompts": _plain_prompts, "append": _plain_append, "cached": _plain_cached}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["c"]["kind"]](state)


# --- what a pass cannot do without -----------------------------------------------------------


def work(case):
    c, kv, hd = case, case["kv_heads"], case["dim"]
    if c["kind"] == "prompts":
        rows, pairs = sum(_lens(c)), sum(n * (n + 1) // 2 for n in _lens(c))
        return {"bytes": rows * (2 * c["heads"] + 2 * kv) * hd * 2, "flops": 4 * hd * c["heads"] * pairs}
    before, new = _before(c), c["new"]
    if c["kind"] == "append":
        b = 0
        for n in before:
            full = ((n + new) // PAGE - n // PAGE) * PAGE
            old = n % PAGE if full else 0
            kept = min(new, (n + new) % PAGE)
            # rows in (with the block's earlier ones), codes or 16-bit rows out, the read-back in and out
            b += (new + old) * 2 + full + kept * 2 + (new - kept) + kept * 2 + new * 2
        return {"bytes": b * kv * hd * 2, "flops": 4 * len(before) * new * kv * hd}
    b = f = 0
    for n in before:
        tail = (n + new) % PAGE
        b += 2 * kv * hd * (n + new - tail + 2 * tail) + 8 * kv * ((n + new) // PAGE) + new * c["heads"] * hd * 4
        f += 4 * hd * c["heads"] * (new * n + new * (new + 1) // 2)
    return {"bytes": b, "flops": f}


# --- the operators' definitions in 64 bits -----------------------------------------------------


def _softmax_rows(q, k, v, first):
    """Query i (place first + i) of q [n][dim] over rows 0 .. first + i of k and v, one head."""
    out = torch.empty(q.shape[0], v.shape[1], dtype=torch.float64, device=DEV)
    step = max(1, (1 << 27) // max(1, k.shape[0]))
    j = torch.arange(k.shape[0], device=DEV)
    for a in range(0, q.shape[0], step):
        i = torch.arange(a, min(a + step, q.shape[0]), device=DEV)
        s = torch.mm(q[i], k.t().contiguous()).masked_fill_(j > (first + i)[:, None], -math.inf)
        out[i] = torch.mm(torch.softmax(s, -1), v)
    return out


def _block64(x):
    """A block's rows as its codes stand for them, in 64 bits."""
    top = float(x.abs().max())
    if top == 0:
        return torch.zeros_like(x)
    d = float((torch.tensor(top, dtype=torch.float32) / 127))
    m, e = math.frexp(d)
    d = math.ldexp(math.ceil(m * 4096), e - 12)                                        # 12 significant bits, upwards
    return torch.round(x / d) * d


def exact(case, seed):
    st = prepare(case, seed)
    c, kv, hd = case, case["kv_heads"], case["dim"]
    if c["kind"] == "prompts":
        q, k, v = (st[x].double() for x in "qkv")
        group, out, r = c["heads"] // kv, torch.empty(q.shape, dtype=torch.float64, device=DEV), 0
        for n in st["lens"]:
            for h in range(c["heads"]):
                out[r:r + n, h] = _softmax_rows(q[r:r + n, h] * hd ** -0.5, k[r:r + n, h // group],
                                                v[r:r + n, h // group], 0)
            r += n
        return out
    table, new = st["table"].tolist(), c["new"]
    if c["kind"] == "append":
        if c["seqs"] * new * kv > 1 << 17:
            return None
        got = {}
        for x, tail in (("k", "tk"), ("v", "tv")):
            rows, old = st[x].double().view(c["seqs"], new, kv, hd), st[tail].double()
            out = torch.empty_like(rows)
            for s, n in enumerate(st["before"]):
                have = n % PAGE
                all_rows = torch.cat([old[s, :, :have], rows[s].transpose(0, 1)], 1)   # (kv, have + new, hd)
                for h in range(kv):
                    seen = all_rows[h].clone()
                    for b in range((have + new) // PAGE):
                        seen[b * PAGE:(b + 1) * PAGE] = _block64(all_rows[h, b * PAGE:(b + 1) * PAGE])
                    out[s, :, h] = seen[have:]
            got[x] = out.view(-1, kv, hd)
        return got
    group = c["heads"] // kv
    q = st["q"].double().view(c["seqs"], new, c["heads"], hd)
    out = torch.empty_like(q)
    for s, n in enumerate(st["before"]):
        total = n + new
        full = total // PAGE
        ids = table[s][:full]
        for h in range(kv):
            d = st["scales"][ids, h].double()
            k = (st["k8"][ids, h].double() * d[:, 0, None, None]).reshape(-1, hd)
            v = (st["v8"][ids, h].double() * d[:, 1, None, None]).transpose(1, 2).reshape(-1, hd)
            k = torch.cat([k, st["tk"][s, h, :total % PAGE].double()])
            v = torch.cat([v, st["tv"][s, h, :total % PAGE].double()])
            for j in range(h * group, (h + 1) * group):
                out[s, :, j] = _softmax_rows(q[s, :, j] * hd ** -0.5, k, v, n)
    return out.view(-1, c["heads"], hd)
