"""Timing cases of the paged latent cache and of attention over packed prompts.

Each case is a dict of plain values; ``kind`` names the operator:

* ``append``  new tokens' latents into the pages of their sequences, one token a sequence or packed
  prompts (``paged.append``), and the pool's entries as the values they stand for;
* ``attend``  attention of the newest token of each sequence, or of its last few, over the sequence's
  pages, or over selected entries of them (``paged.attend``);
* ``packed``  causal attention over whole prompts of different lengths, one after another in one
  tensor (``csa2_attn.packed``);
* ``grow``, ``fork``, ``compact``  the pages themselves: room for new tokens (with a copy of a shared
  last page), sequences that begin as others' copies or end, and used pages moved together.

Latents are K and V at once, heads share them, scores are scaled by D^-0.5 and a head's sink is one
more term of its softmax's denominator.  The plain forms are elementary torch operations in 32 bits.
"""

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
ROPE = {576: 64, 160: 32}  # channels of an 8-bit entry that stay in bfloat16


# ---- the cases ----------------------------------------------------------------------------

def listed():
    return [
        # one new token of each of 64 conversations, 8-bit entries
        dict(name="append b64 fp8", kind="append", batch=64, most=1, ctx=512, dim=576, page=64, fmt="fp8", x="bfloat16"),
        # a serving step that takes in new prompts of different lengths
        dict(name="append 12 prompts fp8", kind="append", batch=12, most=2000, ctx=2000, dim=576, page=64, fmt="fp8",
             x="bfloat16"),
        # one user's chat turn: launches and latency count
        dict(name="attend b1 4k", kind="attend", batch=1, ctx=4096, tokens=1, heads=128, dim=576, page=64, fmt="fp8",
             window=0, topk=0),
        # a full batch at contexts up to 32k, every sequence at its own length
        dict(name="attend b32 32k", kind="attend", batch=32, ctx=32768, tokens=1, heads=128, dim=576, page=64,
             fmt="fp8", window=0, topk=0),
        # the indexer's selection out of long paged caches, half the heads (two cards share a layer)
        dict(name="attend b8 128k top2048", kind="attend", batch=8, ctx=131072, tokens=1, heads=64, dim=576, page=64,
             fmt="fp8", window=0, topk=2048),
        # a smaller model checks four drafted tokens a sequence; pages that end inside a tile
        dict(name="attend b24x4 9k d160", kind="attend", batch=24, ctx=9000, tokens=4, heads=16, dim=160, page=24,
             fmt="bf16", window=0, topk=0),
        # one long prompt, every head
        dict(name="packed 8192 h128", kind="packed", batch=1, most=8192, heads=128, groups=1, dim=576, window=0),
        # a step's ragged prompts in a sliding-window layer, few heads
        dict(name="packed 9 prompts h16 window", kind="packed", batch=9, most=4000, heads=16, groups=1, dim=576,
             window=128),
        # short prompts of a small model with two latents, each for half of its heads
        dict(name="packed 17 prompts h8 d160", kind="packed", batch=17, most=700, heads=8, groups=2, dim=160, window=0),
        # a step of 128 sequences of which some begin a page and some share their last one
        dict(name="grow b128", kind="grow", batch=128, ctx=8192, page=64, pages=16384, dim=576),
        # beams: every sequence continues one of the present ones, some end
        dict(name="fork b64 32k", kind="fork", batch=64, ctx=32768, page=64, pages=32768, dim=0),
        # a cache that was used by many short conversations, half empty, made dense
        dict(name="compact 4096 pages", kind="compact", batch=32, ctx=8192, page=64, pages=4096, dim=576),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "packed", "packed", "packed", "grow", "fork", "compact"])
    page = rng.choice([1, 7, 16, 24, 32, 64, 100, 128])
    if kind == "append":
        fmt = rng.choice(["fp8", "fp8", "bf16"])
        one = rng.random() < 0.4
        batch = _log(rng, 1, 256) if one else _log(rng, 1, 24)
        return dict(kind=kind, batch=batch, most=1 if one else _log(rng, 2, 12000 // batch), ctx=_log(rng, 20, 24000 // batch),
                    dim=rng.choice([160, 576, 576] if fmt == "fp8" else [64, 96, 128, 160, 256, 512, 576]), page=page, fmt=fmt,
                    x=rng.choice(["bfloat16", "bfloat16", "float32", "float16"]))
    if kind == "attend":
        fmt = rng.choice(["fp8", "fp8", "bf16"])
        batch = _log(rng, 1, 96)
        return dict(kind=kind, batch=batch, ctx=_log(rng, 30, min(131072, (1 << 19) // batch)),
                    tokens=rng.choice([1, 1, 1, 2, 5]), heads=rng.choice([1, 5, 8, 16, 32, 64, 128, 128]),
                    dim=rng.choice([160, 576, 576] if fmt == "fp8" else [64, 96, 128, 160, 256, 512, 576]), page=page, fmt=fmt,
                    window=rng.choice([0, 0, 0, 128, 1000]), topk=0) if rng.random() < 0.7 else \
            dict(kind=kind, batch=batch, ctx=_log(rng, 30, min(131072, (1 << 19) // batch)), tokens=1,
                 heads=rng.choice([8, 32, 64, 128]), dim=576, page=page, fmt=fmt, window=0, topk=rng.choice([100, 512, 2048]))
    if kind == "packed":
        heads, groups = rng.choice([(1, 1), (3, 1), (8, 1), (8, 2), (16, 1), (24, 3), (32, 1), (64, 1), (128, 1), (128, 1)])
        batch = _log(rng, 1, 40)
        return dict(kind=kind, batch=batch, most=_log(rng, 4, 8000 // batch), heads=heads, groups=groups,
                    dim=rng.choice([64, 96, 128, 160, 256, 512, 576, 576, 576]), window=rng.choice([0, 0, 0, 1, 64, 500]))
    batch = _log(rng, 1, 200)
    page = rng.choice([16, 32, 64])
    if kind == "fork":
        ctx = _log(rng, 20, 32768)
        return dict(kind=kind, batch=batch, ctx=ctx, page=page, pages=batch * -(-ctx // page) + rng.randrange(1, 5000), dim=0)
    ctx = _log(rng, 20, max(21, 4096 * page // batch))
    spare = batch + rng.randrange(1, 300)
    return dict(kind=kind, batch=batch, ctx=ctx, page=page, pages=batch * -(-ctx // page) + spare,
                dim=rng.choice([64, 160, 576]))


# ---- formats ------------------------------------------------------------------------------

def _pack_fp8(x, rope):
    """[..., D] -> entries uint8: e4m3 codes of all but the last ``rope`` channels, a power-of-two fp32
    scale for each 128 of them, and the rest in bfloat16."""
    x = x.float()
    body, tail = x[..., :-rope], x[..., -rope:].bfloat16()
    blocks = body.unflatten(-1, (-1, 128))
    need = blocks.abs().amax(-1).clamp_min(1e-4) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=x.device)
    mant, ex = torch.frexp(need)
    scale = torch.ldexp(torch.ones_like(need), ex - (mant == 0.5).int())
    codes = (blocks / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    return torch.cat([codes, scale.view(torch.uint8), tail.contiguous().view(torch.uint8)], -1)


def _unpack_fp8(e, dim):
    """Entries -> the float32 values that they stand for."""
    nope = dim - ROPE[dim]
    nb = nope // 128
    val = e[..., :nope].contiguous().view(torch.float8_e4m3fn).float().unflatten(-1, (nb, 128))
    scale = e[..., nope:nope + 4 * nb].contiguous().view(torch.float32)
    tail = e[..., nope + 4 * nb:].contiguous().view(torch.bfloat16).float()
    return torch.cat([(val * scale[..., None]).flatten(-2), tail], -1)


def _values(e, c):
    return _unpack_fp8(e, c["dim"]) if c["fmt"] == "fp8" else e.float()


# ---- inputs -------------------------------------------------------------------------------

def _rnd(seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 23)
    return lambda *shape: torch.randn(*shape, generator=gen, device=DEV)


def _lengths(c):
    """A case's lengths, the longest its largest size: (new tokens, tokens with them) of each sequence."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    b, kind = c["batch"], c["kind"]

    def between(lo, hi):
        return [hi] + [rng.randint(lo, hi) for _ in range(b - 1)]

    if kind == "append":
        new = between(1, c["most"])
        return [(n, n + rng.randrange(0, c["ctx"])) for n in new]
    if kind == "attend":
        n = c["tokens"]
        return [(n, end) for end in between(max(n, c["ctx"] // 4), max(n, c["ctx"]))]
    if kind == "packed":
        return [(n, n) for n in between(1, c["most"])]
    return [(0, n if kind != "compact" else max(1, n // 2)) for n in between(1, c["ctx"])]


def _tables(c, rng, lens):
    """Each sequence's pages, scattered over the pool as after hours of use; -1 behind them, with room
    for one page more.  Returns the table and the pages that nobody holds."""
    page = c["page"]
    free = list(range(c["pages"]))
    rng.shuffle(free)
    wide = -(-(max(max(lens), c["ctx"]) + page) // page)
    out = np.full((len(lens), wide), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            out[b, j] = free.pop()
    return out, free


def _pool(c, seed):
    """Every entry of the pool filled: what earlier conversations left there, and what is read."""
    rnd = _rnd(seed + 1)
    n, page, dim = c["pages"], c["page"], c["dim"]
    if c.get("fmt", "bf16") == "bf16":
        out = torch.empty(n * page, dim, dtype=torch.bfloat16, device=DEV)
    else:
        nope = dim - ROPE[dim]
        out = torch.empty(n * page, nope + nope // 32 + 2 * ROPE[dim], dtype=torch.uint8, device=DEV)
    for i in range(0, n * page, 65536):
        x = rnd(min(65536, n * page - i), dim).bfloat16()
        out[i:i + 65536] = x if out.dtype == torch.bfloat16 else _pack_fp8(x, ROPE[dim])
    return out.view(n, page, -1)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def prepare(c, seed):
    rng = random.Random(seed * 104729 + 7)
    rnd = _rnd(seed)
    c = dict(c)
    s = dict(c=c)
    kind, b = c["kind"], c["batch"]
    both = _lengths(c)
    rng.shuffle(both)
    new, lens = [n for n, _ in both], [n for _, n in both]
    if kind == "append":
        c["pages"] = sum(-(-n // c["page"]) for n in lens) + 3
        table, _ = _tables(c, rng, lens)
        cu = np.concatenate([[0], np.cumsum(new)]).tolist()
        s.update(pool=_pool(c, seed), tables=torch.from_numpy(table).to(DEV), lens=_i64(lens), new=new, ends=lens,
                 x=rnd(cu[-1], c["dim"]).to(getattr(torch, c["x"])), cu=None if c["most"] == 1 else _i64(cu))
    elif kind == "attend":
        c["pages"] = sum(-(-n // c["page"]) for n in lens) + 5
        table, _ = _tables(c, rng, lens)
        t = b * c["tokens"]
        idx = None
        if c["topk"]:
            # the indexer's list: ascending positions, then -1
            idx = torch.full((b, c["topk"]), -1, dtype=torch.int32, device=DEV)
            for i, n in enumerate(lens):
                k = min(n, c["topk"])
                idx[i, :k] = rnd(n).topk(k).indices.sort().values.int()
        s.update(pool=_pool(c, seed), tables=torch.from_numpy(table).to(DEV), lens=_i64(lens), ends=lens, idx=idx,
                 q=rnd(t, c["heads"], c["dim"]).bfloat16(), sinks=rnd(c["heads"]),
                 cu=None if c["tokens"] == 1 else _i64([i * c["tokens"] for i in range(b + 1)]))
    elif kind == "packed":
        cu = np.concatenate([[0], np.cumsum(new)]).tolist()
        s.update(q=rnd(cu[-1], c["heads"], c["dim"]).bfloat16(), kv=rnd(cu[-1], c["groups"], c["dim"]).bfloat16(),
                 sinks=rnd(c["heads"]), cu=_i64(cu), ends=cu)
    else:
        table, _ = _tables(c, rng, lens)
        if kind == "grow":
            # a quarter of the sequences begin as copies of others and share all their pages
            for i in range(b // 4):
                j = rng.randrange(b // 4, b)
                table[i], lens[i] = table[j], lens[j]
            s["tokens"] = _i64([rng.choice([0, 1, 1, 1, 1, 1, 3]) for _ in range(b)])
        if kind == "fork":
            s["parents"] = torch.tensor([rng.choice([-1] + [rng.randrange(b)] * 9) for _ in range(b)], dtype=torch.int32,
                                        device=DEV)
        refs = np.bincount(table[table >= 0].ravel(), minlength=c["pages"]).astype(np.int32)
        s.update(tables=torch.from_numpy(table).to(DEV), lens=_i64(lens), refs=torch.from_numpy(refs).to(DEV),
                 pool=_pool(c, seed) if c["dim"] else None)
    return s


# ---- the operators ------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from mzoo_amd import csa2_attn, paged, quant
    c = s["c"]
    kind = c["kind"]
    rope = ROPE.get(c["dim"], 0)
    if kind == "append":
        paged.append(s["pool"], s["tables"], s["lens"], s["x"], cu=s["cu"], rope=rope)
        if c["fmt"] == "bf16":
            return s["pool"]
        return quant.unpack_latent_fp8_b128(s["pool"], c["dim"] - rope, rope, dtype=torch.float32)
    if kind == "attend":
        return paged.attend(s["q"], s["pool"], s["tables"], s["lens"], cu=s["cu"], window=c["window"] or None,
                            indices=s["idx"], sinks=s["sinks"], rope=rope)
    if kind == "packed":
        return csa2_attn.packed(s["q"], s["kv"], s["cu"], window=c["window"] or None, sinks=s["sinks"])
    if kind == "grow":
        return (*paged.grow(s["tables"], s["lens"], s["refs"], s["tokens"], c["page"], pools=[s["pool"]]), s["pool"])
    if kind == "fork":
        return paged.fork(s["tables"], s["lens"], s["refs"], s["parents"], c["page"])
    return (*paged.compact(s["tables"], s["refs"], pools=[s["pool"]]), s["pool"])


def _slots(s, b, first, n):
    """Entry numbers in the pool of positions first .. first + n - 1 of sequence b."""
    page = s["c"]["page"]
    pos = torch.arange(first, first + n, device=DEV)
    return s["tables"][b].long()[pos // page] * page + pos % page


def _softmax_rows(q, e, seen, sink):
    """q [T, H, D], e [N, D], seen bool [T, N] or None, sink [H] -> (o [T, H, D], lse [T, H])."""
    t, h, d = q.shape
    sc = (q.reshape(t * h, d) @ e.t()).view(t, h, -1) * d ** -0.5
    if seen is not None:
        sc = sc.masked_fill_(~seen[:, None, :], float("-inf"))
    m = torch.maximum(sc.amax(-1), sink)
    w = sc.sub_(m[..., None]).exp_()
    total = w.sum(-1) + (sink - m).exp()
    o = (w.view(t * h, -1) @ e).view(t, h, d) / total[..., None]
    return o, m + total.log()


def _causal(q, e, first, window, sink):
    """Tokens at positions first, first + 1, .. over entries 0 .. of their sequence, in blocks that
    bound the scores' memory."""
    t, h, d = q.shape
    o, z = torch.empty(t, h, d, device=DEV), torch.empty(t, h, device=DEV)
    step = max(1, (1 << 27) // (h * e.shape[0]))
    for i in range(0, t, step):
        n = min(step, t - i)
        pos = first + torch.arange(i, i + n, device=DEV)[:, None]
        lo = max(0, first + i - window + 1) if window else 0
        hi = first + i + n
        col = torch.arange(lo, hi, device=DEV)[None, :]
        seen = col <= pos
        if window:
            seen &= col > pos - window
        o[i:i + n], z[i:i + n] = _softmax_rows(q[i:i + n], e[lo:hi], seen, sink)
    return o, z


def _run_plain(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "append":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        at = torch.cat([_slots(s, i, end - n, n) for i, (n, end) in enumerate(zip(s["new"], s["ends"]))])
        flat[at] = s["x"].bfloat16() if c["fmt"] == "bf16" else _pack_fp8(s["x"], ROPE[c["dim"]])
        return s["pool"] if c["fmt"] == "bf16" else _unpack_fp8(s["pool"], c["dim"])
    if kind == "attend":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        o, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=DEV)
        n = c["tokens"]
        for i, end in enumerate(s["ends"]):
            q = s["q"][i * n:(i + 1) * n].float()
            if s["idx"] is not None:
                at = s["idx"][i, :min(end, c["topk"])].long()
                at = s["tables"][i].long()[at // c["page"]] * c["page"] + at % c["page"]
                got = _softmax_rows(q, _values(flat[at], c), None, s["sinks"])
            else:
                got = _causal(q, _values(flat[_slots(s, i, 0, end)], c), end - n, c["window"], s["sinks"])
            o[i * n:(i + 1) * n], lse[i * n:(i + 1) * n] = got
        return o, lse
    if kind == "packed":
        o, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=DEV)
        per = c["heads"] // c["groups"]
        for a, z in zip(s["ends"], s["ends"][1:]):
            for g in range(c["groups"]):
                hs = slice(g * per, (g + 1) * per)
                o[a:z, hs], lse[a:z, hs] = _causal(s["q"][a:z, hs].float(), s["kv"][a:z, g].float(), 0, c["window"],
                                                   s["sinks"][hs])
        return o, lse
    if kind == "grow":
        return _plain_grow(s)
    if kind == "fork":
        return _plain_fork(s)
    return _plain_compact(s)


def _plain_grow(s):
    """Room for each sequence's new tokens: the lowest free pages, in the order of the sequences.  A last
    page that is partly filled and shared is replaced by a copy.  All or none get theirs."""
    t, lens, refs, new, page = s["tables"].clone(), s["lens"], s["refs"].clone(), s["tokens"], s["c"]["page"]
    pool = s["pool"]
    held = (lens + page - 1) // page
    last = (lens // page).clamp_max(t.shape[1] - 1)
    old = t.gather(1, last[:, None])[:, 0].long()
    split = (new > 0) & (lens % page != 0) & (refs[old.clamp_min(0)] > 1)
    want = (lens + new + page - 1) // page - held + split.long()
    begin = want.cumsum(0) - want
    free = (refs == 0).nonzero()[:, 0]
    short = (want.sum() - free.numel()).clamp_min(0)[None]
    ok = short == 0
    col = torch.arange(t.shape[1], device=DEV)[None, :]
    first = (held - split.long())[:, None]
    fresh = (col >= first) & (col < first + want[:, None]) & ok
    rank = (begin[:, None] + col - first)[fresh]
    t[fresh] = free[rank].int()
    refs.index_add_(0, old[split & ok], -torch.ones_like(old[split & ok], dtype=torch.int32))
    refs[free[rank]] = 1
    src, dst = old[split & ok], t.gather(1, last[:, None])[:, 0].long()[split & ok]
    keep = torch.arange(page, device=DEV)[None, :, None] < (lens % page)[split & ok][:, None, None]
    pool[dst] = torch.where(keep, pool[src], pool[dst])
    return t, torch.where(ok, lens + new, lens), refs, short, pool


def _plain_fork(s):
    """Sequence i goes on from sequence parents[i]'s tokens (none where that is -1)."""
    t, lens, refs, par, page = s["tables"], s["lens"], s["refs"], s["parents"].long(), s["c"]["page"]
    some = par >= 0
    n = torch.where(some, lens[par.clamp_min(0)], torch.zeros_like(par))
    col = torch.arange(t.shape[1], device=DEV)[None, :]
    out = torch.where(col < ((n + page - 1) // page)[:, None], t[par.clamp_min(0)], torch.full_like(t, -1))
    refs = refs.clone()
    for tab, by in ((t, -1), (out, 1)):
        at = tab[tab >= 0].long()
        refs.index_add_(0, at, torch.full_like(at, by, dtype=torch.int32))
    return out, n, refs


def _plain_compact(s):
    """The k-th used page behind the first U, of U used ones, moves to the k-th free page among them."""
    t, refs, pool = s["tables"], s["refs"].clone(), s["pool"]
    at = torch.arange(refs.numel(), device=DEV)
    used = refs > 0
    many = used.sum()
    src, dst = at[used & (at >= many)], at[~used & (at < many)]
    to = at.clone()
    to[src] = dst
    pool[dst] = pool[src]
    refs[dst] = refs[src]
    refs[src] = 0
    return torch.where(t >= 0, to[t.clamp_min(0).long()].int(), t), refs, pool


# ---- what a pass cannot do without -----------------------------------------------------------

def _entry_bytes(c):
    return 2 * c["dim"] if c.get("fmt", "bf16") == "bf16" else c["dim"] - ROPE[c["dim"]] + (c["dim"] - ROPE[c["dim"]]) // 32 \
        + 2 * ROPE[c["dim"]]


def work(c):
    kind, b, d = c["kind"], c["batch"], c["dim"]
    both = _lengths(c)
    new, ends = sum(n for n, _ in both), sum(n for _, n in both)
    if kind == "append":
        size = 4 if c["x"] == "float32" else 2
        pool = c["page"] * (sum(-(-n // c["page"]) for _, n in both) + 3)
        # the new entries; with 8-bit ones, the whole pool read and its values written
        values = pool * (_entry_bytes(c) + 4 * d) if c["fmt"] == "fp8" else 0
        return {"bytes": new * (size * d + _entry_bytes(c)) + values, "flops": 3 * new * d}
    if kind == "attend":
        n, h, w, k = c["tokens"], c["heads"], c["window"], c["topk"]
        pairs = sum(min(end, k) if k else min(p + 1, w) if w else p + 1 for _, end in both for p in range(end - n, end))
        entries = sum(min(end, k) if k else min(end, w + n - 1) if w else end for _, end in both)
        return {"bytes": entries * (_entry_bytes(c) + (4 if k else 0)) + 4 * entries // c["page"] + b * n * h * (4 * d + 4),
                "flops": 4 * d * h * pairs}
    if kind == "packed":
        h, w = c["heads"], c["window"]
        pairs = sum(w * n - w * (w - 1) // 2 if w and n > w else n * (n + 1) // 2 for n, _ in both)
        return {"bytes": new * (2 * d * c["groups"] + h * (4 * d + 4)), "flops": 4 * d * h * pairs}
    state = 8 * b * (-(-(c["ctx"] + c["page"]) // c["page"])) + 16 * b + 8 * c["pages"]
    if kind == "fork":
        return {"bytes": state, "flops": b}
    if kind == "grow":
        # about two fifths of the sequences share a last page; half of it is copied
        return {"bytes": state + 2 * b * c["page"] * 2 * d // 5, "flops": b}
    used = sum(-(-n // c["page"]) for _, n in both)
    return {"bytes": state + used * max(0, c["pages"] - used) // c["pages"] * c["page"] * 4 * d, "flops": b}


# ---- the same from the definitions, in 64 bits -------------------------------------------------

def _e4m3_table():
    out = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if code & 127 == 127 else -v if code & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _exact_values(entries, c):
    if c.get("fmt", "bf16") == "bf16":
        return entries.double()
    nope = c["dim"] - ROPE[c["dim"]]
    code = _e4m3_table()[entries[:, :nope].long()]
    raw = entries[:, nope:nope + nope // 32].long().view(-1, nope // 128, 4)
    bits = raw[..., 0] | raw[..., 1] << 8 | raw[..., 2] << 16 | raw[..., 3] << 24
    scale = torch.pow(2.0, ((bits >> 23) - 127).double())  # the scales are powers of two
    raw = entries[:, nope + nope // 32:].long().view(-1, ROPE[c["dim"]], 2)
    bits = (raw[..., 0] << 16 | raw[..., 1] << 24).to(torch.int64)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
    return torch.cat([code * scale.repeat_interleave(128, 1), bits.view(torch.float32).double()], 1)


def _exact_rows(q, e, lo, hi, sink):
    """q [H, D] of one token over entries lo .. hi - 1."""
    logits = torch.cat([torch.einsum("hd,nd->hn", q, e[lo:hi]) / math.sqrt(q.shape[1]), sink[:, None]], 1)
    p = torch.softmax(logits, 1)
    return p[:, :-1] @ e[lo:hi], torch.logsumexp(logits, 1)


def _exact_many(q, e, first, window, sink):
    """Tokens at positions first, first + 1, ..: weights of unseen entries are zero."""
    t, h, d = q.shape
    outs, zs = [], []
    step = max(1, (1 << 26) // (h * max(e.shape[0], 1)))
    for i in range(0, t, step):
        n = min(step, t - i)
        hi = first + i + n
        lo = max(0, first + i + 1 - window) if window else 0
        gap = (torch.arange(n, device=DEV) + first + i)[:, None] - torch.arange(lo, hi, device=DEV)[None, :]
        hidden = (gap < 0) | (gap >= window) if window else gap < 0
        logits = torch.matmul(q[i:i + n].reshape(n * h, d), e[lo:hi].t().contiguous()).view(n, h, hi - lo) / math.sqrt(d)
        logits[hidden[:, None, :].expand_as(logits)] = -math.inf
        z = torch.logsumexp(torch.cat([logits, sink.view(1, h, 1).expand(n, h, 1)], 2), 2)
        outs.append(torch.matmul((logits - z[..., None]).exp().view(n * h, hi - lo), e[lo:hi]).view(n, h, d))
        zs.append(z)
    return torch.cat(outs), torch.cat(zs)


def exact(c, seed):
    s = prepare(c, seed)
    c = s["c"]
    kind = c["kind"]
    if kind == "append":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        vals = _exact_values(flat, c)
        x, table, page = s["x"].double(), s["tables"].cpu().tolist(), c["page"]
        at = [table[b][p // page] * page + p % page for b, (n, end) in enumerate(zip(s["new"], s["ends"]))
              for p in range(end - n, end)]
        if c["fmt"] == "bf16":
            vals[at] = x.bfloat16().double()
        else:
            nope = c["dim"] - ROPE[c["dim"]]
            grid = _e4m3_table()[:127]
            for k in range(0, nope, 128):
                blk = x[:, k:k + 128]
                need = (blk.abs().amax(1).clamp_min(float(np.float32(1e-4))) * float(np.float32(1 / 448))).float().double()
                scale = torch.pow(2.0, torch.ceil(torch.log2(need)))
                a = (blk / scale[:, None]).abs().clamp_max(448.0)
                up = torch.searchsorted(grid, a.contiguous()).clamp_max(126)
                dn = (up - 1).clamp_min(0)
                gap = (grid[up] - a) - (a - grid[dn])  # nearest; halfway to the even code
                pick = torch.where((gap > 0) | ((gap == 0) & (dn % 2 == 0)), dn, up)
                vals[at, k:k + 128] = grid[pick] * torch.sign(blk) * scale[:, None]
            vals[at, nope:] = x[:, nope:].bfloat16().double()
        return vals.view(c["pages"], page, -1)
    if kind == "attend":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        n, page = c["tokens"], c["page"]
        outs, zs = [], []
        sink = s["sinks"].double()
        for i, end in enumerate(s["ends"]):
            pos = torch.arange(end, device=DEV) if s["idx"] is None else s["idx"][i][s["idx"][i] >= 0].long()
            e = _exact_values(flat[s["tables"][i][pos // page].long() * page + pos % page], c)
            q = s["q"][i * n:(i + 1) * n].double()
            if n == 1:
                lo = max(0, e.shape[0] - c["window"]) if c["window"] else 0
                o, z = _exact_rows(q[0], e, lo, e.shape[0], sink)
                o, z = o[None], z[None]
            else:
                o, z = _exact_many(q, e, end - n, c["window"], sink)
            outs.append(o)
            zs.append(z)
        return torch.cat(outs), torch.cat(zs)
    if kind == "packed":
        outs, zs = [], []
        per = c["heads"] // c["groups"]
        for a, z in zip(s["ends"], s["ends"][1:]):
            got = [_exact_many(s["q"][a:z, g * per:(g + 1) * per].double(), s["kv"][a:z, g].double(), 0, c["window"],
                               s["sinks"][g * per:(g + 1) * per].double()) for g in range(c["groups"])]
            outs.append(torch.cat([o for o, _ in got], 1))
            zs.append(torch.cat([l for _, l in got], 1))
        return torch.cat(outs), torch.cat(zs)
    table, lens, refs, page = s["tables"].tolist(), s["lens"].tolist(), s["refs"].tolist(), c["page"]
    wide = len(table[0])
    if kind == "fork":
        new, ends = [], []
        for p in s["parents"].tolist():
            n = lens[p] if p >= 0 else 0
            keep = -(-n // page)
            new.append((table[p][:keep] if p >= 0 else []) + [-1] * (wide - keep))
            ends.append(n)
        for row, by in [(r, -1) for r in table] + [(r, 1) for r in new]:
            for p in row:
                if p >= 0:
                    refs[p] += by
        return (torch.tensor(new, dtype=torch.int32), torch.tensor(ends), torch.tensor(refs, dtype=torch.int32))
    pool = s["pool"].double()
    if kind == "grow":
        free = [p for p, r in enumerate(refs) if r == 0]
        now, wants = list(refs), []
        for b, n in enumerate(s["tokens"].tolist()):
            held, end = -(-lens[b] // page), -(-(lens[b] + n) // page)
            copy = n > 0 and lens[b] % page and now[table[b][lens[b] // page]] > 1
            wants.append((held - bool(copy), end, bool(copy)))
        missing = max(0, sum(e - f for f, e, _ in wants) - len(free))
        if not missing:
            k = 0
            for b, (f, e, copy) in enumerate(wants):
                for j in range(f, e):
                    if copy and j == f:
                        refs[table[b][j]] -= 1
                        pool[free[k], :lens[b] % page] = pool[table[b][j], :lens[b] % page]
                    table[b][j], refs[free[k]] = free[k], 1
                    k += 1
            lens = [a + n for a, n in zip(lens, s["tokens"].tolist())]
        return (torch.tensor(table, dtype=torch.int32), torch.tensor(lens), torch.tensor(refs, dtype=torch.int32),
                torch.tensor([missing]), pool)
    many = sum(r > 0 for r in refs)
    holes = iter([p for p in range(many) if refs[p] == 0])
    to = {}
    for p in range(many, len(refs)):
        if refs[p] > 0:
            to[p] = next(holes)
            pool[to[p]], refs[to[p]], refs[p] = pool[p].clone(), refs[p], 0
    return (torch.tensor([[to.get(p, p) for p in r] for r in table], dtype=torch.int32),
            torch.tensor(refs, dtype=torch.int32), pool)
