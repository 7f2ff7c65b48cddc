"""Timing cases of what a generation loop needs around its cache.

Each case is a dict of plain values; ``kind`` names the operator:

* ``attend``  attention of a sequence's newest tokens over its pages, behind a sliding window beside
  which the sequence's first tokens stay visible (``paged.attend``);
* ``packed``  the same of whole prompts, one after another in one tensor (``csa2_attn.packed``);
* ``sample``  tokens drawn from logits with temperature, top-k, top-p and min-p, and their log
  probabilities (``sampling.sample``);
* ``verify``  how many drafted tokens of each sequence stay, and the token behind them
  (``sampling.verify``);
* ``beams``   which beams go on with which token (``sampling.beams``).

Random numbers are inputs.  A token is drawn from the tokens that the filters leave, in the order of
falling logits (equal ones by rising index): the first whose running sum of probabilities exceeds the
random number.  The plain forms are elementary torch operations, those of the attention in 32 bits;
those that choose tokens in 64, since a token next to a border of the running sum has to be the right one.
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
        # one conversation that has gone on for long: few entries are seen, launches and latency count
        dict(name="attend b1 window 1k first 4", kind="attend", batch=1, ctx=40000, tokens=1, heads=128, dim=576, page=64,
             fmt="fp8", window=1024, first=4),
        # a full batch of such conversations in a model with a wide window
        dict(name="attend b32 window 4k first 64", kind="attend", batch=32, ctx=32768, tokens=1, heads=128, dim=576, page=64,
             fmt="fp8", window=4096, first=64),
        # a smaller model checks four drafted tokens a sequence; pages that end inside a tile
        dict(name="attend b24x4 d160 first 10", kind="attend", batch=24, ctx=9000, tokens=4, heads=16, dim=160, page=24,
             fmt="bf16", window=2000, first=10),
        # a step's ragged prompts in a sliding-window layer
        dict(name="packed 6 prompts window 512", kind="packed", batch=6, most=4000, heads=128, groups=1, dim=576, window=512,
             first=16),
        # one user's next token, all filters: latency
        dict(name="sample b1 131k", kind="sample", batch=1, vocab=131072, dtype="float32", top_k=50, top_p=0.95, min_p=0.0,
             temperature=0.8),
        # a step of 64 conversations, nucleus only, logits as the model's last product leaves them
        dict(name="sample b64 131k bf16", kind="sample", batch=64, vocab=131072, dtype="bfloat16", top_k=0, top_p=0.9,
             min_p=0.0, temperature=0.7),
        # the largest batch, each request with settings of its own, an odd vocabulary
        dict(name="sample b256 200k mixed", kind="sample", batch=256, vocab=200019, dtype="float32", top_k=-1, top_p=-1.0,
             min_p=-1.0, temperature=-1.0),
        # a small vocabulary in half precision, min-p alone
        dict(name="sample b16 32k f16", kind="sample", batch=16, vocab=32000, dtype="float16", top_k=0, top_p=1.0, min_p=0.05,
             temperature=1.2),
        # four tokens guessed from the text itself for each of 32 conversations
        dict(name="verify b32x5 131k bf16", kind="verify", batch=32, drafts=4, ragged=False, vocab=131072, dtype="bfloat16",
             probs=False, top_k=0, top_p=0.95, temperature=0.8),
        # a draft model's tokens with its probabilities, other numbers of them in every sequence
        dict(name="verify b12 ragged probs 50k", kind="verify", batch=12, drafts=7, ragged=True, vocab=50001, dtype="float32",
             probs=True, top_k=0, top_p=1.0, temperature=1.0),
        # a translator's search, four beams each for two sentences
        dict(name="beams 2x4 32k", kind="beams", groups=2, width=4, keep=4, vocab=32000, dtype="float32"),
        # a batch of wide searches that look at twice as many continuations, as ended ones leave
        dict(name="beams 16x8 131k bf16", kind="beams", groups=16, width=8, keep=16, vocab=131072, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "packed", "packed", "sample", "sample", "sample", "verify", "verify", "beams"])
    if kind == "attend":
        fmt = rng.choice(["fp8", "fp8", "bf16"])
        batch = _log(rng, 1, 96)
        return dict(kind=kind, batch=batch, ctx=_log(rng, 30, min(131072, (1 << 19) // batch)), tokens=rng.choice([1, 1, 1, 2, 5]),
                    heads=rng.choice([1, 5, 8, 16, 32, 64, 128, 128]),
                    dim=rng.choice([160, 576, 576] if fmt == "fp8" else [64, 96, 128, 160, 256, 512, 576]),
                    page=rng.choice([1, 7, 16, 24, 32, 64, 100, 128]), fmt=fmt, window=_log(rng, 1, 8000), first=_log(rng, 1, 300))
    if kind == "packed":
        heads, groups = rng.choice([(1, 1), (3, 1), (8, 1), (8, 2), (16, 1), (24, 3), (32, 1), (64, 1), (128, 1)])
        batch = _log(rng, 1, 40)
        return dict(kind=kind, batch=batch, most=_log(rng, 4, 8000 // batch), heads=heads, groups=groups,
                    dim=rng.choice([64, 96, 128, 160, 256, 512, 576, 576, 576]), window=_log(rng, 1, 1000), first=_log(rng, 1, 100))
    dtype = rng.choice(["float32", "float32", "bfloat16", "bfloat16", "float16"])
    vocab = _log(rng, 100, 262144)
    if kind == "beams":
        groups, width = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 6, 8, 16])
        return dict(kind=kind, groups=groups, width=width, keep=width * rng.choice([1, 1, 2]),
                    vocab=max(100, min(vocab, (1 << 25) // (groups * width))), dtype=dtype)
    filters = dict(top_k=rng.choice([0, 0, 1, _log(rng, 2, 2000)]), top_p=rng.choice([1.0, 1.0, 0.95, rng.uniform(0.05, 0.999)]),
                   temperature=rng.choice([1.0, rng.uniform(0.2, 2.0), 0.0]))
    if kind == "verify":
        batch, drafts = _log(rng, 1, 64), rng.choice([1, 2, 3, 4, 7])
        return dict(kind=kind, batch=batch, drafts=drafts, ragged=rng.random() < 0.5,
                    vocab=max(100, min(vocab, (1 << 25) // (batch * (drafts + 1)))), dtype=dtype, probs=rng.random() < 0.5, **filters)
    batch = _log(rng, 1, 256)
    vocab = max(100, min(vocab, (1 << 25) // batch))
    if rng.random() < 0.3:
        return dict(kind=kind, batch=batch, vocab=vocab, dtype=dtype, top_k=-1, top_p=-1.0, min_p=-1.0, temperature=-1.0)
    return dict(kind=kind, batch=batch, vocab=vocab, dtype=dtype, min_p=rng.choice([0.0, 0.0, 0.1, rng.uniform(0.001, 0.5)]), **filters)


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


def _values(e, c):
    """Entries -> the float32 values that they stand for."""
    if c["fmt"] == "bf16":
        return e.float()
    nope = c["dim"] - ROPE[c["dim"]]
    nb = nope // 128
    val = e[..., :nope].contiguous().view(torch.float8_e4m3fn).float().unflatten(-1, (nb, 128))
    scale = e[..., nope:nope + 4 * nb].contiguous().view(torch.float32)
    tail = e[..., nope + 4 * nb:].contiguous().view(torch.bfloat16).float()
    return torch.cat([(val * scale[..., None]).flatten(-2), tail], -1)


# ---- inputs -------------------------------------------------------------------------------

def _rnd(seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)
    return (lambda *shape: torch.randn(*shape, generator=gen, device=DEV)), (lambda *shape: torch.rand(*shape, generator=gen, device=DEV))


def _lengths(c):
    """A case's lengths, the longest its largest size."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    if c["kind"] == "verify":
        n = c["drafts"]
        return [n] + [rng.randint(0, n) if c["ragged"] else n for _ in range(c["batch"] - 1)]
    lo, hi = (max(c["tokens"], c["ctx"] // 4), max(c["tokens"], c["ctx"])) if c["kind"] == "attend" else (1, c["most"])
    return [hi] + [rng.randint(lo, hi) for _ in range(c["batch"] - 1)]


def _tables(c, rng, lens):
    """Each sequence's pages, scattered over the pool as after hours of use; -1 behind them."""
    page = c["page"]
    free = list(range(c["pages"]))
    rng.shuffle(free)
    out = np.full((len(lens), -(-(max(lens) + page) // page)), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        for j in range(-(-n // page)):
            out[b, j] = free.pop()
    return torch.from_numpy(out).to(DEV)


def _pool(c, randn):
    """Every entry of the pool filled: what earlier conversations left there, and what is read."""
    n, page, dim = c["pages"], c["page"], c["dim"]
    if c["fmt"] == "bf16":
        out = torch.empty(n * page, dim, dtype=torch.bfloat16, device=DEV)
    else:
        nope = dim - ROPE[dim]
        out = torch.empty(n * page, nope + nope // 32 + 2 * ROPE[dim], dtype=torch.uint8, device=DEV)
    for i in range(0, n * page, 65536):
        x = randn(min(65536, n * page - i), dim).bfloat16()
        out[i:i + 65536] = x if out.dtype == torch.bfloat16 else _pack_fp8(x, ROPE[dim])
    return out.view(n, page, -1)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def _logits(c, rows, randn, rand):
    """A model's logits: a broad bulk, in some rows flatter than in others, and a few tokens that the
    text makes likely."""
    v = c["vocab"]
    x = randn(rows, v) * (1.0 + 2.0 * rand(rows, 1))
    at = (rand(rows, 24) * v).long().clamp_max(v - 1)
    return x.scatter_add_(1, at, 12.0 * rand(rows, 24)).to(getattr(torch, c["dtype"]))


def _settings(c, rows, rng):
    """The filters: one for all rows, or (-1) one for each, some of them off."""
    def each(name, options, off, dtype):
        v = c.get(name, off)
        if v >= 0:
            return v if v != off else None
        return torch.tensor([rng.choice(options) for _ in range(rows)], dtype=dtype, device=DEV)
    return dict(temperature=each("temperature", [0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.5], 1.0, torch.float32),
                top_k=each("top_k", [0, 0, 1, 20, 40, 50, 1000], 0, torch.int32),
                top_p=each("top_p", [1.0, 0.8, 0.9, 0.95, 0.99], 1.0, torch.float32),
                min_p=each("min_p", [0.0, 0.0, 0.02, 0.1], 0.0, torch.float32))


def prepare(c, seed):
    rng = random.Random(seed * 104729 + 11)
    randn, rand = _rnd(seed)
    c = dict(c)
    s = dict(c=c)
    kind = c["kind"]
    if kind == "attend":
        lens, b = _lengths(c), c["batch"]
        rng.shuffle(lens)
        c["pages"] = sum(-(-n // c["page"]) for n in lens) + 5
        s.update(pool=_pool(c, randn), tables=_tables(c, rng, lens), lens=_i64(lens), ends=lens,
                 q=randn(b * c["tokens"], c["heads"], c["dim"]).bfloat16(), sinks=randn(c["heads"]),
                 cu=None if c["tokens"] == 1 else _i64([i * c["tokens"] for i in range(b + 1)]))
    elif kind == "packed":
        lens = _lengths(c)
        rng.shuffle(lens)
        cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
        s.update(q=randn(cu[-1], c["heads"], c["dim"]).bfloat16(), kv=randn(cu[-1], c["groups"], c["dim"]).bfloat16(),
                 sinks=randn(c["heads"]), cu=_i64(cu), ends=cu)
    elif kind == "sample":
        s.update(logits=_logits(c, c["batch"], randn, rand), u=rand(c["batch"]), **_settings(c, c["batch"], rng))
    elif kind == "verify":
        drafts = _lengths(c)
        rng.shuffle(drafts)
        cu = np.concatenate([[0], np.cumsum([n + 1 for n in drafts])]).tolist()
        t = cu[-1]
        x = _logits(c, t, randn, rand)
        # the draft guesses like the model, not quite: a sharper one's most likely tokens, or a noisy one's draws
        noise = -torch.log(-torch.log(rand(t, c["vocab"]).clamp(1e-30, 1 - 1e-7)))
        near = x.float() + 0.5 * randn(t, c["vocab"])
        best = (near + (noise if c["probs"] else 0.5 * noise)).argmax(1)
        tokens = torch.cat([best[:1], best[:-1]])  # row i is token i's; it predicts the next
        s.update(logits=x, tokens=tokens, cu=_i64(cu), ends=cu, u=rand(t), draw=rand(c["batch"]),
                 probs=torch.softmax(near, 1) if c["probs"] else None, **_settings(c, t, rng))
    else:
        rows = c["groups"] * c["width"]
        s.update(logits=_logits(c, rows, randn, rand), scores=-20.0 * rand(rows))
    return s


# ---- the operators ------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from mzoo_amd import csa2_attn, paged, sampling
    c = s["c"]
    kind = c["kind"]
    if kind == "attend":
        return paged.attend(s["q"], s["pool"], s["tables"], s["lens"], cu=s["cu"], window=c["window"], first=c["first"],
                            sinks=s["sinks"], rope=ROPE.get(c["dim"], 0))
    if kind == "packed":
        return csa2_attn.packed(s["q"], s["kv"], s["cu"], window=c["window"], first=c["first"], sinks=s["sinks"])
    if kind == "beams":
        return sampling.beams(s["logits"], s["scores"], c["width"], c["keep"])
    filters = dict(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if kind == "sample":
        return sampling.sample(s["logits"], s["u"], **filters)
    return sampling.verify(s["logits"], s["tokens"], s["cu"], s["u"], s["draw"], draft_probs=s["probs"], **filters)


def _softmax_rows(q, e, seen, sink):
    """q [T, H, D], e [N, D], seen bool [T, N], sink [H] -> (o [T, H, D], lse [T, H])."""
    t, h, d = q.shape
    sc = (q.reshape(t * h, d) @ e.t()).view(t, h, -1) * d ** -0.5
    sc = sc.masked_fill_(~seen[:, None, :], float("-inf"))
    m = torch.maximum(sc.amax(-1), sink)
    w = sc.sub_(m[..., None]).exp_()
    total = w.sum(-1) + (sink - m).exp()
    o = (w.view(t * h, -1) @ e).view(t, h, d) / total[..., None]
    return o, m + total.log()


def _causal(q, e, start, window, first, sink):
    """Tokens at positions start, start + 1, .. over entries 0 .. of their sequence, in blocks that
    bound the scores' memory: the last ``window`` positions and the ``first`` of all."""
    t, h, d = q.shape
    o, z = torch.empty(t, h, d, device=DEV), torch.empty(t, h, device=DEV)
    step = max(1, min(t, (1 << 26) // (h * min(e.shape[0], 2 * window + first))))
    for i in range(0, t, step):
        n = min(step, t - i)
        pos = start + torch.arange(i, i + n, device=DEV)[:, None]
        lo = max(0, start + i - window + 1)
        col = torch.cat([torch.arange(min(first, lo), device=DEV), torch.arange(lo, start + i + n, device=DEV)])
        seen = (col <= pos) & ((col > pos - window) | (col < first))
        o[i:i + n], z[i:i + n] = _softmax_rows(q[i:i + n], e[col], seen, sink)
    return o, z


def _kept(x, temperature, top_k, top_p, min_p):
    """Rows of logits -> (their tokens by falling logit, weights in that order, 0 where a filter drops
    them, the weights before the filters).  A filter is a number, a tensor [rows] or None."""
    rows, v = x.shape

    def col(f, off):
        f = off if f is None else f
        return f.double()[:, None] if torch.is_tensor(f) else torch.full((rows, 1), float(np.float32(f)), dtype=torch.float64, device=DEV)
    l, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    t = col(temperature, 1.0)
    greedy = t <= 0
    w = ((l.double() - l[:, :1].double()) / torch.where(greedy, 1.0, t)).exp()
    at = torch.arange(v, device=DEV)[None, :]
    k = col(top_k, 0)
    k = torch.where(greedy, 1.0, torch.where(k > 0, k, float(v)))
    kept = torch.where(at < k, w, 0.0)
    sums = kept.cumsum(1)
    p = col(top_p, 1.0)
    before = sums - kept
    kept = torch.where((p >= 1) | (at == 0) | (before < p * sums[:, -1:]), kept, 0.0)
    kept = torch.where((at == 0) | (w >= col(min_p, 0.0)), kept, 0.0)
    return order, kept, w


def _drawn(order, w, u):
    """The first token of the order whose running sum exceeds u of the whole, and its place there."""
    sums = w.cumsum(1)
    at = (sums <= u.double()[:, None] * sums[:, -1:]).sum(1, keepdim=True).clamp_max(w.shape[1] - 1)
    return order.gather(1, at)[:, 0], at


def _filters(s, rows=None):
    f = [s["temperature"], s["top_k"], s["top_p"], s["min_p"]]
    return f if rows is None else [x[rows] if torch.is_tensor(x) else x for x in f]


def _run_plain(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "attend":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        o, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=DEV)
        n, page = c["tokens"], c["page"]
        for i, end in enumerate(s["ends"]):
            pos = torch.arange(end, device=DEV)
            e = _values(flat[s["tables"][i].long()[pos // page] * page + pos % page], c)
            o[i * n:(i + 1) * n], lse[i * n:(i + 1) * n] = _causal(s["q"][i * n:(i + 1) * n].float(), e, end - n, c["window"],
                                                                   c["first"], s["sinks"])
        return o, lse
    if kind == "packed":
        o, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=DEV)
        per = c["heads"] // c["groups"]
        for a, z in zip(s["ends"], s["ends"][1:]):
            for g in range(c["groups"]):
                hs = slice(g * per, (g + 1) * per)
                o[a:z, hs], lse[a:z, hs] = _causal(s["q"][a:z, hs].float(), s["kv"][a:z, g].float(), 0, c["window"], c["first"],
                                                   s["sinks"][hs])
        return o, lse
    if kind == "sample":
        tokens, logprobs = [], []
        step = max(1, (1 << 24) // c["vocab"])
        for i in range(0, c["batch"], step):
            order, kept, _ = _kept(s["logits"][i:i + step], *_filters(s, slice(i, i + step)))
            tok, at = _drawn(order, kept, s["u"][i:i + step])
            tokens.append(tok)
            logprobs.append((kept.gather(1, at)[:, 0] / kept.sum(1)).log().float())
        return torch.cat(tokens), torch.cat(logprobs)
    if kind == "verify":
        return _plain_verify(s)
    l = s["logits"].double()
    m = l.amax(1, keepdim=True)
    val = s["scores"].double()[:, None] + (l - m) - (l - m).exp().sum(1, keepdim=True).log()
    g, w, v = c["groups"], c["width"], c["vocab"]
    val, at = torch.sort(val.view(g, w * v), dim=1, descending=True, stable=True)
    val, at = val[:, :c["keep"]], at[:, :c["keep"]]
    parents = at // v + torch.arange(g, device=DEV)[:, None] * w
    return parents.int().flatten(), (at % v).flatten(), val.float().flatten()


def _plain_verify(s):
    c, cu = s["c"], s["cu"]
    t, b, v = s["logits"].shape[0], c["batch"], c["vocab"]
    row = torch.arange(t, device=DEV)
    tested = torch.ones(t, dtype=torch.bool, device=DEV)
    tested[cu[1:] - 1] = False  # a sequence's last row predicts what nobody drafted
    drafted = torch.where(tested, s["tokens"].roll(-1), 0)
    p = torch.empty(t, v, dtype=torch.float64, device=DEV)  # the target's probabilities, by token
    step = max(1, (1 << 24) // v)
    for i in range(0, t, step):
        order, kept, _ = _kept(s["logits"][i:i + step], *_filters(s, slice(i, i + step)))
        p[i:i + step].scatter_(1, order, kept / kept.sum(1, keepdim=True))
    q = s["probs"][row, drafted].double() if s["probs"] is not None else 1.0
    refused = tested & ~(s["u"].double() * q < p[row, drafted])
    accepted = torch.empty(b, dtype=torch.int64, device=DEV)
    at = torch.empty(b, dtype=torch.int64, device=DEV)
    for i, (a, z) in enumerate(zip(s["ends"], s["ends"][1:])):
        accepted[i] = torch.where(refused[a:z], row[a:z] - a, z - 1 - a).amin()
    at = cu[:-1] + accepted
    no = refused[at]
    rest = p[at]
    if s["probs"] is not None:
        # what the target has above the draft, by rising token; where nothing is left, the target itself
        less = (rest - s["probs"][at].double()).clamp_min(0.0)
        above = less.sum(1, keepdim=True) > 0
        by_token = no[:, None] & above
        rest = torch.where(by_token, less, rest)
    else:
        by_token = torch.zeros_like(no)[:, None]
        rest = torch.where(no[:, None] & (torch.arange(v, device=DEV)[None, :] == drafted[at][:, None]), 0.0, rest)
    order = torch.sort(s["logits"][at].float(), dim=1, descending=True, stable=True).indices
    order = torch.where(by_token, torch.arange(v, device=DEV)[None, :], order)
    return accepted, _drawn(order, rest.gather(1, order), s["draw"])[0]


# ---- what a pass cannot do without -----------------------------------------------------------

def _seen(window, first, start, n):
    """(entries that n tokens from position start on read, pairs of a token and an entry that it sees)"""
    lo = max(0, start - window + 1)
    pairs = sum(min(p + 1, window) + min(first, max(0, p - window + 1)) for p in range(start, start + n))
    return start + n - lo + min(first, lo), pairs


def work(c):
    kind = c["kind"]
    if kind in ("attend", "packed"):
        d, h = c["dim"], c["heads"]
        lens = _lengths(c)
        news = [c["tokens"] if kind == "attend" else n for n in lens]
        both = [_seen(c["window"], c["first"], n - new, new) for n, new in zip(lens, news)]
        size = 2 * d * c.get("groups", 1)
        if c.get("fmt") == "fp8":
            size = d - ROPE[d] + (d - ROPE[d]) // 32 + 2 * ROPE[d]
        return {"bytes": sum(e for e, _ in both) * size + sum(news) * h * (4 * d + 4), "flops": 4 * d * h * sum(n for _, n in both)}
    size = 4 if c["dtype"] == "float32" else 2
    v = c["vocab"]
    if kind == "sample":
        return {"bytes": c["batch"] * (v * size + 16), "flops": 4 * c["batch"] * v}
    if kind == "verify":
        rows = sum(n + 1 for n in _lengths(c))
        # with the draft's probabilities: most sequences refuse a token, and read a row of them
        return {"bytes": rows * (v * size + 16) + (c["batch"] * v * 4 if c["probs"] else 0) + 16 * c["batch"], "flops": 4 * rows * v}
    rows = c["groups"] * c["width"]
    return {"bytes": rows * (v * size + 4) + c["groups"] * c["keep"] * 16, "flops": 4 * rows * v}


# ---- the same from the definitions, in 64 bits -------------------------------------------------

def _e4m3_table():
    out = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(math.nan if code & 127 == 127 else -v if code & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=DEV)


def _exact_values(entries, c):
    if c["fmt"] == "bf16":
        return entries.double()
    nope = c["dim"] - ROPE[c["dim"]]
    code = _e4m3_table()[entries[:, :nope].long()]
    raw = entries[:, nope:nope + nope // 32].long().view(-1, nope // 128, 4)
    bits = raw[..., 0] | raw[..., 1] << 8 | raw[..., 2] << 16 | raw[..., 3] << 24
    scale = torch.pow(2.0, ((bits >> 23) - 127).double())  # the scales are powers of two
    tail = entries[:, nope + nope // 32:].contiguous().view(torch.bfloat16)
    return torch.cat([code * scale.repeat_interleave(128, 1), tail.double()], 1)


def _exact_many(q, e, start, window, first, sink):
    """Tokens at positions start, start + 1, ..: weights of unseen entries are zero."""
    t, h, d = q.shape
    outs, zs = [], []
    step = max(1, (1 << 25) // (h * min(max(e.shape[0], 1), 2 * window + first)))
    for i in range(0, t, step):
        n = min(step, t - i)
        hi = start + i + n
        lo = max(0, start + i + 1 - window)
        at = torch.tensor([*range(min(first, lo)), *range(lo, hi)], device=DEV)
        gap = (torch.arange(n, device=DEV) + start + i)[:, None] - at[None, :]
        hidden = (gap < 0) | (gap >= window) & (at >= first)[None, :]
        logits = torch.matmul(q[i:i + n].reshape(n * h, d), e[at].t().contiguous()).view(n, h, len(at)) / math.sqrt(d)
        logits[hidden[:, None, :].expand_as(logits)] = -math.inf
        z = torch.logsumexp(torch.cat([logits, sink.view(1, h, 1).expand(n, h, 1)], 2), 2)
        outs.append(torch.matmul((logits - z[..., None]).exp().view(n * h, len(at)), e[at]).view(n, h, d))
        zs.append(z)
    return torch.cat(outs), torch.cat(zs)


def _number(f, i, off):
    return off if f is None else float(f[i]) if torch.is_tensor(f) else float(np.float32(f))


def _exact_log_probs(s, i):
    """Log probabilities of row i's tokens behind the filters, by token, and the tokens by falling probability."""
    x = s["logits"][i].double()
    t = _number(s["temperature"], i, 1.0)
    order = torch.argsort(-x, stable=True)
    lp = torch.log_softmax(x / (t if t > 0 else 1.0), 0)[order]
    n = x.numel()
    k = int(_number(s["top_k"], i, 0))
    n = min(n, k) if k > 0 else n
    n = n if t > 0 else 1
    p = _number(s["top_p"], i, 1.0)
    if p < 1:
        share = (lp[:n] - torch.logsumexp(lp[:n], 0)).exp().cumsum(0)
        n = min(n, int((share < p).sum()) + 1)
    least = _number(s["min_p"], i, 0.0)
    if least > 0:
        n = max(1, min(n, int((lp - lp[0] >= math.log(least)).sum())))
    out = torch.full_like(x, -math.inf)
    out[order[:n]] = lp[:n] - torch.logsumexp(lp[:n], 0)
    return out, order


def _exact_draw(probs, order, u):
    share = probs[order].cumsum(0)
    # behind the last token that has any weight the running sum stays; u is below 1
    return int(order[min(int((share <= u * float(share[-1])).sum()), probs.numel() - 1)])


def exact(c, seed):
    s = prepare(c, seed)
    c = s["c"]
    kind = c["kind"]
    if kind == "attend":
        flat = s["pool"].view(-1, s["pool"].shape[-1])
        n, page = c["tokens"], c["page"]
        outs, zs = [], []
        for i, end in enumerate(s["ends"]):
            pos = torch.arange(end, device=DEV)
            e = _exact_values(flat[s["tables"][i][pos // page].long() * page + pos % page], c)
            o, z = _exact_many(s["q"][i * n:(i + 1) * n].double(), e, end - n, c["window"], c["first"], s["sinks"].double())
            outs.append(o)
            zs.append(z)
        return torch.cat(outs), torch.cat(zs)
    if kind == "packed":
        outs, zs = [], []
        per = c["heads"] // c["groups"]
        for a, z in zip(s["ends"], s["ends"][1:]):
            got = [_exact_many(s["q"][a:z, g * per:(g + 1) * per].double(), s["kv"][a:z, g].double(), 0, c["window"], c["first"],
                               s["sinks"][g * per:(g + 1) * per].double()) for g in range(c["groups"])]
            outs.append(torch.cat([o for o, _ in got], 1))
            zs.append(torch.cat([l for _, l in got], 1))
        return torch.cat(outs), torch.cat(zs)
    if kind == "sample":
        tokens, logprobs = [], []
        for i, u in enumerate(s["u"].tolist()):
            lp, order = _exact_log_probs(s, i)
            tokens.append(_exact_draw(lp.exp(), order, u))
            logprobs.append(float(lp[tokens[-1]]))
        return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)
    if kind == "verify":
        accepted, chosen = [], []
        tokens, u, draw = s["tokens"].tolist(), s["u"].tolist(), s["draw"].tolist()
        for b, (a, z) in enumerate(zip(s["ends"], s["ends"][1:])):
            for i in range(a, z):
                lp, order = _exact_log_probs(s, i)
                p = lp.exp()
                if i == z - 1:
                    break
                d = tokens[i + 1]
                q = s["probs"][i].double() if s["probs"] is not None else torch.zeros_like(p).index_fill_(0, torch.tensor([d], device=DEV), 1.0)
                if u[i] * float(q[d]) < float(p[d]):
                    continue
                left = (p - q).clamp_min(0.0)
                if s["probs"] is not None and float(left.sum()) > 0:
                    p, order = left, torch.arange(p.numel(), device=DEV)
                elif s["probs"] is None:
                    p = left
                break
            accepted.append(i - a)
            chosen.append(_exact_draw(p, order, draw[b]))
        return torch.tensor(accepted), torch.tensor(chosen)
    parents, tokens, values = [], [], []
    for g in range(c["groups"]):
        rows = range(g * c["width"], (g + 1) * c["width"])
        every = torch.cat([torch.log_softmax(s["logits"][i].double(), 0) + s["scores"][i].double() for i in rows])
        best = torch.argsort(-every, stable=True)[:c["keep"]]
        parents.append(best // c["vocab"] + rows[0])
        tokens.append(best % c["vocab"])
        values.append(every[best])
    return torch.cat(parents).int(), torch.cat(tokens), torch.cat(values)
