"""GPU: the paged latent cache -- entries into pages, attention over them, growing, forking, compacting --
against plain restatements in 64 bits (bounds: ``tests/ragged_ref.py``) and the CPU quantizer."""

import numpy as np
import pytest
import torch

from mzoo_amd import paged
from oracle import quant as OQ
from tests import ragged_ref as R

pytestmark = pytest.mark.gpu
ROPE = {576: 64, 160: 32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _entries(pool, dim):
    """[P * page, D] float64 values of a pool, on the CPU."""
    flat = pool.reshape(-1, pool.shape[-1]).cpu()
    if pool.dtype == torch.bfloat16:
        return flat.double()
    rope = ROPE[dim]
    return torch.from_numpy(OQ.unpack_latent_fp8_b128(flat.numpy(), dim - rope, rope)).double()


def _setup(dev, lens, page, dim, fmt, seed, spare=3, width=None, poison=True):
    """Scattered pages holding random latents; everything else in the pool is NaN."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            tables[b, j] = perm.pop()
    rope = ROPE.get(dim, 64)
    pool = paged.new_pool(pages, page, dim, fmt, rope=rope, device=dev)
    if poison:
        if fmt == "bf16":
            pool.fill_(float("nan"))
        else:
            pool.fill_(0xff)
    tables = tables.to(dev)
    n64 = torch.tensor(lens, dtype=torch.int64, device=dev)
    x = torch.randn(sum(lens), dim, generator=g).bfloat16().to(dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
    if sum(lens):
        paged.append(pool, tables, n64, x, cu=cu, rope=rope)
    return pool, tables, n64, x, cu


def _of(tables, b, n, page):
    return [int(tables[b, p // page]) * page + p % page for p in range(n)]


# ---- append -------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("dim,fmt,page", [(576, "fp8", 64), (160, "fp8", 7), (576, "bf16", 16), (96, "bf16", 1), (8, "bf16", 5)])
def test_append_packed(dev, dim, fmt, page, dtype):
    g = _gen(dim + page)
    rope = ROPE.get(dim, 0)
    new, lens = [5, 0, 1, 70, 3], [5, 9, 40, 100, 3]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    perm = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((5, max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            tables[b, j] = perm.pop()
    tables[3, 0] = pages + 4                       # no such page: its tokens are skipped
    x = (4 * torch.randn(sum(new) + 2, dim + 16, generator=g)).to(dtype)[:, :dim]  # rows of a wider tensor; two of no sequence
    if fmt == "fp8":
        x[0, :dim - rope] = 0
        x[2, 3] = float("inf")
        x[3, 5] = float("nan")
    pool = paged.new_pool(pages, page, dim, fmt, rope=rope, device=dev)
    pool.fill_(7)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int64)
    want = pool.cpu().reshape(pages * page, -1)
    vals = x if fmt == "bf16" else torch.from_numpy(OQ.pack_latent_fp8_b128(x.float().numpy(), dim - rope))
    for b, (n, end) in enumerate(zip(new, lens)):
        for i in range(n):
            pid = int(tables[b, (end - n + i) // page])
            if 0 <= pid < pages:
                v = vals[int(cu[b]) + i]
                want[pid * page + (end - n + i) % page] = v.bfloat16() if fmt == "bf16" else v
    wide = torch.empty(x.shape[0], dim + 16, dtype=dtype, device=dev)
    wide[:, :dim] = x.to(dev)
    paged.append(pool, tables.to(dev), torch.tensor(lens).to(dev), wide[:, :dim], cu=cu.to(dev), rope=rope)
    got = pool.cpu().reshape(pages * page, -1)
    if fmt == "bf16":
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
        return
    # a NaN's code is 0x7f or 0xff (the sign of inf / inf is the machine's): equal in value, and byte
    # for byte in every entry without one
    gv, wv = (OQ.unpack_latent_fp8_b128(t.numpy(), dim - rope, rope) for t in (got, want))
    assert np.array_equal(gv, wv, equal_nan=True)
    fine = torch.from_numpy(np.isfinite(wv).all(-1))
    assert int((~fine).sum()) == 2 and torch.equal(got[fine], want[fine])


def test_append_one_token_each(dev):
    lens, page = [1, 0, 64, 65, 200], 32
    pool, tables, n64, x, cu = _setup(dev, lens, page, 576, "fp8", 3)
    new = torch.randn(5, 576, generator=_gen(4)).bfloat16()
    before = pool.cpu().reshape(-1, 656)
    paged.append(pool, tables, n64, new.to(dev))
    for b, n in enumerate(lens):                  # a sequence of no tokens writes nothing
        if n:
            before[int(tables[b, (n - 1) // page]) * page + (n - 1) % page] = torch.from_numpy(
                OQ.pack_latent_fp8_b128(new[b:b + 1].float().numpy()))[0]
    assert torch.equal(pool.cpu().reshape(-1, 656), before)


# ---- attend -------------------------------------------------------------------------------

def _check_attend(dev, lens, tokens, heads, dim, fmt, page, window, seed, sinks=True, workspace=None):
    """tokens: new tokens of each sequence (an int: one each, without cu)."""
    print(f"attend: lens {lens} tokens {tokens} heads {heads} dim {dim} {fmt} page {page} window {window}", flush=True)
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, fmt, seed)
    g = _gen(seed + 1)
    one = isinstance(tokens, int)
    new = [1] * len(lens) if one else tokens
    q = torch.randn(sum(new), heads, dim, generator=g).bfloat16().to(dev)
    sk = torch.randn(heads, generator=g).to(dev) if sinks else None
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int64, device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=None if one else cu, window=window, sinks=sk, rope=ROPE.get(dim, 64),
                          workspace=workspace)
    vals = _entries(pool, dim).to(dev)
    t = tables.cpu()
    for b, (n, end) in enumerate(zip(new, lens)):
        if n == 0:
            continue
        at = int(cu[b])
        e = vals[_of(t, b, end, page)]
        pos = (end - n + torch.arange(n))[:, None]
        col = torch.arange(end)[None, :]
        seen = (col <= pos) & (col > pos - (window or 1 << 40))
        R.check(o[at:at + n], lse[at:at + n], R.attend(q[at:at + n], e, seen.to(dev), sk), f"sequence {b}")
    return o, lse


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (512, "bf16"), (160, "fp8"), (160, "bf16"), (64, "bf16"),
                                     (96, "bf16"), (128, "bf16"), (256, "bf16")])
@pytest.mark.parametrize("heads", [1, 16, 128])
def test_attend_lengths(dev, dim, fmt, heads):
    _check_attend(dev, [1, 0, 31, 32, 33, 65, 190], 1, heads, dim, fmt, 16, None, dim + heads)


@pytest.mark.parametrize("heads", [3, 40, 64, 72, 200])
@pytest.mark.parametrize("page", [1, 24, 64, 100])
def test_attend_heads_and_pages(dev, heads, page):
    _check_attend(dev, [130, 2, 1000], 1, heads, 576, "fp8", page, None, heads + page, sinks=heads % 2 == 0)


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (160, "bf16")])
@pytest.mark.parametrize("window", [1, 2, 33, 500])
def test_attend_window(dev, dim, fmt, window):
    _check_attend(dev, [1, 40, 33, 700], 1, 64, dim, fmt, 24, window, window)
    _check_attend(dev, [3, 40, 33, 700], [3, 0, 7, 5], 16, dim, fmt, 24, window, window + 1)


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (512, "bf16"), (160, "bf16"), (64, "bf16")])
@pytest.mark.parametrize("heads", [1, 2, 5, 16, 64, 128])
def test_attend_several_tokens(dev, dim, fmt, heads):
    _check_attend(dev, [4, 100, 64, 37, 260, 9], [4, 1, 33, 0, 70, 12], heads, dim, fmt, 32, None, heads + dim)  # one with more tokens than entries


@pytest.mark.parametrize("heads,lens", [(128, [9000]), (64, [20000, 1, 3000]), (16, [5000] * 7), (128, [70, 6000, 40, 12345])])
def test_attend_long(dev, heads, lens):
    """Sequences long enough to be split and joined."""
    _check_attend(dev, lens, 1, heads, 576, "fp8", 64, None, len(lens))
    _check_attend(dev, [n + 3 for n in lens], [3] * len(lens), heads, 160, "bf16", 24, None, len(lens) + 5)


@pytest.mark.parametrize("fmt", ["fp8", "bf16"])
@pytest.mark.parametrize("k", [1, 37, 512, 2048])
def test_attend_list(dev, fmt, k):
    """Lists in any order, with empty, foreign and repeated positions (a position twice counts twice)."""
    lens, page, heads = [1, 0, 50, 5000], 48, 72
    pool, tables, n64, _, _ = _setup(dev, lens, page, 576, fmt, k)
    g = _gen(k + 1)
    idx = torch.randint(-3, 5200, (4, k), generator=g).int()
    idx[3, :k // 2] = torch.randint(0, 5000, (k // 2,), generator=g).int()
    idx[0, k // 3] = 0
    q = torch.randn(4, heads, 576, generator=g).bfloat16().to(dev)
    wide = torch.full((4, k + 5), 7, dtype=torch.int32, device=dev)  # rows of a wider tensor
    wide[:, :k] = idx.to(dev)
    for sinks in (None, torch.randn(heads, generator=g).to(dev)):
        o, lse = paged.attend(q, pool, tables, n64, indices=wide[:, :k], sinks=sinks)
        vals = _entries(pool, 576).to(dev)
        t = tables.cpu()
        for b, n in enumerate(lens):
            sel = [int(i) for i in idx[b] if 0 <= i < n]
            at = _of(t, b, n, page)
            e = vals[[at[i] for i in sel]] if sel else vals[:0]
            seen = torch.ones(1, len(sel), dtype=torch.bool, device=dev)
            R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], e, seen, sinks), f"sequence {b}")


def test_attend_bad_pages(dev):
    """Positions on no page are empty; a sequence of nothing but such pages sees nothing."""
    lens, page = [400, 300, 64], 32
    pool, tables, n64, _, _ = _setup(dev, lens, page, 576, "fp8", 11)
    tables[0, 0], tables[0, 5], tables[0, 12] = -1, pool.shape[0], 2 ** 31 - 1
    tables[1, :] = -7
    tables[2, 0] = -1
    q = torch.randn(3, 128, 576, generator=_gen(12)).bfloat16().to(dev)
    sinks = torch.randn(128, generator=_gen(13)).to(dev)
    o, lse = paged.attend(q, pool, tables, n64, sinks=sinks)
    vals, t = _entries(pool, 576).to(dev), tables.cpu()
    for b, n in enumerate(lens):
        at = [a for p, a in enumerate(_of(t, b, n, page)) if 0 <= int(t[b, p // page]) < pool.shape[0]]
        seen = torch.ones(1, len(at), dtype=torch.bool, device=dev)
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], vals[at] if at else vals[:0], seen, sinks), f"sequence {b}")
    assert torch.equal(o[1], torch.zeros_like(o[1])) and torch.equal(lse[1], sinks)


@pytest.mark.parametrize("dim", [576, 160])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attend_unseen_entries_do_not_reach(dev, dim, bad):
    """An entry that is not finite reaches the tokens that see it and no other."""
    lens, new, page, heads = [90, 40], [6, 3], 16, 16
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, "bf16", 21)
    t = tables.cpu()
    flat = pool.view(-1, dim)
    flat[_of(t, 0, 90, page)[87], 5] = bad
    flat[_of(t, 1, 40, page)[30], 9] = bad        # behind the window of the last two
    q = torch.randn(9, heads, dim, generator=_gen(22)).bfloat16().to(dev)
    cu = torch.tensor([0, 6, 9], device=dev)
    for window in (None, 8):
        o, lse = paged.attend(q, pool, tables, n64, cu=cu, window=window)
        for b in range(2):
            for i in range(new[b]):
                pos = lens[b] - new[b] + i
                lo = max(0, pos - window + 1) if window else 0
                hit = lo <= (87 if b == 0 else 30) <= pos
                row = o[int(cu[b]) + i]
                if hit:
                    assert not bool(torch.isfinite(row).all())
                else:
                    e = flat[_of(t, b, pos + 1, page)[lo:]].double()
                    seen = torch.ones(1, pos + 1 - lo, dtype=torch.bool, device=dev)
                    R.check(row[None], lse[int(cu[b]) + i][None], R.attend(q[int(cu[b]) + i][None], e, seen, None), f"{b} {i}")


@pytest.mark.parametrize("scale", [0.0, 30.0, 1e4])
def test_attend_wide_scores(dev, scale):
    """Scores that rise by hundreds along the sequence, or are all alike."""
    lens, page, heads = [3000, 200], 64, 64
    pool, tables, n64, x, cu = _setup(dev, lens, page, 576, "bf16", 31)
    q = torch.randn(2, heads, 576, generator=_gen(32)).bfloat16().to(dev)
    flat, t = pool.view(-1, 576), tables.cpu()
    for b, n in enumerate(lens):
        at = _of(t, b, n, page)
        ramp = torch.linspace(-scale, scale, n, device=dev)[:, None]
        flat[at] = (ramp * q[b, 3].float()[None, :] / 24.0).bfloat16()
    o, lse = paged.attend(q, pool, tables, n64)
    for b, n in enumerate(lens):
        e = flat[_of(t, b, n, page)].double()
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], e, torch.ones(1, n, dtype=torch.bool, device=dev), None), f"{b}")


def test_attend_far_pages(dev):
    """Entries past 2^32 bytes of the pool."""
    page, pages = 64, 120000                      # 5.0 GB
    pool = paged.new_pool(pages, page, 576, "fp8", device=dev)
    lens = [300, 64]
    tables = torch.full((2, 8), -1, dtype=torch.int32)
    tables[0, :5] = torch.tensor([pages - 1, 0, 102305, 51153, pages - 2])
    tables[1, 0] = 102304
    tables = tables.to(dev)
    n64 = torch.tensor(lens, device=dev)
    x = torch.randn(364, 576, generator=_gen(41)).bfloat16().to(dev)
    cu = torch.tensor([0, 300, 364], device=dev)
    paged.append(pool, tables, n64, x, cu=cu)
    q = torch.randn(2, 16, 576, generator=_gen(42)).bfloat16().to(dev)
    o, lse = paged.attend(q, pool, tables, n64)
    for b, n in enumerate(lens):
        e = torch.from_numpy(OQ.unpack_latent_fp8_b128(OQ.pack_latent_fp8_b128(x[int(cu[b]):int(cu[b]) + n].float().cpu().numpy())))
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], e.to(dev), torch.ones(1, n, dtype=torch.bool, device=dev), None), f"{b}")


def test_attend_rows_of_no_sequence(dev):
    pool, tables, n64, _, _ = _setup(dev, [50, 70], 16, 160, "bf16", 51)
    q = torch.randn(9, 8, 160, generator=_gen(52)).bfloat16().to(dev)
    cu = torch.tensor([0, 2, 5], device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=cu)
    assert torch.equal(o[5:], torch.zeros_like(o[5:])) and bool((lse[5:] == float("-inf")).all())
    out, l2 = torch.full_like(o, 3.0), torch.full_like(lse, 4.0)
    paged.attend(q, pool, tables, n64, cu=cu, out=out, lse=l2)
    assert torch.equal(out[:5], o[:5]) and torch.equal(l2[:5], lse[:5])
    assert bool((out[5:] == 3.0).all()) and bool((l2[5:] == 4.0).all())


def test_attend_padded_batch_and_other_stream(dev):
    """Sequences of length 0 among others; the call on a stream of its own, twice at once."""
    lens = [2000, 0, 1, 0, 900]
    pool, tables, n64, _, _ = _setup(dev, lens, 32, 576, "fp8", 61)
    q = torch.randn(2, 5, 128, 576, generator=_gen(62)).bfloat16().to(dev)
    want = [paged.attend(q[i], pool, tables, n64) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(paged.attend(q[i], pool, tables, n64))
    torch.cuda.synchronize()
    for (a, b), (c, d) in zip(want, got):
        assert torch.equal(a, c) and torch.equal(b, d)
        assert bool((a[1] == 0).all()) and bool((b[3] == float("-inf")).all())


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (512, "bf16")])
@pytest.mark.parametrize("heads", [1, 2, 15, 16, 17, 31, 32, 33])
def test_attend_few_heads(dev, dim, fmt, heads):
    """One token of few heads: whole, split and joined, behind a window."""
    _check_attend(dev, [1, 0, 31, 32, 33, 370], 1, heads, dim, fmt, 16, None, heads)
    _check_attend(dev, [6000, 1, 900], 1, heads, dim, fmt, 64, None, heads + 1, sinks=heads % 2 == 0)
    _check_attend(dev, [600, 3, 900], 1, heads, dim, fmt, 24, 500, heads + 2)


@pytest.mark.parametrize("heads,dim,fmt", [(4, 576, "fp8"), (128, 576, "fp8"), (16, 160, "bf16")])
def test_attend_many_sequences(dev, heads, dim, fmt):
    """More sequences than lanes: their units found together, split where one of them is long."""
    g = _gen(heads)
    lens = torch.randint(0, 90, (70,), generator=g).tolist()
    lens[40] = 4000
    _check_attend(dev, lens, 1, heads, dim, fmt, 32, None, heads)
    new = torch.randint(0, 4, (70,), generator=g).tolist()
    _check_attend(dev, lens, [min(a, b) for a, b in zip(new, lens)], heads, dim, fmt, 32, None, heads + 1)
    _check_attend(dev, [n % 9 + 1 for n in range(1100)], 1, min(heads, 8), dim, fmt, 8, None, heads + 2)  # too many to split
    _check_attend(dev, [n % 9 + 2 for n in range(1100)], [n % 3 for n in range(1100)], min(heads, 8), dim, fmt, 8, None, heads + 3)


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (160, "bf16")])
@pytest.mark.parametrize("heads", [3, 40])
def test_attend_long_runs_of_no_page(dev, dim, fmt, heads):
    """Chunks of entry codes of which none is there, before, between and behind others, in one unit (so many
    sequences are not split)."""
    page, lens = 64, [9000, 8000] + [1] * 520
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, fmt, 14)
    tables[0, :70] = -1
    tables[0, 75:130] = -1
    tables[1, 2:] = -1
    q = torch.randn(522, heads, dim, generator=_gen(15)).bfloat16().to(dev)
    o, lse = paged.attend(q, pool, tables, n64, rope=ROPE[dim])
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    for b in (0, 1, 2, 521):
        at = [a for p, a in enumerate(_of(t, b, lens[b], page)) if int(t[b, p // page]) >= 0]
        seen = torch.ones(1, len(at), dtype=torch.bool, device=dev)
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], vals[at], seen, None), f"sequence {b}")


@pytest.mark.parametrize("blocks", [128, 129, 256, 257, 512, 513])
@pytest.mark.parametrize("dim", [576, 64])
def test_attend_splits_by_blocks(dev, blocks, dim):
    """Either side of the numbers of blocks at which a call is split otherwise, one sequence long enough for it."""
    lens = [n % 5 for n in range(blocks)]
    lens[blocks // 3] = 16 * blocks + 40
    _check_attend(dev, lens, 1, 3, dim, "bf16", 16, None, blocks)


@pytest.mark.parametrize("heads,new", [(16, None), (20, None), (64, None), (16, [5, 2]), (1, [40, 2])])
@pytest.mark.parametrize("dim", [576, 160])
def test_attend_unseen_entries_of_shares(dev, dim, heads, new):
    """An entry that is not finite, in one share of a long sequence: the tokens that see it, and no other."""
    lens, page = [3000, 40], 64
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, "bf16", 25)
    t, flat = tables.cpu(), pool.view(-1, dim)
    count = new or [1, 1]
    flat[_of(t, 0, 3000, page)[2998 if new else 2100], 5] = float("nan")   # the second last token's, or an old one
    q = torch.randn(sum(count), heads, dim, generator=_gen(26)).bfloat16().to(dev)
    cu = torch.tensor([0, count[0], sum(count)], device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=cu if new else None)
    for b in range(2):
        for i in range(count[b]):
            pos, at = lens[b] - count[b] + i, int(cu[b]) + i
            if b == 0 and pos >= (2998 if new else 2100):
                assert not bool(torch.isfinite(o[at]).all(-1).any())
                continue
            e = flat[_of(t, b, pos + 1, page)].double()
            seen = torch.ones(1, pos + 1, dtype=torch.bool, device=dev)
            R.check(o[at:at + 1], lse[at:at + 1], R.attend(q[at:at + 1], e, seen, None), f"{b} {i}")


@pytest.mark.parametrize("heads", [8, 24, 64])
@pytest.mark.parametrize("scale", [30.0, 1e4])
@pytest.mark.parametrize("down", [False, True])
def test_attend_wide_scores_of_shares(dev, heads, scale, down):
    """As test_attend_wide_scores, for few heads too, rising or falling, split and whole."""
    lens, page = [3000, 300], 64
    for dim in (576, 160):
        pool, tables, n64, x, cu = _setup(dev, lens, page, dim, "bf16", 33)
        q = torch.randn(2, heads, dim, generator=_gen(34)).bfloat16().to(dev)
        flat, t = pool.view(-1, dim), tables.cpu()
        for b, n in enumerate(lens):
            ramp = torch.linspace(-scale, scale, n, device=dev)[:, None]
            flat[_of(t, b, n, page)] = ((-ramp if down else ramp) * q[b, 3].float()[None, :] / 24.0).bfloat16()
        for last in (n64, n64.clamp(max=300)):
            for tab in (tables, tables[:, :5].contiguous()):
                o, lse = paged.attend(q, pool, tab, last)
                for b in range(2):
                    n = min(int(last[b]), tab.shape[1] * page)
                    e = flat[_of(t, b, n, page)].double()
                    R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], e, torch.ones(1, n, dtype=torch.bool, device=dev), None), f"{b}")


def test_attend_nothing(dev):
    """No tokens; no sequences; a window wider than anything; tokens that no sequence holds."""
    pool, tables, n64, _, _ = _setup(dev, [50, 70], 16, 576, "fp8", 53)
    q = torch.randn(5, 40, 576, generator=_gen(54)).bfloat16().to(dev)
    o, lse = paged.attend(q[:0], pool, tables, n64, cu=torch.tensor([0, 0, 0], device=dev))
    assert o.shape == (0, 40, 576) and lse.shape == (0, 40)
    for none in (paged.attend(q, pool, tables[:0], n64[:0], cu=torch.tensor([0], device=dev)),
                 paged.attend(q, pool, tables, n64, cu=torch.tensor([0, 0, 0], device=dev))):
        assert bool((none[0] == 0).all()) and bool((none[1] == float("-inf")).all())
    cu = torch.tensor([0, 2, 5], device=dev)
    want = paged.attend(q, pool, tables, n64, cu=cu)
    for window in (70, 2 ** 30, 2 ** 62, 2 ** 64 + 1):
        got = paged.attend(q, pool, tables, n64, cu=cu, window=window)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attend_shares_in_a_graph(dev):
    """A captured call over split sequences, replayed with other lengths, tables and queries, and with
    eager calls of the same workspace between the replays."""
    lens, page, heads = [5000, 40, 2500], 32, 16
    pool, tables, n64, _, _ = _setup(dev, lens, page, 576, "fp8", 63)
    q = torch.randn(3, heads, 576, generator=_gen(64)).bfloat16().to(dev)
    ws = torch.empty(paged.attend_workspace_bytes(3, heads, 576, 3, False), dtype=torch.uint8, device=dev)
    out, lse = torch.empty_like(q), torch.empty(3, heads, device=dev)
    s_q, s_t, s_n = q.clone(), tables.clone(), n64.clone()
    paged.attend(s_q, pool, s_t, s_n, workspace=ws, out=out, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(s_q, pool, s_t, s_n, workspace=ws, out=out, lse=lse)
    for i, order in enumerate(([0, 1, 2], [2, 0, 1], [1, 1, 0], [0, 2, 2])):
        s_t.copy_(tables[order])
        s_n.copy_((n64[order] - 7 * i).clamp(min=0))
        s_q.copy_(q.roll(i, 1))
        want = paged.attend(s_q, pool, s_t, s_n)
        paged.attend(q, pool, tables, n64, workspace=ws)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


# ---- the pages ----------------------------------------------------------------------------

def _grow_ref(tables, lens, refs, new, page, pool):
    tables, lens, refs, pool = tables.clone(), lens.clone(), refs.clone(), pool.clone()
    free = [p for p in range(len(refs)) if refs[p] == 0]
    plan, over = [], 0
    for b, n in enumerate(new.tolist()):
        held, end = -(-int(lens[b]) // page), -(-(int(lens[b]) + n) // page)
        if n == 0:
            plan.append((0, 0, False))
            continue
        if end > tables.shape[1]:
            over += end - tables.shape[1]
            plan.append((0, 0, False))
            continue
        cow = bool(int(lens[b]) % page) and 0 <= tables[b, held - 1] < len(refs) and int(refs[tables[b, held - 1]]) > 1
        plan.append((held - cow, end, cow))
    lack = over + max(0, sum(e - f for f, e, _ in plan) - len(free))
    if lack:
        return tables, lens, refs, lack, pool
    now = refs.clone()
    for b, (f, e, cow) in enumerate(plan):
        for j in range(f, e):
            p = free.pop(0)
            if cow and j == f:
                src = int(tables[b, j])
                refs[src] -= 1
                pool[p, :int(lens[b]) % page] = pool[src, :int(lens[b]) % page]
            tables[b, j], refs[p] = p, 1
    return tables, lens + new, refs, 0, pool


def _book(seed, batch, page, pages, most, width, shared=True):
    """A random consistent state: (tables, lens, refs)."""
    g = _gen(seed)
    lens = torch.randint(0, most + 1, (batch,), generator=g)
    perm = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((batch, width), -1, dtype=torch.int32)
    for b in range(batch):
        if shared and b and b % 3 == 0:
            tables[b], lens[b] = tables[b - 1], lens[b - 1]
            continue
        for j in range(-(-int(lens[b]) // page)):
            tables[b, j] = perm.pop()
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in tables[tables >= 0].tolist():
        refs[p] += 1
    return tables, lens, refs


@pytest.mark.parametrize("batch,page,pages,most", [(1, 16, 20, 40), (7, 1, 500, 30), (64, 16, 5000, 300), (300, 64, 20000, 2000)])
@pytest.mark.parametrize("inplace", [False, True])
def test_grow(dev, batch, page, pages, most, inplace):
    width = -(-most // page) + 2
    tables, lens, refs = _book(batch, batch, page, pages, most, width)
    new = torch.randint(0, 3, (batch,), generator=_gen(5)) * torch.randint(0, page + 1, (batch,), generator=_gen(6)) // 2
    pools = [torch.randn(pages, page, 24, generator=_gen(7)).bfloat16(), torch.randint(0, 256, (pages, page, 12), generator=_gen(8)).byte()]
    want = [_grow_ref(tables, lens, refs, new, page, p) for p in pools]
    d = [t.to(dev) for t in (tables, lens, refs)]
    dp = [p.to(dev) for p in pools]
    got = paged.grow(*d, new.to(dev), page, pools=dp, out=d if inplace else None)
    for a, b in zip(got[:3], want[0][:3]):
        assert torch.equal(a.cpu(), b)
    assert int(got[3]) == want[0][3] == 0
    for a, w in zip(dp, want):
        assert torch.equal(a.cpu(), w[4])
    if not inplace:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(d, (tables, lens, refs)))


@pytest.mark.parametrize("inplace", [False, True])
def test_grow_short_changes_nothing(dev, inplace):
    tables, lens, refs = _book(3, 8, 16, 40, 60, 6)
    for new in (torch.full((8,), 400), torch.tensor([0, 0, 90, 0, 0, 0, 0, 0])):  # too few pages; past the table
        pool = torch.randn(40, 16, 8, generator=_gen(9))
        want = _grow_ref(tables, lens, refs, new, 16, pool)
        d = [t.to(dev) for t in (tables, lens, refs)]
        dp = pool.to(dev)
        got = paged.grow(*d, new.to(dev), 16, pools=[dp], out=d if inplace else None)
        assert int(got[3]) == want[3] > 0
        for a, b in zip(got[:3], (tables, lens, refs)):
            assert torch.equal(a.cpu(), b)
        assert torch.equal(dp.cpu(), pool)


@pytest.mark.parametrize("batch,rows,page,pages,most", [(1, 1, 16, 20, 40), (9, 9, 1, 800, 40), (64, 64, 16, 5000, 300), (5, 20, 16, 900, 200),
                                                        (30, 4, 16, 900, 200)])
@pytest.mark.parametrize("inplace", [False, True])
def test_fork(dev, batch, rows, page, pages, most, inplace):
    if inplace and batch != rows:
        pytest.skip("in place: as many rows out as in")
    width = -(-most // page) + 1
    tables, lens, refs = _book(batch, batch, page, pages, most, width)
    refs[:3] += 2                                 # pages that something else holds too
    for b in range(batch):                        # a page held beyond the tokens is given back
        j = -(-int(lens[b]) // page)
        free = (refs == 0).nonzero()
        if b % 4 == 1 and j < width and len(free):
            tables[b, j] = free[0, 0]
            refs[free[0, 0]] = 1
    par = torch.randint(-1, batch, (rows,), generator=_gen(11)).int()
    par[-1] = batch + 3
    want_t = torch.full((rows, width), -1, dtype=torch.int32)
    want_l, want_r = torch.zeros(rows, dtype=torch.int64), refs.clone()
    for p in tables[tables >= 0].tolist():
        want_r[p] -= 1
    for i, p in enumerate(par.tolist()):
        if 0 <= p < batch:
            n = -(-int(lens[p]) // page)
            want_t[i, :n], want_l[i] = tables[p, :n], lens[p]
    for p in want_t[want_t >= 0].tolist():
        want_r[p] += 1
    d = [t.to(dev) for t in (tables, lens, refs)]
    got = paged.fork(*d, par.to(dev), page, out=d if inplace else None)
    for a, b in zip(got, (want_t, want_l, want_r)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("batch,page,pages,most", [(1, 16, 20, 40), (7, 1, 500, 30), (64, 16, 9000, 900), (2, 16, 4096, 100), (3, 16, 8192, 20000),
                                                   (4, 16, 7, 0)])
@pytest.mark.parametrize("inplace", [False, True])
def test_compact(dev, batch, page, pages, most, inplace):
    tables, lens, refs = _book(batch + 1, batch, page, pages, most, -(-most // page) + 1)
    refs[-2:] += 1                                # held by something else only
    pool = torch.randn(pages, page, 8, generator=_gen(12))
    used = (refs > 0).nonzero()[:, 0].tolist()
    u = len(used)
    holes = [p for p in range(u) if refs[p] == 0]
    to = dict(zip([p for p in used if p >= u], holes))
    want_r, want_p, want_t = refs.clone(), pool.clone(), tables.clone()
    for a, b in to.items():
        want_r[b], want_r[a], want_p[b] = refs[a], 0, pool[a]
        want_t[tables == a] = b
    d = [t.to(dev) for t in (tables, refs)]
    dp = pool.to(dev)
    got = paged.compact(*d, pools=[dp], out=d if inplace else None)
    assert torch.equal(got[0].cpu(), want_t) and torch.equal(got[1].cpu(), want_r) and torch.equal(dp.cpu(), want_p)


def test_grow_and_compact_many_pools(dev):
    """More pools than one launch takes, of different entries."""
    tables, lens, refs = _book(4, 12, 16, 400, 100, 9)
    new = torch.randint(0, 20, (12,), generator=_gen(5))
    pools = [torch.randint(0, 256, (400, 16, 4 * (1 + i % 5)), generator=_gen(i)).byte() for i in range(35)]
    want = [_grow_ref(tables, lens, refs, new, 16, p) for p in pools]
    assert want[0][3] == 0
    dp = [p.to(dev) for p in pools]
    got = paged.grow(*[t.to(dev) for t in (tables, lens, refs)], new.to(dev), 16, pools=dp)
    for a, w in zip(dp, want):
        assert torch.equal(a.cpu(), w[4])
    moved = paged.compact(got[0], got[2], pools=dp)
    t, m = got[0].cpu(), moved[0].cpu()
    for b in range(12):
        for j in range(-(-int(got[1][b]) // 16)):
            for a, w in zip(dp, want):
                assert torch.equal(a[int(m[b, j])].cpu(), w[4][int(t[b, j])])
    used = int((moved[1] > 0).sum())
    assert bool((moved[1][:used] > 0).all()) and used == int((got[2] > 0).sum())


# ---- together -----------------------------------------------------------------------------

def test_a_captured_loop_of_steps(dev):
    """grow, append and attend in one captured step, replayed across page boundaries with eager
    work between the replays, after a fork: every step equals the eager one and the plain attention."""
    page, pages, heads, steps = 16, 400, 64, 20
    lens = [30, 5, 47, 0]
    pool, tables, n64, x, cu = _setup(dev, lens, page, 576, "fp8", 71, spare=300, width=12)
    pages = pool.shape[0]
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in tables[tables >= 0].cpu().tolist():
        refs[p] += 1
    refs = refs.to(dev)
    hist = [x[int(cu[b]):int(cu[b]) + n] for b, n in enumerate(lens)]
    tables, n64, refs = paged.fork(tables, n64, refs, torch.tensor([0, 2, 2, 0], dtype=torch.int32, device=dev), page)
    hist = [hist[0], hist[2], hist[2], hist[0]]
    g = _gen(72)
    kv = torch.randn(steps, 4, 576, generator=g).bfloat16().to(dev)
    q = torch.randn(steps, 4, heads, 576, generator=g).bfloat16().to(dev)
    sinks = torch.randn(heads, generator=g).to(dev)
    ones = torch.tensor([1, 1, 1, 1], device=dev)
    missing = torch.zeros(1, dtype=torch.int64, device=dev)
    s_kv, s_q = kv[0].clone(), q[0].clone()
    state = (tables, n64, refs)
    ws = torch.empty(paged.workspace_bytes(4, 12, pages), dtype=torch.uint8, device=dev)
    aws = torch.empty(paged.attend_workspace_bytes(4, heads, 576, 4, False), dtype=torch.uint8, device=dev)
    o, lse = torch.empty_like(s_q), torch.empty(4, heads, device=dev)

    def step():
        paged.grow(*state, ones, page, pools=[pool], out=state, missing=missing, workspace=ws)
        paged.append(pool, tables, n64, s_kv)
        paged.attend(s_q, pool, tables, n64, sinks=sinks, workspace=aws, out=o, lse=lse)

    keep = [t.clone() for t in (*state, pool)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, k in zip((*state, pool), keep):
        t.copy_(k)
    for i in range(steps):
        s_kv.copy_(kv[i])
        s_q.copy_(q[i])
        before = [t.clone() for t in (*state, pool)]
        graph.replay()
        after = [t.clone() for t in (*state, pool, o, lse)]
        torch.cuda.synchronize()
        assert int(missing) == 0
        for t, k in zip((*state, pool), before):
            t.copy_(k)
        step()
        for a, t in zip(after, (*state, pool, o, lse)):
            assert torch.equal(a.view(torch.uint8) if a.dtype == torch.bfloat16 else a, t.view(torch.uint8) if t.dtype == torch.bfloat16 else t)
        for b in range(4):
            hist[b] = torch.cat([hist[b], kv[i, b:b + 1]])
            e = torch.from_numpy(OQ.unpack_latent_fp8_b128(OQ.pack_latent_fp8_b128(hist[b].float().cpu().numpy()))).to(dev)
            seen = torch.ones(1, e.shape[0], dtype=torch.bool, device=dev)
            R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[i, b:b + 1], e, seen, sinks), f"step {i} sequence {b}")
    moved = paged.compact(tables, refs, pools=[pool])
    o2, _ = paged.attend(s_q, pool, moved[0], n64, sinks=sinks)
    assert torch.equal(o2, o)
