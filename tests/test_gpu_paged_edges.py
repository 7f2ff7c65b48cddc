"""GPU: the paged cache at its edges, against plain restatements."""

import numpy as np
import pytest
import torch

from mzoo_amd import _lib, paged
from tests import ragged_ref as R
from tests.test_gpu_paged import ROPE, _entries, _gen, _of, _setup

pytestmark = pytest.mark.gpu


# ---- grow: pages behind the tokens --------------------------------------------------------------

def _counts(tables, pages):
    return torch.bincount(tables[tables >= 0].long().cpu(), minlength=pages).int()


@pytest.mark.parametrize("inplace", [False, True])
def test_grow_after_refused_tokens(dev, inplace):
    """Four drafted tokens a step that cross a page's end, all refused again: the row keeps its second page."""
    page, pages = 16, 6
    tables = torch.full((2, 4), -1, dtype=torch.int32, device=dev)
    tables[0, 0] = 0
    lens = torch.tensor([14, 0], device=dev)
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    refs[0] = 1
    pool = torch.randn(pages, page, 4, device=dev)
    four = torch.tensor([4, 0], device=dev)
    for _ in range(6):
        state = (tables, lens, refs)
        tables, lens, refs, missing = paged.grow(*state, four, page, pools=[pool], out=state if inplace else None)
        assert int(missing) == 0 and lens.tolist() == [18, 0]
        assert tables.tolist() == [[0, 1, -1, -1], [-1] * 4]
        assert torch.equal(refs.cpu(), _counts(tables, pages))
        lens = lens - torch.tensor([4, 0], device=dev)


def _grow_kept(tables, lens, refs, new, page, pool):
    """grow where rows may hold pages behind their tokens: a row's own ones are used first, those that others
    hold too are given up."""
    tables, lens, refs, pool = tables.clone(), lens.clone(), refs.clone(), pool.clone()
    pages, width = refs.numel(), tables.shape[1]
    free = [p for p in range(pages) if refs[p] == 0]
    plan, over = [], 0
    for b, n in enumerate(new.tolist()):
        held, end = -(-int(lens[b]) // page), -(-(int(lens[b]) + n) // page)
        fresh, gone, copy = [], [], None
        if n > 0 and end > width:
            over += end - width
        elif n > 0:
            if int(lens[b]) % page:
                p = int(tables[b, held - 1])
                if 0 <= p < pages and refs[p] > 1:
                    fresh, gone, copy = [held - 1], [p], p
            for j in range(held, end):
                p = int(tables[b, j])
                count = int(refs[p]) if 0 <= p < pages else 0
                if count != 1:
                    fresh.append(j)
                if count > 1:
                    gone.append(p)
        plan.append((fresh, gone, copy))
    lack = over + max(0, sum(len(f) for f, _, _ in plan) - len(free))
    if lack:
        return tables, lens, refs, lack, pool
    for b, (fresh, gone, copy) in enumerate(plan):
        for i, j in enumerate(fresh):
            p = free.pop(0)
            tables[b, j], refs[p] = p, 1
            if i == 0 and copy is not None:
                pool[p, :int(lens[b]) % page] = pool[copy, :int(lens[b]) % page]
        for p in gone:
            refs[p] -= 1
    return tables, lens + new, refs, 0, pool


def _rolled_back(seed, batch, page, pages, most, spare):
    """Consistent rows of which many hold pages behind their tokens, some of them shared."""
    g = _gen(seed)
    width = -(-most // page) + 4
    perm = torch.randperm(pages - spare, generator=g).tolist()
    tables = torch.full((batch, width), -1, dtype=torch.int32)
    lens = torch.randint(0, most + 1, (batch,), generator=g)
    for b in range(batch):
        if b and b % 3 == 0:
            tables[b], lens[b] = tables[b - 1], lens[b - 1]
        else:
            for j in range(-(-int(lens[b]) // page)):
                tables[b, j] = perm.pop()
    for b in range(0, batch, 2):
        lens[b] = int(torch.randint(0, int(lens[b]) + 1, (1,), generator=g))
        held = -(-int(lens[b]) // page)
        if b % 4 == 0 and held + 2 < width and tables[b, held] >= 0:
            tables[b, held + 1] = -1              # a hole among them
    return tables, lens, _counts(tables, pages)


@pytest.mark.parametrize("batch,page,most", [(2, 16, 60), (9, 1, 300), (40, 4, 1500), (150, 16, 900)])
@pytest.mark.parametrize("inplace", [False, True])
def test_grow_uses_the_pages_that_a_row_holds(dev, batch, page, most, inplace):
    pages = batch * (-(-most // page)) + 40
    tables, lens, refs = _rolled_back(batch + page, batch, page, pages, most, 30)
    new = torch.randint(0, most // 2, (batch,), generator=_gen(3)) * torch.randint(0, 2, (batch,), generator=_gen(4))
    new = torch.minimum(new, tables.shape[1] * page - lens)
    pool = torch.randn(pages, page, 4, generator=_gen(5))
    want = _grow_kept(tables, lens, refs, new, page, pool)
    assert want[3] == 0 and torch.equal(want[2], _counts(want[0], pages))
    d, dp = [t.to(dev) for t in (tables, lens, refs)], pool.to(dev)
    got = paged.grow(*d, new.to(dev), page, pools=[dp], out=d if inplace else None)
    assert int(got[3]) == 0
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a.cpu(), b)
    assert torch.equal(dp.cpu(), want[4])


def test_grow_needs_no_free_page_for_a_row_that_holds_one(dev):
    tables = torch.tensor([[2, 0, -1], [1, 3, -1]], dtype=torch.int32, device=dev)
    lens, refs = torch.tensor([6, 16], device=dev), torch.ones(4, dtype=torch.int32, device=dev)
    got = paged.grow(tables, lens, refs, torch.tensor([6, 0], device=dev), 8)
    assert int(got[3]) == 0 and torch.equal(got[0], tables) and got[1].tolist() == [12, 16] and torch.equal(got[2], refs)
    got = paged.grow(tables, lens, refs, torch.tensor([12, 1], device=dev), 8)      # two pages lack
    assert int(got[3]) == 2 and torch.equal(got[0], tables) and torch.equal(got[1], lens) and torch.equal(got[2], refs)


# ---- attend -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (160, "bf16")])
@pytest.mark.parametrize("lens", [[50, 1, 0], [5000, 40, 0]])
def test_attend_empty_list(dev, dim, fmt, lens):
    """A list of no positions: every token sees nothing."""
    pool, tables, n64, _, _ = _setup(dev, lens, 16, dim, fmt, 81)
    q = torch.randn(3, 24, dim, generator=_gen(82)).bfloat16().to(dev)
    sinks = torch.randn(24, generator=_gen(83)).to(dev)
    for idx in (torch.empty(3, 0, dtype=torch.int32, device=dev), torch.zeros(3, 7, dtype=torch.int32, device=dev)[:, :0]):
        o, lse = paged.attend(q, pool, tables, n64, indices=idx, sinks=sinks, rope=ROPE[dim])
        assert bool((o == 0).all()) and torch.equal(lse, sinks.expand(3, 24))
        o, lse = paged.attend(q, pool, tables, n64, indices=idx, rope=ROPE[dim])
        assert bool((o == 0).all()) and bool((lse == float("-inf")).all())


def test_no_pages_and_no_columns(dev):
    """A pool of no pages, or tables of no columns: nothing is written, and tokens see nothing."""
    q = torch.randn(2, 8, 576, generator=_gen(84)).bfloat16().to(dev)
    x, sinks = q[:, 0].contiguous(), torch.randn(8, generator=_gen(85)).to(dev)
    lens = torch.tensor([3, 40], device=dev)
    some = paged.new_pool(4, 16, 576, device=dev)
    cu = torch.tensor([0, 1, 2], device=dev)
    for pool, tables in ((some, torch.empty(2, 0, dtype=torch.int32, device=dev)),
                         (paged.new_pool(0, 16, 576, device=dev), torch.zeros(2, 3, dtype=torch.int32, device=dev))):
        for c in (None, cu):
            paged.append(pool, tables, lens, x, cu=c)
            o, lse = paged.attend(q, pool, tables, lens, cu=c, sinks=sinks)
            assert bool((o == 0).all()) and torch.equal(lse, sinks.expand(2, 8))
        o, lse = paged.attend(q, pool, tables, lens, indices=torch.zeros(2, 5, dtype=torch.int32, device=dev))
        assert bool((o == 0).all()) and bool((lse == float("-inf")).all())
    assert bool((some == 0).all())


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (160, "fp8"), (160, "bf16")])
@pytest.mark.parametrize("window", [None, 1, 4, 100])
@pytest.mark.parametrize("width", [5, 100])
def test_attend_past_the_table(dev, dim, fmt, window, width):
    """Sequences longer than their table: a token stays at its own position, and the entries past the
    table are on no page."""
    page = 16
    room = width * page
    lens = [room + 5, room, room - 1, room + 3, room + 130, room + 40, 20]
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, fmt, width)
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    sinks = torch.randn(16, generator=_gen(86)).to(dev)
    for new in (None, [4, 2, 3, 4, 1, 70, 20]):
        count = new or [1] * len(lens)
        q = torch.randn(sum(count), 16, dim, generator=_gen(87)).bfloat16().to(dev)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(count)]), device=dev)
        o, lse = paged.attend(q, pool, tables[:, :width], n64, cu=cu if new else None, window=window, sinks=sinks, rope=ROPE[dim])
        for b, (n, end) in enumerate(zip(count, lens)):
            a, e = int(cu[b]), vals[_of(t, b, min(end, room), page)]
            pos, col = (end - n + torch.arange(n))[:, None], torch.arange(min(end, room))[None, :]
            seen = (col <= pos) & (col > pos - (window or 1 << 40))
            R.check(o[a:a + n], lse[a:a + n], R.attend(q[a:a + n], e, seen.to(dev), sinks), f"sequence {b} of {n}")


@pytest.mark.parametrize("dim", [576, 64])
@pytest.mark.parametrize("window", [None, 3])
def test_attend_lengths_past_any_table(dev, dim, window):
    """Lengths beyond 32 bits, over a table of 64 entries."""
    pool, tables, _, _, _ = _setup(dev, [64, 64, 64], 16, dim, "bf16", 91)
    q = torch.randn(6, 8, dim, generator=_gen(92)).bfloat16().to(dev)
    cu = torch.tensor([0, 2, 4, 6], device=dev)
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    for far in ([2 ** 31, 2 ** 33 + 5, 2 ** 62], [66, 2 ** 31 - 1, 2 ** 32 + 64]):
        o, lse = paged.attend(q, pool, tables, torch.tensor(far, device=dev), cu=cu, window=window)
        for b in range(3):
            pos, col = (far[b] - 2 + torch.arange(2))[:, None], torch.arange(64)[None, :]
            seen = (col > pos - (window or 1 << 63)) if window else torch.ones(2, 64, dtype=torch.bool)
            R.check(o[2 * b:2 * b + 2], lse[2 * b:2 * b + 2],
                    R.attend(q[2 * b:2 * b + 2], vals[_of(t, b, 64, 16)], seen.to(dev), None), f"{far[b]}")


@pytest.mark.parametrize("dim,fmt,chunk", [(576, "bf16", 1280), (512, "bf16", 1280), (576, "fp8", 2048), (160, "bf16", 512)])
def test_attend_hidden_entries_of_a_later_chunk(dev, dim, fmt, chunk):
    """32 tokens in one unit (so many sequences are not split) behind a window that ends in the first tile of a
    second chunk of entries.  Of the unit's first tile only the first token's entry is there, so the
    others' exponents start from 0; the entries that tokens 1 to 3 see score -200, the later ones of
    that last tile, hidden from them, 0."""
    n, window, first = 32, chunk, 64
    end = first + window + n - 1
    lens = [end] + [1] * 520
    pool, tables, n64, _, _ = _setup(dev, lens, 1, dim, fmt, 95, poison=False)
    g = _gen(96)
    base = torch.zeros(dim)
    base[:16] = 4.0                                              # in 8-bit entries these channels are exact
    ends = torch.randn(end, dim, generator=g) * 0.25
    ends[:, :16] = 0.0
    ends[:first + window + 3] -= 200.0 * dim ** 0.5 / (base @ base) * base
    ends[first, :16] = 0.0
    sub = tables[:1].clone()
    paged.append(pool, sub, n64[:1], ends.bfloat16().to(dev), cu=torch.tensor([0, end], device=dev), rope=ROPE.get(dim, 64))
    tables[0, first + 1:first + 32] = -1
    q = torch.zeros(n + 520, 1, dim)
    q[:n, 0] = base
    q[n:] = torch.randn(520, 1, dim, generator=g)
    q = q.bfloat16().to(dev)
    cu = torch.tensor([0] + list(range(n, n + 521)), device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=cu, window=window, rope=ROPE.get(dim, 64))
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    there = (t[0] >= 0)[:end]
    pos, col = (end - n + torch.arange(n))[:, None], torch.arange(end)[None, :]
    seen = (col <= pos) & (col > pos - window) & there[None, :]
    at = t[0, :end].clamp(min=0).long()
    R.check(o[:n], lse[:n], R.attend(q[:n], vals[at.to(dev)], seen.to(dev), None), "the window's sequence")


def test_attend_more_than_2_30_entries(dev):
    """A sequence of 2^30 + 65536 entries (its table names two pages again and again) without a window: its first
    entry, the only one whose score is not 0, counts."""
    page, dim, heads = 65536, 64, 2
    width = (1 << 30) // page + 1
    n = width * page
    pool = torch.zeros(2, page, dim, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(1, heads, dim, dtype=torch.bfloat16, device=dev)
    q[:, :, 0] = 8.0
    pool[0, 0, 0], pool[0, 0, 1] = 20.75, 3.0                    # score 8 * 20.75 / 8, about log(n)
    tables = torch.ones(1, width, dtype=torch.int32, device=dev)
    tables[0, 0] = 0
    weight = np.exp(20.75) / (np.exp(20.75) + n - 1)
    want = torch.tensor([20.75 * weight, 3.0 * weight], dtype=torch.float64)
    lens = torch.tensor([n], device=dev)
    for window in (None, n, n - 1):
        o, lse = paged.attend(q, pool, tables, lens, window=window)
        if window == n - 1:                                      # all but the first
            assert bool((o == 0).all()) and bool(((lse.double() - np.log(n - 1)).abs() < 2.0 ** -10).all())
            continue
        # the shares without the first entry sum ones, exactly; its own adds 2^22 weights of 2^-30, 2^-8 of the sum, in
        # lanes of 2^18 terms, off by 2^-6 of that; exponent, join and logarithm 2^-16; the result's rounding 2^-8
        err = (o[0, :, :2].double().cpu() - want).abs()
        assert bool((err <= (2.0 ** -8 + 2.0 ** -10) * want).all()), o[0, 0, :2]
        assert bool((o[0, :, 2:] == 0).all())
        assert bool(((lse.double() - np.log(np.exp(20.75) + n - 1)).abs() < 2.0 ** -10).all())


def test_grow_counts_past_any_table(dev):
    """Numbers of tokens whose pages' sum passes 64 bits: they lack, and nothing changes."""
    rows = 16
    tables = torch.full((rows, 4), -1, dtype=torch.int32, device=dev)
    lens, refs = torch.zeros(rows, dtype=torch.int64, device=dev), torch.zeros(100, dtype=torch.int32, device=dev)
    for n in (2 ** 60, 2 ** 62, 2 ** 63 - 1):
        got = paged.grow(tables, lens, refs, torch.full((rows,), n, device=dev), 1)
        assert int(got[3]) > 0
        for a, b in zip(got[:3], (tables, lens, refs)):
            assert torch.equal(a, b)


# ---- fork ---------------------------------------------------------------------------------------


def test_fork_in_place_of_tables_without_columns(dev):
    """The C entry takes tables of no width; lengths alone change places."""
    lens, refs = torch.tensor([5, 7, 9], device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    parents = torch.tensor([1, -1, 0], dtype=torch.int32, device=dev)
    some = torch.zeros(4, dtype=torch.int32, device=dev)
    ws = torch.full((256,), 0x55, dtype=torch.uint8, device=dev)
    _lib.call("mzk_paged_fork", some.data_ptr(), 0, 3, 0, lens.data_ptr(), refs.data_ptr(), 4, parents.data_ptr(), 3, 16,
              some.data_ptr(), 0, lens.data_ptr(), refs.data_ptr(), ws.data_ptr(), 256, _lib.raw_stream(lens.device))
    assert lens.tolist() == [7, 0, 5]


# ---- compact ------------------------------------------------------------------------------------


@pytest.mark.parametrize("pages", [7, 40, 4096, 9000])
@pytest.mark.parametrize("inplace", [False, True])
def test_compact_says_where_pages_went(dev, pages, inplace):
    """Pages that something beside the tables holds are found again by `moved`."""
    g = _gen(pages)
    tables = torch.randperm(pages, generator=g)[:pages // 3].int().view(1, -1)
    refs = _counts(tables, pages)
    other = torch.randperm(pages, generator=g)[:pages // 4]
    refs[other] += 1
    pool = torch.randn(pages, 2, 4, generator=g)
    d = [t.to(dev) for t in (tables, refs)]
    dp, moved = pool.to(dev), torch.full((pages,), 99, dtype=torch.int32, device=dev)
    got = paged.compact(*d, pools=[dp], out=d if inplace else None, moved=moved)
    m = moved.cpu().long()
    used = int((refs > 0).sum())
    assert torch.equal(dp.cpu()[m[other]], pool[other])
    assert torch.equal(got[0].cpu().long(), m[tables.long()]) and torch.equal(got[1].cpu()[m[refs > 0]], refs[refs > 0])
    assert sorted(m[refs > 0].tolist()) == list(range(used)) and torch.equal(m[refs == 0], (refs == 0).nonzero()[:, 0])


def test_attend_of_short_sequences_takes_no_room_for_shares(dev):
    """400 sequences of ten tokens are not split, so nothing is allocated but the results."""
    pool, tables, n64, _, _ = _setup(dev, [10] * 400, 16, 576, "fp8", 97)
    q = torch.randn(400, 16, 576, generator=_gen(98)).bfloat16().to(dev)
    want = paged.attend(q, pool, tables, n64)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = paged.attend(q, pool, tables, n64)
    assert torch.cuda.max_memory_allocated() - before < 2 * (q.numel() * 2 + 400 * 16 * 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
