"""GPU: sliding-window attention beside which a sequence's first positions stay visible (``first=`` of
``paged.attend`` and ``csa2_attn.packed``) against plain attention in 64 bits (bounds: ``tests/ragged_ref.py``)."""

import numpy as np
import pytest
import torch

from mzoo_amd import csa2_attn, paged
from tests import ragged_ref as R
from tests.test_gpu_paged import ROPE, _entries, _gen, _of, _setup

pytestmark = pytest.mark.gpu


def _seen(n, end, window, first, dev):
    pos = (end - n + torch.arange(n, device=dev))[:, None]
    col = torch.arange(max(end, 0), device=dev)[None, :]
    return (col <= pos) & ((col > pos - window) | (col < first))


def _attend(dev, lens, tokens, heads, dim, fmt, page, window, first, seed, sinks=True):
    """tokens: new tokens of each sequence (1: one each, without cu)."""
    print(f"attend: lens {lens} tokens {tokens} heads {heads} dim {dim} {fmt} page {page} window {window} first {first}", flush=True)
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, fmt, seed)
    g = _gen(seed + 1)
    new = [1] * len(lens) if tokens == 1 else tokens
    q = torch.randn(sum(new), heads, dim, generator=g).bfloat16().to(dev)
    sk = torch.randn(heads, generator=g).to(dev) if sinks else None
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int64, device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=None if tokens == 1 else cu, window=window, first=first, sinks=sk,
                          rope=ROPE.get(dim, 64))
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    for b, (n, end) in enumerate(zip(new, lens)):
        if n:
            at = int(cu[b])
            R.check(o[at:at + n], lse[at:at + n],
                    R.attend(q[at:at + n], vals[_of(t, b, end, page)], _seen(n, end, window, first, dev), sk), f"sequence {b}")


FORMATS = [(576, "fp8"), (576, "bf16"), (512, "bf16"), (160, "fp8"), (160, "bf16"), (64, "bf16")]


@pytest.mark.parametrize("dim,fmt", FORMATS)
@pytest.mark.parametrize("first", [1, 4, 32, 33, 100])
def test_one_token_each(dev, dim, fmt, first):
    for heads, window in ((1, 1), (16, 40), (40, 64), (128, 33)):
        _attend(dev, [1, 0, 31, 33, 65, 100, 133, 400], 1, heads, dim, fmt, 16, window, first, dim + first, sinks=heads != 16)


@pytest.mark.parametrize("dim,fmt", FORMATS)
@pytest.mark.parametrize("heads", [1, 2, 5, 64])
def test_several_tokens(dev, dim, fmt, heads):
    # tokens before, across and behind the first positions and the window's begin; more tokens than entries
    for window, first in ((1, 1), (7, 20), (50, 3), (64, 130), (500, 8)):
        _attend(dev, [4, 100, 64, 37, 260, 9], [4, 1, 33, 0, 70, 12], heads, dim, fmt, 24, window, first, heads + dim)


@pytest.mark.parametrize("heads,lens", [(128, [9000]), (64, [20000, 1, 3000]), (16, [5000] * 7), (128, [70, 6000, 40, 12345])])
@pytest.mark.parametrize("window,first", [(1000, 4), (30, 2000), (3000, 700)])
def test_long(dev, heads, lens, window, first):
    """Windows and first positions long enough to be split and joined, the border between them inside a share."""
    _attend(dev, lens, 1, heads, 576, "fp8", 64, window, first, len(lens))
    _attend(dev, [n + 3 for n in lens], [3] * len(lens), heads, 160, "bf16", 24, window, first, len(lens) + 5)


@pytest.mark.parametrize("batch", [65, 200])
def test_many_sequences(dev, batch):
    lens = [(37 * i) % 900 for i in range(batch)]
    _attend(dev, lens, 1, 8, 576, "fp8", 32, 100, 5, batch)


def test_pages_given_up(dev):
    """Pages between the first positions and the window are never read: they may belong to others."""
    page, n, window, first = 16, 1000, 100, 20
    pool, tables, n64, _, _ = _setup(dev, [n, n], page, 576, "fp8", 5)
    q = torch.randn(2, 64, 576, generator=_gen(6)).bfloat16().to(dev)
    want = paged.attend(q, pool, tables, n64, window=window, first=first)
    cut = tables.clone()
    cut[:, (first + page - 1) // page:(n - window) // page] = -1
    got = paged.attend(q, pool, cut, n64, window=window, first=first)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cut[:, 1] = -1                                        # four first positions are on no page
    o, lse = paged.attend(q, pool, cut, n64, window=window, first=first)
    vals, t = _entries(pool, 576).to(dev), tables.cpu()
    for b in range(2):
        seen = _seen(1, n, window, 16, dev)
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], vals[_of(t, b, n, page)], seen, None), f"sequence {b}")


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (160, "bf16")])
def test_past_the_table(dev, dim, fmt):
    """A token whose window lies behind the table still sees the first positions."""
    page, width, heads = 8, 5, 16
    pool, tables, n64, _, _ = _setup(dev, [40, 40, 40], page, dim, fmt, 7, width=width)
    lens = torch.tensor([45, 60, 1 << 40], device=dev)
    q = torch.randn(6, heads, dim, generator=_gen(8)).bfloat16().to(dev)
    cu = torch.tensor([0, 2, 4, 6], device=dev)
    vals, t = _entries(pool, dim).to(dev), tables.cpu()
    for window, first in ((10, 3), (4, 39), (30, 300)):
        o, lse = paged.attend(q, pool, tables, lens, cu=cu, window=window, first=first, rope=ROPE.get(dim, 64))
        for b, end in enumerate(lens.tolist()):
            pos = (end - 2 + torch.arange(2, device=dev))[:, None]
            col = torch.arange(40, device=dev)[None, :]
            seen = (col <= pos) & ((col > pos - window) | (col < first))
            R.check(o[2 * b:2 * b + 2], lse[2 * b:2 * b + 2], R.attend(q[2 * b:2 * b + 2], vals[_of(t, b, 40, page)], seen, None),
                    f"sequence {b}")


@pytest.mark.parametrize("dim", [576, 160])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_unseen_entries_do_not_reach(dev, dim, bad):
    """An entry that is not finite reaches the tokens that see it -- one of the first: all -- and no other."""
    lens, new, page, heads, window, first = [90, 60], [6, 3], 16, 16, 8, 5
    pool, tables, n64, _, _ = _setup(dev, lens, page, dim, "bf16", 21)
    t = tables.cpu()
    flat = pool.view(-1, dim)
    flat[_of(t, 0, 90, page)[80], 5] = bad         # behind the window of the later tokens
    flat[_of(t, 0, 90, page)[5], 5] = bad          # behind the first positions: nobody's
    flat[_of(t, 1, 60, page)[4], 9] = bad          # the last of the first
    q = torch.randn(9, heads, dim, generator=_gen(22)).bfloat16().to(dev)
    cu = torch.tensor([0, 6, 9], device=dev)
    o, lse = paged.attend(q, pool, tables, n64, cu=cu, window=window, first=first)
    for b in range(2):
        for i in range(new[b]):
            pos = lens[b] - new[b] + i
            row = o[int(cu[b]) + i]
            if b == 1 or pos - window < 80:
                assert not bool(torch.isfinite(row).all())
            else:
                e = flat[_of(t, b, pos + 1, page)].double()
                seen = _seen(1, pos + 1, window, first, dev)
                R.check(row[None], lse[int(cu[b]) + i][None], R.attend(q[int(cu[b]) + i][None], e, seen, None), f"{b} {i}")


@pytest.mark.parametrize("scale", [30.0, 1e4])
def test_wide_scores(dev, scale):
    """First positions that outweigh the window, and the other way round."""
    lens, page, heads = [300, 700], 32, 64
    pool, tables, n64, _, _ = _setup(dev, lens, page, 576, "bf16", 31)
    t = tables.cpu()
    flat = pool.view(-1, 576)
    flat[_of(t, 0, 300, page)[:4]] *= scale
    flat[_of(t, 1, 700, page)[690:]] *= scale
    q = torch.randn(2, heads, 576, generator=_gen(32)).bfloat16().to(dev)
    o, lse = paged.attend(q, pool, tables, n64, window=64, first=4)
    for b, n in enumerate(lens):
        R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], flat[_of(t, b, n, page)].double(), _seen(1, n, 64, 4, dev), None), f"{b}")


# ---- packed prompts -----------------------------------------------------------------------------

@pytest.mark.parametrize("heads,groups,dim", [(64, 1, 576), (8, 2, 160), (3, 1, 576), (128, 2, 512), (1, 1, 64), (40, 1, 96)])
@pytest.mark.parametrize("window,first", [(1, 1), (7, 40), (64, 4), (33, 100), (600, 5)])
def test_packed(dev, heads, groups, dim, window, first):
    new, tail = [1, 0, 70, 33, 200, 517], 3
    print(f"packed: heads {heads}/{groups} dim {dim} window {window} first {first}", flush=True)
    g = _gen(heads + first)
    total = sum(new) + tail
    q = torch.randn(total, heads, dim, generator=g).bfloat16().to(dev)
    kv = torch.randn(total, groups, dim, generator=g).bfloat16().to(dev)
    sk = torch.randn(heads, generator=g).to(dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int64, device=dev)
    o, lse = csa2_attn.packed(q, kv, cu, window=window, first=first, sinks=sk)
    per, at = heads // groups, 0
    for b, n in enumerate(new):
        for j in range(groups if n else 0):
            hs = slice(j * per, (j + 1) * per)
            R.check(o[at:at + n, hs], lse[at:at + n, hs],
                    R.attend(q[at:at + n, hs], kv[at:at + n, j], _seen(n, n, window, first, dev), sk[hs]), f"sequence {b} latent {j}")
        at += n
    assert bool((o[at:] == 0).all()) and bool((lse[at:] == float("-inf")).all())


@pytest.mark.parametrize("dim", [576, 160])
def test_packed_unseen_entries_do_not_reach(dev, dim):
    n, heads, window, first = 150, 4, 10, 6
    q = torch.randn(n, heads, dim, generator=_gen(41)).bfloat16().to(dev)
    kv = torch.randn(n, 1, dim, generator=_gen(42)).bfloat16().to(dev)
    kv[70, 0, 3] = float("nan")
    cu = torch.tensor([0, n], device=dev)
    o, lse = csa2_attn.packed(q, kv, cu, window=window, first=first)
    hit = [t for t in range(n) if 70 <= t < 70 + window]
    fine = [t for t in range(n) if t not in hit]
    assert bool(torch.isnan(o[hit]).any(-1).all())
    e = kv[:, 0].double().nan_to_num()
    seen = _seen(n, n, window, first, dev)
    R.check(o[fine], lse[fine], R.attend(q[fine], e, seen[fine], None), "others")


def test_ends_of_the_range(dev):
    """first 0 is the call without; a window that nothing leaves, and first positions past every sequence, hide nothing."""
    lens, page = [300, 45], 16
    pool, tables, n64, _, _ = _setup(dev, lens, page, 576, "fp8", 51)
    q = torch.randn(2, 16, 576, generator=_gen(52)).bfloat16().to(dev)
    x, y = paged.attend(q, pool, tables, n64, window=50), paged.attend(q, pool, tables, n64, window=50, first=0)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    vals, t = _entries(pool, 576).to(dev), tables.cpu()
    for kw in (dict(window=300, first=7), dict(window=1 << 40, first=7), dict(window=50, first=(1 << 30) - 1)):
        o, lse = paged.attend(q, pool, tables, n64, **kw)
        for b, n in enumerate(lens):
            seen = torch.ones(1, n, dtype=torch.bool, device=dev)
            R.check(o[b:b + 1], lse[b:b + 1], R.attend(q[b:b + 1], vals[_of(t, b, n, page)], seen, None), f"{kw} {b}")
    kv = torch.randn(345, 1, 576, generator=_gen(53)).bfloat16().to(dev)
    q = torch.randn(345, 16, 576, generator=_gen(54)).bfloat16().to(dev)
    cu = torch.tensor([0, 300, 345], device=dev)
    x, y = csa2_attn.packed(q, kv, cu, window=50), csa2_attn.packed(q, kv, cu, window=50, first=0)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_captured(dev):
    """Recorded once; lengths, tables and queries change between the replays."""
    pool, tables, n64, _, _ = _setup(dev, [6000, 200, 3000], 64, 576, "fp8", 61)
    q = torch.randn(3, 128, 576, generator=_gen(62)).bfloat16().to(dev)
    lens = n64.clone()
    o, lse = torch.empty_like(q), torch.empty(3, 128, device=dev)
    ws = torch.empty(paged.attend_workspace_bytes(3, 128, 576, 3, False, tables.shape[1], 64, 4096, -1, 10), dtype=torch.uint8, device=dev)
    kw = dict(window=4096, first=10, workspace=ws)
    paged.attend(q, pool, tables, lens, out=o, lse=lse, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(q, pool, tables, lens, out=o, lse=lse, **kw)
    for i in range(4):
        q.copy_(torch.randn(3, 128, 576, generator=_gen(63 + i)).bfloat16())
        lens.copy_(n64 - torch.tensor([7 * i, 50 * i, 900 * i], device=dev))
        graph.replay()
        got = (o.clone(), lse.clone())
        want = paged.attend(q, pool, tables, lens, window=4096, first=10)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
