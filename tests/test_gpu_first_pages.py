"""GPU: sequences without end beside a window with first positions: the pages between, which no token sees any more, go back to
the pool by the caller's own hand (table entries to -1, ``refs`` lowered), and ``grow``, ``append``, ``attend`` and ``fork`` go on."""

import pytest
import torch

from mzoo_amd import paged
from tests import ragged_ref as R

pytestmark = pytest.mark.gpu


def _give_back(tables, lens, refs, page, window, first):
    """The pages of which every position lies behind the first ones and before every window to come."""
    col = torch.arange(tables.shape[1], device=tables.device)[None, :]
    old = (col * page >= first) & ((col + 1) * page <= lens[:, None] - window) & (tables >= 0)
    refs.index_add_(0, torch.where(old, tables, 0).flatten().long(), -old.flatten().int())
    tables.masked_fill_(old, -1)


@pytest.mark.parametrize("dim,fork", [(160, False), (576, False), (64, True)])
def test_a_sequence_without_end(dev, dim, fork):
    page, window, first, batch, heads, steps = 8, 30, 11, 3, 4, 40
    pages = batch * (2 + 6)                           # first positions 2, a window and its ends 5, one new
    g = torch.Generator().manual_seed(dim)
    pool = paged.new_pool(pages, page, dim, "bf16", device=dev)
    tables = torch.full((batch, 64), -1, dtype=torch.int32, device=dev)
    lens, refs = torch.zeros(batch, dtype=torch.int64, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
    missing = torch.zeros(1, dtype=torch.int64, device=dev)
    state, text = (tables, lens, refs), [torch.empty(0, dim).bfloat16() for _ in range(batch)]
    for step in range(steps):
        new = [1 + (step + b) % 7 for b in range(batch)]
        n = torch.tensor(new, device=dev)
        paged.grow(*state, n, page, pools=[pool], out=state, missing=missing)
        assert int(missing) == 0
        x = torch.randn(sum(new), dim, generator=g).bfloat16()
        cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), n.cumsum(0)])
        paged.append(pool, tables, lens, x.to(dev), cu=cu, rope=0)
        text = [torch.cat([t, e]) for t, e in zip(text, x.split(new))]
        q = torch.randn(sum(new), heads, dim, generator=g).bfloat16().to(dev)
        o, lse = paged.attend(q, pool, tables, lens, cu=cu, window=window, first=first, rope=0)
        assert lens.tolist() == [len(t) for t in text]
        for b in range(batch):
            end, at = len(text[b]), int(cu[b])
            pos = (end - new[b] + torch.arange(new[b], device=dev))[:, None]
            col = torch.arange(end, device=dev)[None, :]
            seen = (col <= pos) & ((col > pos - window) | (col < first))
            R.check(o[at:at + new[b]], lse[at:at + new[b]], R.attend(q[at:at + new[b]], text[b].to(dev), seen, None), f"step {step} sequence {b}")
        _give_back(tables, lens, refs, page, window, first)
        if fork and step % 5 == 4:
            parents = torch.tensor([1, 1, 2] if step % 2 else [0, 2, 0], dtype=torch.int32, device=dev)
            paged.fork(*state, parents, page, out=state)
            text = [text[p] for p in parents.tolist()]
        count = torch.zeros(pages, dtype=torch.int32, device=dev)
        held = tables[tables >= 0].long()
        assert torch.equal(count.index_add_(0, held, torch.ones_like(held, dtype=torch.int32)), refs)
    assert int(lens.sum()) > 2 * pages * page         # far more than the pool holds
