"""GPU: causal attention over packed prompts (``csa2_attn.packed``) against plain attention in 64 bits."""

import numpy as np
import pytest
import torch

from mzoo_amd import csa2_attn, paged
from oracle import quant as OQ
from tests import ragged_ref as R

pytestmark = pytest.mark.gpu


def _check(dev, new, heads, groups, dim, window, seed, sinks=True, tail=0, strided=False):
    print(f"packed: {new} heads {heads}/{groups} dim {dim} window {window}", flush=True)
    g = torch.Generator().manual_seed(seed)
    t = sum(new) + tail
    q = torch.randn(t, heads, dim, generator=g).bfloat16().to(dev)
    kv = torch.randn(t, groups * dim + 24, generator=g).bfloat16().to(dev)
    kv = kv[:, 8:8 + groups * dim].view(t, groups, dim) if strided else kv[:, :groups * dim].contiguous().view(t, groups, dim)
    sk = torch.randn(heads, generator=g).to(dev) if sinks else None
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int64, device=dev)
    o, lse = csa2_attn.packed(q, kv, cu, window=window, sinks=sk)
    per = heads // groups
    at = 0
    for b, n in enumerate(new):
        if n:
            pos, col = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None, :]
            seen = (col <= pos) & (col > pos - (window or 1 << 40))
            for j in range(groups):
                hs = slice(j * per, (j + 1) * per)
                R.check(o[at:at + n, hs], lse[at:at + n, hs],
                        R.attend(q[at:at + n, hs], kv[at:at + n, j], seen, None if sk is None else sk[hs]), f"sequence {b} latent {j}")
        at += n
    assert bool((o[at:] == 0).all()) and bool((lse[at:] == float("-inf")).all())


@pytest.mark.parametrize("dim", [64, 96, 128, 160, 256, 512, 576])
@pytest.mark.parametrize("heads,groups", [(1, 1), (16, 1), (128, 1), (24, 3)])
def test_packed_lengths(dev, dim, heads, groups):
    _check(dev, [1, 0, 33, 32, 64, 2, 97], heads, groups, dim, None, dim + heads)


@pytest.mark.parametrize("window", [1, 7, 64, 100])
@pytest.mark.parametrize("heads,groups,dim", [(64, 1, 576), (8, 2, 160), (3, 1, 576), (128, 2, 512)])
def test_packed_window(dev, window, heads, groups, dim):
    _check(dev, [150, 1, 0, 70], heads, groups, dim, window, window)


@pytest.mark.parametrize("heads,groups", [(2, 1), (5, 1), (40, 1), (100, 1), (12, 4), (6, 6)])
def test_packed_heads(dev, heads, groups):
    _check(dev, [77, 40], heads, groups, 576, None, heads, sinks=False)


def test_packed_strided_and_tail(dev):
    _check(dev, [50, 9], 16, 2, 160, None, 1, tail=6, strided=True)
    _check(dev, [50, 9], 64, 1, 576, 20, 2, tail=3, strided=True)
    _check(dev, [0, 0], 64, 1, 576, None, 3, tail=5)


def test_packed_many_sequences(dev):
    _check(dev, [1 + i % 5 for i in range(600)], 4, 1, 64, None, 4)
    _check(dev, [0] * 300 + [3] + [0] * 300 + [40], 128, 1, 576, None, 5)


def test_packed_long(dev):
    _check(dev, [1500, 900], 16, 1, 576, None, 6)


def test_packed_empty(dev):
    q, kv = torch.empty(0, 8, 64, dtype=torch.bfloat16, device=dev), torch.empty(0, 1, 64, dtype=torch.bfloat16, device=dev)
    o, lse = csa2_attn.packed(q, kv, torch.zeros(3, dtype=torch.int64, device=dev))
    assert o.shape == (0, 8, 64) and lse.shape == (0, 8)


def test_packed_given_outputs_keep_their_tail(dev):
    q = torch.randn(9, 16, 160, device=dev).bfloat16()
    kv = torch.randn(9, 1, 160, device=dev).bfloat16()
    cu = torch.tensor([0, 4, 6], device=dev)
    out, lse = torch.full_like(q, 5.0), torch.full((9, 16), 6.0, device=dev)
    csa2_attn.packed(q, kv, cu, out=out, lse=lse)
    o, l = csa2_attn.packed(q, kv, cu)
    assert torch.equal(out[:6], o[:6]) and torch.equal(lse[:6], l[:6])
    assert bool((out[6:] == 5.0).all()) and bool((lse[6:] == 6.0).all())


@pytest.mark.parametrize("heads,dim", [(16, 576), (1, 576), (16, 160), (1, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_packed_later_tokens_do_not_reach(dev, heads, dim, bad):
    """A latent that is not finite reaches no earlier token, and none that it is behind the window of."""
    g = torch.Generator().manual_seed(7)
    n, at = 90, 41
    q = torch.randn(n, heads, dim, generator=g).bfloat16().to(dev)
    kv = torch.randn(n, 1, dim, generator=g).bfloat16().to(dev)
    kv[at, 0, 2] = bad
    cu = torch.tensor([0, n], device=dev)
    for window in (None, 9):
        o, lse = csa2_attn.packed(q, kv, cu, window=window)
        last = n if window is None else at + window
        assert not bool(torch.isfinite(o[at:last]).all(-1).any())
        pos, col = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None, :]
        seen = (col <= pos) & (col > pos - (window or 1 << 40))
        clean = kv[:, 0].double().nan_to_num(0.0, 0.0, 0.0)
        ref = R.attend(q, clean, seen, None)
        for part in (slice(0, at), slice(last, n)):
            R.check(o[part], lse[part], tuple(x[part] for x in ref), f"window {window} {part}")


@pytest.mark.parametrize("scale", [0.0, 40.0, 5e3])
@pytest.mark.parametrize("window", [None, 5])
def test_packed_wide_scores(dev, scale, window):
    """Scores that rise by hundreds along the prompt."""
    n, heads, dim = 400, 16, 576
    g = torch.Generator().manual_seed(8)
    base = torch.randn(dim, generator=g)
    q = (base[None, None] + 0.01 * torch.randn(n, heads, dim, generator=g)).bfloat16().to(dev)
    kv = (torch.linspace(-scale, scale, n)[:, None, None] * base / 24.0).bfloat16().to(dev)
    o, lse = csa2_attn.packed(q, kv, torch.tensor([0, n], device=dev), window=window)
    pos, col = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None, :]
    seen = (col <= pos) & (col > pos - (window or 1 << 40))
    R.check(o, lse, R.attend(q, kv[:, 0], seen, None), "ramp")


def test_packed_captured(dev):
    q = torch.randn(300, 16, 576, device=dev).bfloat16()
    kv = torch.randn(300, 1, 576, device=dev).bfloat16()
    cu = torch.tensor([0, 100, 101, 300], device=dev)
    out, lse = torch.empty_like(q), torch.empty(300, 16, device=dev)
    csa2_attn.packed(q, kv, cu, out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        csa2_attn.packed(q, kv, cu, out=out, lse=lse)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        cu.copy_(torch.tensor([0, 50 * i, 200 + i, 300]))
        want = csa2_attn.packed(q, kv, cu)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_nothing(dev):
    """No tokens, no sequences, sequences of no tokens."""
    q = torch.randn(70, 8, 160, device=dev).bfloat16()
    for t, cu in ((0, [0]), (0, [0, 0, 0]), (3, [0]), (70, [0]), (70, [0, 0, 0])):
        o, lse = csa2_attn.packed(q[:t], q[:t, :2].contiguous(), torch.tensor(cu, device=dev))
        assert o.shape == (t, 8, 160) and bool((o == 0).all()) and bool((lse == float("-inf")).all())
    cu = torch.tensor([0, 30, 70], device=dev)
    want = csa2_attn.packed(q, q[:, :2].contiguous(), cu)
    for window in (40, 2 ** 30, 2 ** 62, 2 ** 64 + 1):
        got = csa2_attn.packed(q, q[:, :2].contiguous(), cu, window=window)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dim,fmt", [(576, "fp8"), (576, "bf16"), (160, "bf16")])
def test_prompts_then_steps(dev, dim, fmt):
    """As a server runs them: pages for prompts of different lengths, their attention packed, and from the
    pages in two chunks; then steps of one token, one sequence ending and another forked on the way."""
    page, pages, heads, rope = 16, 90, 24, 64 if dim == 576 else 32
    g = torch.Generator().manual_seed(dim)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)
    lens = [50, 1, 33, 80]
    pool = paged.new_pool(pages, page, dim, fmt, rope=rope, device=dev)
    tables = torch.full((4, 12), -1, dtype=torch.int32, device=dev)
    n, refs = torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
    state, sinks = (tables, n, refs), torch.randn(heads, generator=g).to(dev)
    hist = [rnd(k, dim) for k in lens]
    q = [rnd(k, heads, dim) for k in lens]

    def values(x):  # what a page gives back of x
        if fmt == "bf16" or len(x) == 0:
            return x.double()
        return torch.from_numpy(OQ.unpack_latent_fp8_b128(OQ.pack_latent_fp8_b128(x.float().cpu().numpy(), dim - rope), dim - rope, rope)).to(dev)

    def see(o, lse, qs, x, first, sink, what):
        if len(qs) == 0:
            return
        seen = torch.arange(x.shape[0], device=dev)[None, :] <= first + torch.arange(qs.shape[0], device=dev)[:, None]
        R.check(o, lse, R.attend(qs, x.double(), seen, sink), what)

    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), device=dev)
    o, lse = csa2_attn.packed(torch.cat(q), torch.cat(hist)[:, None], cu, sinks=sinks)
    for b in range(4):
        see(o[cu[b]:cu[b + 1]], lse[cu[b]:cu[b + 1]], q[b], hist[b], 0, sinks, f"prompt {b}")
    half = [k // 2 for k in lens]
    for lo, hi in ((lambda b: 0, lambda b: half[b]), (lambda b: half[b], lambda b: lens[b])):
        new = [hi(b) - lo(b) for b in range(4)]
        c = torch.tensor(np.concatenate([[0], np.cumsum(new)]), device=dev)
        assert int(paged.grow(*state, torch.tensor(new, device=dev), page, pools=[pool], out=state)[3]) == 0
        paged.append(pool, tables, n, torch.cat([hist[b][lo(b):hi(b)] for b in range(4)]), cu=c, rope=rope)
        o, lse = paged.attend(torch.cat([q[b][lo(b):hi(b)] for b in range(4)]), pool, tables, n, cu=c, sinks=sinks, rope=rope)
        for b in range(4):
            see(o[c[b]:c[b + 1]], lse[c[b]:c[b + 1]], q[b][lo(b):hi(b)], values(hist[b][:hi(b)]), lo(b), sinks, f"chunk {b}")
    ones = torch.ones(4, dtype=torch.int64, device=dev)
    for i in range(6):
        if i == 3:  # sequence 1 ends, its row goes on from sequence 3
            paged.fork(*state, torch.tensor([0, 3, 2, 3], dtype=torch.int32, device=dev), page, out=state)
            hist[1] = hist[3]
        kv, qs = rnd(4, dim), rnd(4, heads, dim)
        assert int(paged.grow(*state, ones, page, pools=[pool], out=state)[3]) == 0
        paged.append(pool, tables, n, kv, rope=rope)
        o, lse = paged.attend(qs, pool, tables, n, sinks=sinks, rope=rope)
        for b in range(4):
            hist[b] = torch.cat([hist[b], kv[b:b + 1]])
            see(o[b:b + 1], lse[b:b + 1], qs[b:b + 1], values(hist[b]), hist[b].shape[0] - 1, sinks, f"step {i} {b}")
    used = -(-n // page)  # rows 1 and 3 share their whole pages of the fork
    assert int((refs > 0).sum()) == int(used.sum()) - 83 // page
