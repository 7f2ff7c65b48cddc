"""GPU: tokens from logits -- draws, drafted tokens' verification, beams -- against plain restatements in
64 bits (``tests/sampling_ref.py``)."""

import numpy as np
import pytest
import torch

from mzoo_amd import paged, sampling
from tests import sampling_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _logits(rows, v, seed, dtype=torch.float32, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * (std * (0.4 + torch.rand(rows, 1, generator=g)))
    if v > 8:
        at = torch.randint(0, v, (rows, 6), generator=g)
        x.scatter_add_(1, at, 10 * torch.rand(rows, 6, generator=g))
    return x.to(dtype)


def _u(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed))


def _row(f, i):
    return f[i].item() if torch.is_tensor(f) else f


def _check_sample(dev, logits, u, workspace=None, given=None, **filters):
    print(f"sample {list(logits.shape)} {logits.dtype} {logits.stride()} " +
          " ".join(f"{k}={'tensor' if torch.is_tensor(f) else f}" for k, f in filters.items()), flush=True)
    on = {k: f.to(dev) if torch.is_tensor(f) else f for k, f in filters.items()}
    tokens, logprobs = sampling.sample(given if given is not None else logits.to(dev), u.to(dev), workspace=workspace, **on)
    got, lp = tokens.cpu().numpy(), logprobs.cpu().double().numpy()
    for i in range(logits.shape[0]):
        f = {k: _row(x, i) for k, x in filters.items() if x is not None}
        token, want, clear = R.sample(logits[i].float().numpy(), u[i].item(), **f)
        assert clear, f"row {i}: a border is near"
        assert got[i] == token, f"row {i}: token {got[i]}, expected {token}"
        if token < 0:
            assert lp[i] == -np.inf
        else:
            # the weights' 2^-49, sums of whole numbers of 2^-43 in 512 bins, and float32's half step
            assert abs(lp[i] - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -30, f"row {i}: {lp[i]} {want}"
    return tokens, logprobs


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05),
           dict(temperature=1.3, top_k=200, top_p=0.8), dict(top_k=1000, min_p=0.01), dict(top_p=0.95, min_p=0.1, temperature=1.7),
           dict(temperature=0.6, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0),
           dict(temperature=0.0, top_k=5, top_p=0.5)]


# ---- sample ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 8, 9, 100, 2047, 2048, 2049, 8193, 32000])
def test_sample_sizes(dev, dtype, v):
    for i, f in enumerate(FILTERS):
        _check_sample(dev, _logits(3, v, v + i, dtype), _u(3, i), **f)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", [(1, 131072), (5, 50257), (40, 131072), (33, 151936)])
def test_sample_large(dev, dtype, rows, v):
    logits = _logits(rows, v, rows, dtype)
    for i, f in enumerate((dict(), dict(top_p=0.9, temperature=0.8), dict(top_k=50, top_p=0.95), dict(min_p=0.05, temperature=1.5))):
        _check_sample(dev, logits, _u(rows, i), **f)


def test_sample_longest_row(dev):
    _check_sample(dev, _logits(1, 1 << 20, 3), _u(1, 4), top_p=0.9)
    _check_sample(dev, _logits(1, (1 << 20) - 1, 5, torch.bfloat16, 0.3), _u(1, 6), top_k=5000)


@pytest.mark.parametrize("v", [40, 5000, 70001])
def test_sample_settings_of_each_row(dev, v):
    rows, g = 48, torch.Generator().manual_seed(v)

    def one(options, dt):
        return torch.tensor(options)[torch.randint(0, len(options), (rows,), generator=g)].to(dt)
    _check_sample(dev, _logits(rows, v, v), _u(rows, v), temperature=one([0.0, 0.3, 1.0, 2.0, -1.0], torch.float32),
                  top_k=one([0, 1, 3, 40, 1000, 1 << 30, -4], torch.int32), top_p=one([0.0, 0.3, 0.9, 1.0, 1.5], torch.float32),
                  min_p=one([0.0, 0.0, 0.01, 0.3, 1.0], torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_ties(dev, dtype):
    """Few different logits: cuts and draws fall among equal ones."""
    for step in (0.5, 2.0, 100.0):
        x = (torch.round(_logits(12, 9001, 7).clamp(-8, 8) / step) * step).to(dtype)
        for i, f in enumerate((dict(), dict(top_k=100), dict(top_k=5000), dict(top_p=0.7), dict(min_p=0.2), dict(top_k=777, top_p=0.31))):
            _check_sample(dev, x, _u(12, 70 + i), **f)


@pytest.mark.parametrize("v", [1, 64, 1000, 4096, 131072])
def test_sample_equal_logits(dev, v):
    """All weights 1: running sums are exact, and so are borders that are hit exactly."""
    x = torch.full((8, v), -3.25)
    u = torch.tensor([0.0, 2.0 ** -24, 0.25, 0.5, 0.5 - 2.0 ** -24, 0.75, 1 - 2.0 ** -24, 0.125])
    for f in (dict(), dict(top_k=max(1, v // 2)), dict(top_p=0.5), dict(top_p=0.25, top_k=max(1, v // 2)), dict(min_p=1.0)):
        _check_sample(dev, x, u, **f)


def test_sample_flat_rows(dev):
    """So many tokens between the cuts that they are not listed but read again."""
    for std in (0.01, 0.2):
        x = torch.randn(3, 131072, generator=torch.Generator().manual_seed(9)) * std
        for i, f in enumerate((dict(), dict(top_k=60000), dict(top_p=0.6), dict(min_p=0.95), dict(top_k=90000, top_p=0.5, min_p=0.5))):
            _check_sample(dev, x, _u(3, i), **f)
            _check_sample(dev, x.bfloat16(), _u(3, i + 9), **f)


def test_sample_odd_values(dev):
    inf, nan, big = float("inf"), float("nan"), 3.4e38
    x = _logits(12, 3001, 11)
    x[0, :] = -inf
    x[1, :] = nan
    x[2, :] = -inf
    x[2, 17] = -5.0                                # the only one
    x[3, ::2] = nan
    x[4, 100:2900] = -inf                          # a masked vocabulary
    x[5, 5], x[5, 9] = inf, inf
    x[6, 3] = big
    x[7, :] = -big
    x[8, :] = 0.0
    x[8, ::3] = -0.0                               # equal to 0
    x[9, :] = torch.finfo(torch.float32).min       # a mask of the type's lowest value
    x[9, 70:80] = 1.0
    x[10, 1:] -= 1e6
    x[11, :] = 1e-42                               # subnormal
    x[11, 7] = 2e-42
    for i, f in enumerate(FILTERS):
        _check_sample(dev, x, _u(12, 100 + i), **f)
    for i, t in enumerate((1e-45, 1e-30, 1e-3, 1e3, 1e30, 3.4e38, inf)):
        _check_sample(dev, x, _u(12, 200 + i), temperature=t)
        _check_sample(dev, x, _u(12, 300 + i), temperature=t, top_k=20, top_p=0.9)
    h = x.clamp(-6e4, 6e4).half()
    h[5, 5] = inf
    h[9, 0:70] = torch.finfo(torch.float16).min
    _check_sample(dev, h, _u(12, 400), top_p=0.9)


def test_sample_random_numbers_at_the_ends(dev):
    x = _logits(6, 5000, 13)
    u = torch.tensor([0.0, 1.0, -0.5, 7.0, float("nan"), 1 - 2.0 ** -24])
    for f in (dict(), dict(top_k=10), dict(top_p=0.5)):
        got = sampling.sample(x.to(dev), u.to(dev), **f)[0].cpu()
        for i in range(6):
            order, w, _ = R.kept(x[i].numpy(), **f)
            if i in (0, 2, 4):
                assert got[i] == order[0]
            elif f:
                assert got[i] == order[-1]
            else:
                # beyond the last border: a token behind which nothing has weight that counts
                place = int(np.flatnonzero(order == int(got[i]))[0])
                assert float(w[place + 1:].sum() / w.sum()) <= 2.0 ** -24 + 2.0 ** -28


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_strides_and_alignment(dev, dtype):
    wide = _logits(9, 4200, 17, dtype)
    on = wide.to(dev)
    for a, z in ((0, 4200), (1, 4200), (3, 4110), (7, 4096), (5, 6)):
        _check_sample(dev, wide[:, a:z], _u(9, a), given=on[:, a:z], top_p=0.9)
    _check_sample(dev, wide[::2, 1:], _u(5, 3), given=on[::2, 1:], top_k=30)
    _check_sample(dev, wide[:, ::3], _u(9, 4), given=on[:, ::3])
    _check_sample(dev, wide[:1].expand(6, 4200), _u(6, 5), given=on[:1].expand(6, 4200), top_k=300)


def test_sample_is_the_same_in_any_batch(dev):
    """The rows' chunks are of two sizes, by the batch; their tokens and probabilities agree."""
    x, u = _logits(64, 100000, 19), _u(64, 20)
    x, u = x.to(dev), u.to(dev)
    for f in (dict(), dict(top_p=0.9, temperature=0.9), dict(top_k=500)):
        tok, lp = sampling.sample(x, u, **f)
        again = sampling.sample(x, u, **f)
        assert torch.equal(tok, again[0]) and torch.equal(lp, again[1])
        for i in (0, 31, 63):
            one = sampling.sample(x[i:i + 1], u[i:i + 1], **f)
            assert torch.equal(one[0], tok[i:i + 1])
            assert float((one[1] - lp[i:i + 1]).abs()) <= 2.0 ** -23 * float(lp[i].abs()) + 2.0 ** -29


def test_sample_nothing_and_given_outputs(dev):
    tok, lp = sampling.sample(torch.empty(0, 50, device=dev), torch.empty(0, device=dev))
    assert tok.shape == (0,) and lp.shape == (0,)
    x, u = _logits(5, 3000, 23).to(dev), _u(5, 24).to(dev)
    out = (torch.full((5,), -7, device=dev), torch.full((5,), 7.0, device=dev))
    ws = torch.full((sampling.sample_workspace_bytes(5, 3000),), 0xff, dtype=torch.uint8, device=dev)
    got = sampling.sample(x, u, top_k=40, out=out, workspace=ws)
    assert got[0] is out[0] and got[1] is out[1]
    want = sampling.sample(x, u, top_k=40)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    small = sampling.sample(x[:2, :100], u[:2], top_p=0.9, workspace=ws)   # what a larger call left there
    want = sampling.sample(x[:2, :100], u[:2], top_p=0.9)
    assert torch.equal(small[0], want[0])


def test_sample_on_another_stream(dev):
    x, u = _logits(6, 40000, 25).to(dev), _u(6, 26).to(dev)
    want = sampling.sample(x, u, top_p=0.8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = sampling.sample(x, u, top_p=0.8)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sample_captured(dev):
    """Settings and logits change between the replays of a recorded call; two graphs share a workspace."""
    rows, v = 7, 60000
    x, u = _logits(rows, v, 27).to(dev), _u(rows, 28).to(dev)
    t = torch.ones(rows, device=dev)
    k = torch.zeros(rows, dtype=torch.int32, device=dev)
    p = torch.ones(rows, device=dev)
    ws = torch.empty(sampling.sample_workspace_bytes(rows, v), dtype=torch.uint8, device=dev)
    outs = [(torch.empty(rows, dtype=torch.int64, device=dev), torch.empty(rows, device=dev)) for _ in range(2)]
    calls = [lambda: sampling.sample(x, u, temperature=t, top_k=k, top_p=p, workspace=ws, out=outs[0]),
             lambda: sampling.sample(x[:3], u[:3], min_p=0.1, workspace=ws, out=(outs[1][0][:3], outs[1][1][:3]))]
    graphs = []
    for c in calls:
        c()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c()
        graphs.append(g)
    for i in range(4):
        x.copy_(_logits(rows, v, 30 + i))
        u.copy_(_u(rows, 40 + i))
        t.fill_(0.5 + 0.5 * i)
        k.fill_(10 * i)
        p.fill_(1 - 0.2 * i)
        for g in graphs:
            g.replay()
        got = [o.clone() for o in (*outs[0], *outs[1])]
        want = sampling.sample(x, u, temperature=t, top_k=k, top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        want = sampling.sample(x[:3], u[:3], min_p=0.1)
        assert torch.equal(got[2][:3], want[0]) and torch.equal(got[3][:3], want[1])


# ---- verify ---------------------------------------------------------------------------------

def _check_verify(dev, logits, tokens, cu, u, draw, probs=None, **filters):
    print(f"verify {list(logits.shape)} {logits.dtype} {cu} probs {probs is not None} {filters if not any(map(torch.is_tensor, filters.values())) else ''}",
          flush=True)
    on = {k: f.to(dev) if torch.is_tensor(f) else f for k, f in filters.items()}
    acc, nxt = sampling.verify(logits.to(dev), tokens.to(dev), torch.tensor(cu, device=dev), u.to(dev), draw.to(dev),
                               draft_probs=None if probs is None else probs.to(dev), **on)
    acc, nxt = acc.cpu().tolist(), nxt.cpu().tolist()
    for b, (a, z) in enumerate(zip(cu, cu[1:])):
        f = {k: x[a:z].numpy() if torch.is_tensor(x) else x for k, x in filters.items() if x is not None}
        n, t, clear = R.verify(logits[a:z].float().numpy(), tokens[a:z].tolist(), u[a:z].numpy(), draw[b].item(),
                               None if probs is None else probs[a:z].numpy(), **f)
        assert clear, f"sequence {b}: a border is near"
        assert (acc[b], nxt[b]) == (n, t), f"sequence {b}: {acc[b]} accepted, then {nxt[b]}; expected {n}, {t}"
    return acc, nxt


def _drafts(logits, cu, seed, probs):
    """Drafted tokens: mostly the likely ones, some of any kind; the draft's probabilities."""
    g = torch.Generator().manual_seed(seed)
    rows, v = logits.shape
    near = logits.float() + torch.randn(rows, v, generator=g)
    q = torch.softmax(near, 1)
    guess = torch.multinomial(q, 1, generator=g)[:, 0] if probs else near.argmax(1)
    any_ = torch.randint(0, v, (rows,), generator=g)
    guess = torch.where(torch.rand(rows, generator=g) < 0.1, any_, guess)
    return guess.roll(1).contiguous(), q if probs else None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("v", [5, 1000, 9001, 70000])
def test_verify(dev, dtype, probs, v):
    cu = [0, 5, 6, 6, 9, 17, 17]
    for i, f in enumerate((dict(), dict(temperature=0.7, top_p=0.9), dict(top_k=3), dict(top_k=40, min_p=0.02), dict(temperature=0.0))):
        logits = _logits(20, v, v + i, dtype, 2.0)              # three rows of no sequence
        tokens, q = _drafts(logits, cu, i, probs)
        _check_verify(dev, logits, tokens, cu, _u(20, 50 + i), _u(6, 60 + i), q, **f)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_many(dev, probs):
    g = torch.Generator().manual_seed(3)
    cu = [0] + torch.cumsum(torch.randint(0, 6, (150,), generator=g), 0).tolist()
    logits = _logits(cu[-1], 3000, 4, std=1.0)
    tokens, q = _drafts(logits, cu, 5, probs)
    acc, _ = _check_verify(dev, logits, tokens, cu, _u(cu[-1], 6), _u(150, 7), q, top_p=0.97)
    assert len(set(acc)) >= 4


def test_verify_settings_of_each_row(dev):
    cu = [0, 4, 9, 10]
    logits = _logits(10, 2000, 8, std=1.0)
    tokens, q = _drafts(logits, cu, 9, True)
    f = dict(temperature=torch.tensor([0.0, 1.0, 0.5, 2.0, 0.7, 1.0, 1.0, 0.0, 1.0, 1.0]), top_k=torch.tensor([0, 5, 0, 50, 1, 0, 9, 0, 0, 3]).int(),
             top_p=torch.tensor([1.0, 0.9, 0.5, 1.0, 1.0, 0.8, 0.9, 1.0, 1.0, 0.95]))
    for i in range(4):
        _check_verify(dev, logits, tokens, cu, _u(10, 20 + i), _u(3, 30 + i), q, **f)
        _check_verify(dev, logits, tokens, cu, _u(10, 40 + i), _u(3, 50 + i), None, **f)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_odd_drafts(dev, probs):
    """Tokens outside the vocabulary, masked ones, a certain target, the draft's own probabilities, u of 0."""
    inf = float("inf")
    v = 700
    logits = _logits(24, v, 10)
    cu = list(range(0, 25, 3))
    tokens, q = _drafts(logits, cu, 11, probs)
    tokens[1], tokens[4], tokens[7] = -1, v, 1 << 40
    logits[9, int(tokens[10])] = -inf                          # refused, whatever u is
    logits[12] = -inf
    logits[12, int(tokens[13])] = 4.0                          # certain
    logits[15] = -inf                                          # no token at all
    logits[18, :] = float("nan")
    logits[18, 3] = 0.0
    tokens[19] = 5
    if probs:
        q[21] = torch.softmax(logits[21], 0)                   # the draft is the target
        q[0] = 0.0
        q[3, :] = 1.0                                          # nothing of the target is above it
    u = _u(24, 12)
    for case in range(3):
        if case:
            u = torch.zeros(24) if case == 1 else torch.full((24,), 1 - 2.0 ** -24)
        _check_verify(dev, logits, tokens, cu, u, _u(8, 13), q)
        _check_verify(dev, logits, tokens, cu, u, torch.zeros(8), q, top_k=30)


def test_verify_refused_top_token(dev):
    """The refused token holds nearly all weight, or is the first of equals, or the last kept one."""
    v = 4000
    x = torch.randn(40, v, generator=torch.Generator().manual_seed(14))
    tokens = torch.zeros(40, dtype=torch.int64)
    for b in range(20):
        r = 2 * b
        if b % 4 == 0:
            x[r, 100 + b] += 12.0 + b
        elif b % 4 == 1:
            x[r] = torch.round(x[r])
        elif b % 4 == 2:
            x[r] = 1.5
        tokens[r + 1] = int(x[r].argmax()) if b % 4 < 3 else int(x[r].topk(50).indices[49])
    cu = list(range(0, 41, 2))
    u = torch.full((40,), 1 - 2.0 ** -24)
    for i, f in enumerate((dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=2))):
        _check_verify(dev, x, tokens, cu, u, _u(20, 15 + i), None, **f)
        _check_verify(dev, x, tokens, cu, u, torch.zeros(20), None, **f)


def test_verify_nothing(dev):
    e = torch.empty
    acc, nxt = sampling.verify(e(0, 9, device=dev), e(0, dtype=torch.int64, device=dev), torch.zeros(4, dtype=torch.int64, device=dev),
                               e(0, device=dev), torch.rand(3, device=dev))
    assert acc.tolist() == [0, 0, 0] and nxt.tolist() == [-1, -1, -1]
    acc, nxt = sampling.verify(e(2, 9, device=dev), torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(1, dtype=torch.int64, device=dev),
                               e(2, device=dev), e(0, device=dev))
    assert acc.shape == (0,)


def test_verify_captured(dev):
    """A padded batch: the sequences of a recorded call change between its replays."""
    rows, v, batch = 12, 20000, 4
    x, u, draw = _logits(rows, v, 16).to(dev), _u(rows, 17).to(dev), _u(batch, 18).to(dev)
    tokens, q = _drafts(x.cpu(), None, 19, True)
    tokens, q = tokens.to(dev), q.to(dev)
    cu = torch.tensor([0, 3, 6, 9, 12], device=dev)
    ws = torch.empty(sampling.verify_workspace_bytes(rows, batch, v, probs=True), dtype=torch.uint8, device=dev)
    out = (torch.empty(batch, dtype=torch.int64, device=dev), torch.empty(batch, dtype=torch.int64, device=dev))
    call = lambda: sampling.verify(x, tokens, cu, u, draw, draft_probs=q, top_p=0.95, workspace=ws, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i, c in enumerate(([0, 3, 6, 9, 12], [0, 1, 1, 7, 8], [0, 0, 0, 0, 0], [0, 12, 12, 12, 12])):
        cu.copy_(torch.tensor(c))
        u.copy_(_u(rows, 60 + i))
        draw.copy_(_u(batch, 70 + i))
        graph.replay()
        got = [t.cpu() for t in out]
        want = _check_verify(dev, x.cpu(), tokens.cpu(), c, u.cpu(), draw.cpu(), q.cpu(), top_p=0.95)
        assert [t.tolist() for t in got] == [want[0], want[1]]


# ---- beams ----------------------------------------------------------------------------------

def _check_beams(dev, logits, scores, width, keep):
    print(f"beams {list(logits.shape)} {logits.dtype} {width} {keep}", flush=True)
    p, t, s = sampling.beams(logits.to(dev), scores.to(dev), width, keep)
    wp, wt, ws = R.beams(logits.float().numpy(), scores.numpy(), width, keep)
    assert np.array_equal(p.cpu().numpy(), wp) and np.array_equal(t.cpu().numpy(), wt)
    got = s.cpu().double().numpy()
    inf = np.isinf(ws)
    assert np.array_equal(got[inf], ws[inf])
    # float32's half step of a sum that is off by no more than 2^-30
    assert (np.abs(got[~inf] - ws[~inf]) <= 2.0 ** -24 * np.abs(ws[~inf]) + 2.0 ** -29).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [3, 50, 2049, 32000, 131072])
def test_beams(dev, dtype, v):
    for groups, width, keep in ((1, 1, 1), (2, 4, 4), (3, 3, 6), (2, 8, 16), (1, 5, 40)):
        _check_beams(dev, _logits(groups * width, v, v + keep, dtype), -9 * _u(groups * width, keep), width, keep)


def test_beams_of_one_score(dev):
    """A search's begin: one beam alive; beams that are copies of each other; a group without any."""
    x = _logits(12, 5000, 31)
    x[4:8] = x[4]
    s = torch.tensor([0.0] + [-float("inf")] * 3 + [-2.0] * 4 + [float("nan"), -float("inf"), -float("inf"), float("nan")])
    _check_beams(dev, x, s, 4, 4)
    _check_beams(dev, x, s, 4, 8)


def test_beams_odd_rows(dev):
    inf = float("inf")
    x = _logits(12, 3000, 33)
    x[0] = -inf                                     # no continuation
    x[1] = -inf
    x[1, 5:8] = 1.0                                 # fewer than wanted
    x[2] = torch.round(x[2])                        # equal ones at the cut
    x[3] -= 200.0
    x[3, 40] = 0.0                                  # the second best is far below what sums count
    x[4] = 0.25
    x[5] = float("nan")
    x[5, 9] = 3.0
    x[6, 8] = inf
    x[7, 1:] = torch.finfo(torch.float32).min
    x[8:12] = -inf                                  # a group of nothing
    s = -_u(12, 34)
    for keep in (1, 4, 7, 60):
        _check_beams(dev, x, s, 4, keep)
        _check_beams(dev, x, s, 1, keep)
    _check_beams(dev, x[:, :40], s, 4, 100)         # more than there are tokens


def test_beams_most(dev):
    _check_beams(dev, _logits(64, 9000, 35, std=0.5), -_u(64, 36), 64, 64)
    _check_beams(dev, _logits(2, 9000, 37), -_u(2, 38), 1, 4096)


def test_beams_captured(dev):
    x, s = _logits(8, 30000, 39).to(dev), (-_u(8, 40)).to(dev)
    ws = torch.empty(sampling.beams_workspace_bytes(8, 30000, 4), dtype=torch.uint8, device=dev)
    out = (torch.empty(8, dtype=torch.int32, device=dev), torch.empty(8, dtype=torch.int64, device=dev), s)
    first = s.clone()
    sampling.beams(x, s, 4, workspace=ws, out=out)
    s.copy_(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.beams(x, s, 4, workspace=ws, out=out)          # the scores are replaced
    s.copy_(first)
    for i in range(4):
        x.copy_(_logits(8, 30000, 41 + i))
        want = sampling.beams(x, s.clone(), 4)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---- together -------------------------------------------------------------------------------

def test_a_loop_of_drafts_draws_and_beams(dev):
    """Prompts, steps with drafted tokens of which some are refused, single draws and a fork by beams, over
    one paged cache with a window and first positions: every step's entries are those of a cache built anew."""
    g = torch.Generator().manual_seed(50)
    batch, page, pages, dim, heads, vocab, width = 4, 8, 400, 64, 4, 300, 2
    emb = torch.randn(vocab, dim, generator=g).bfloat16().to(dev)
    head = (torch.randn(heads * dim, vocab, generator=g) * 0.3).to(dev)
    pool = paged.new_pool(pages, page, dim, "bf16", device=dev)
    state = (torch.full((batch, 40), -1, dtype=torch.int32, device=dev), torch.zeros(batch, dtype=torch.int64, device=dev),
             torch.zeros(pages, dtype=torch.int32, device=dev))
    tables, lens, refs = state
    missing = torch.zeros(1, dtype=torch.int64, device=dev)
    text = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (30, 5, 17, 44)]  # tokens in the cache, the last included
    ref_text = [list(t) for t in text]

    def put(new):
        n = torch.tensor([len(t) for t in new], device=dev)
        cu = torch.tensor(np.concatenate([[0], np.cumsum([len(t) for t in new])]), device=dev)
        paged.grow(*state, n, page, pools=[pool], out=state, missing=missing)
        flat = torch.tensor([t for s in new for t in s], device=dev)
        paged.append(pool, tables, lens, emb[flat], cu=cu, rope=0)
        o, _ = paged.attend(emb[flat][:, None].expand(-1, heads, -1).contiguous(), pool, tables, lens, cu=cu, window=16, first=3, rope=0)
        return flat, cu, o.flatten(1).float() @ head

    def entries():
        assert int(missing) == 0 and lens.tolist() == [len(t) for t in ref_text]
        flat, t = pool.view(-1, dim), tables.cpu()
        for b, text_b in enumerate(ref_text):
            at = [int(t[b, p // page]) * page + p % page for p in range(len(text_b))]
            assert torch.equal(flat[at], emb[torch.tensor(text_b, device=dev)])

    _, cu, logits = put(text)
    tok, _ = sampling.sample(logits[cu[1:] - 1], _u(batch, 51).to(dev), temperature=0.8, top_k=20)
    entries()
    refused = 0
    for step in range(6):
        drafts = [[int(t)] + torch.randint(0, vocab, (n,), generator=g).tolist() for t, n in zip(tok.tolist(), (3, 0, 1, 4))]
        flat, cu, logits = put(drafts)
        # make some drafts good: the first of them the likeliest token of its row
        for b in range(batch):
            if len(drafts[b]) > 1 and step % 2:
                logits[int(cu[b]), drafts[b][1]] += 30.0
        u, draw = _u(len(flat), 60 + step), _u(batch, 70 + step)
        acc, tok = sampling.verify(logits, flat, cu, u.to(dev), draw.to(dev), temperature=0.7, top_p=0.9)
        want = [R.verify(logits[a:z].cpu().numpy(), flat[a:z].tolist(), u[a:z].numpy(), draw[b].item(), temperature=0.7, top_p=0.9)[:2]
                for b, (a, z) in enumerate(zip(cu.tolist(), cu.tolist()[1:]))]
        assert list(zip(acc.tolist(), tok.tolist())) == want
        lens -= cu[1:] - cu[:-1] - 1 - acc
        for b in range(batch):
            ref_text[b] += drafts[b][:1 + int(acc[b])]
            refused += len(drafts[b]) - 1 - int(acc[b])
        entries()
    assert refused > 0
    # two searches of two beams each
    scores = torch.tensor([0.0, -1.0, -0.5, -0.1], device=dev)
    for step in range(4):
        _, _, logits = put([[int(t)] for t in tok.tolist()])
        for b in range(batch):
            ref_text[b].append(int(tok[b]))
        entries()
        want = R.beams(logits.cpu().numpy(), scores.cpu().numpy(), width, width)
        parents, tok, scores = sampling.beams(logits, scores, width)
        assert parents.tolist() == want[0].tolist() and tok.tolist() == want[1].tolist()
        paged.fork(*state, parents, page, out=state)
        ref_text = [list(ref_text[p]) for p in parents.tolist()]
        entries()
