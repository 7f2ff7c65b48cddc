"""GPU: the ways a row is read -- bf16 rows counted by value, rows in chunks, rows of one workgroup, too many tokens
for the list -- against the restatements of ``tests/sampling_ref.py``, on rows that are hard for each."""

import numpy as np
import pytest
import torch

from mzoo_amd import sampling
from tests import sampling_ref as R
from tests.test_gpu_sampling import _check_beams, _check_sample, _check_verify, _drafts, _logits, _u

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
MANY = 73                                             # rows: more than are read in chunks, of bf16 of any length


def _of_each(rows, seed):
    """Settings of each row: all filters and their absence, in turn."""
    g = torch.Generator().manual_seed(seed)
    on = torch.rand(4, rows, generator=g) < 0.6
    return dict(temperature=torch.where(on[0], 0.3 + 1.5 * torch.rand(rows, generator=g), torch.ones(rows)),
                top_k=torch.where(on[1], torch.randint(1, 3000, (rows,), generator=g), torch.zeros(rows, dtype=torch.int64)).int(),
                top_p=torch.where(on[2], torch.rand(rows, generator=g), torch.ones(rows)),
                min_p=torch.where(on[3], 0.2 * torch.rand(rows, generator=g), torch.zeros(rows)))


def _hard(v, dtype):
    """MANY bf16 or fp16 rows: values whose number passes 16 bits among them."""
    inf, nan, top = float("inf"), float("nan"), torch.finfo(dtype).max
    g = torch.Generator().manual_seed(v)
    x = _logits(MANY, v, v + 1, dtype)
    most = int(v * 0.9)
    at = torch.randperm(v, generator=g)
    x[0] = -inf
    x[1] = nan
    x[2, at[:most]] = -inf                            # a masked vocabulary
    x[3, at[:most]] = torch.finfo(dtype).min
    x[4, at[:most]] = nan
    x[5] = 0.5
    x[6, at[:most]] = 1.0                             # most tokens equal, and they count
    x[7, at[:most]] = -90.0                           # and they do not
    x[8, at[:most]] = 0.0
    x[8, at[:most:2]] = -0.0
    x[9, at[:most]] = inf
    x[9, at[0]] = top
    x[10] = -inf
    x[10, v - 1] = -1.0                               # the only one
    x[11] = -top
    x[12] = (x[12].float() * 1e-40).to(dtype)         # subnormal
    x[13, at[:65536]] = x[13, 0].item()               # 65535, 65536, 65537 and their like of one value
    x[14, at[:65535]] = x[14, 0].item()
    x[15, at[:131072]] = x[15, 0].item()
    x[16, at[:65536]], x[16, at[65536:131072]] = 1.0, -1.0
    x[17, at[:most]] = -inf
    x[17, at[most:]] = 3.0
    x[18] = torch.round(x[18])                        # cuts among equal ones
    x[19] = torch.where(torch.rand(v, generator=g) < 0.5, 2.0, -2.0).to(dtype)
    x[20] = 1e-5
    x[20, ::3] = -0.0
    return x, torch.where(x == inf, top, x)


def _check_near(got, plain, u, filters):
    """As ``_check_sample``; but of a row whose draw is within 2^-28 of the sum W of a border each token whose part of the
    running sums [before, upto] meets u W -+ 2^-28 W is right: one running sum is off by less than 2^-29 W (the
    restatements' header: less than 2^-29 of the largest weight, and W is at least that), and so is u times the
    other, W, so that the kernel's token is among those.  Its cuts have to be clear."""
    for i in range(len(u)):
        logits = plain[i].float().numpy()
        token, want, clear = R.sample(logits, u[i].item(), **filters)
        at, lp = got[0][i].item(), got[1][i].item()
        if not clear:
            order, w, sure = R.kept(logits, **filters)
            assert sure, f"row {i}: a cut is near"
            sums = np.cumsum(w) / w.sum()
            x, eps = float(u[i]), 2.0 ** -28
            right = order[(sums >= x - eps) & (sums - w / w.sum() <= x + eps)].tolist()
            assert at in right, f"row {i}: token {at}, expected one of {right}"
            want = float(np.log(w[order == at][0] / w.sum()))
        else:
            assert at == token, f"row {i}: token {at}, expected {token}"
        if at >= 0:
            assert abs(lp - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -29, f"row {i}: {lp} {want}"
        else:
            assert lp == -np.inf


@pytest.mark.parametrize("v", [16385, 30001, 131072])
def test_sample_by_value(dev, v):
    for seed in range(2):
        x = _logits(MANY, v, v + seed, torch.bfloat16)
        _check_sample(dev, x, _u(MANY, seed), **_of_each(MANY, seed))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [20000, 70000, 150000])
def test_sample_hard_rows(dev, v, dtype):
    x, plain = _hard(v, dtype)
    rows = 21
    filters = (dict(), dict(top_k=1000), dict(min_p=0.3), dict(temperature=0.0), dict(top_k=v - v // 20, temperature=1.5))
    for i, f in enumerate(filters):
        u = _u(MANY, v + i)
        for n in (MANY, rows):                        # a workgroup a row; in chunks
            print(f"{n} rows of {v} {dtype} {f}", flush=True)
            on = {k: torch.full((n,), val, dtype=torch.int32 if k == "top_k" else torch.float32, device=dev) for k, val in f.items()}
            got = sampling.sample(x[:n].to(dev), u[:n].to(dev), **f)
            same = sampling.sample(x[:n].to(dev), u[:n].to(dev), **on)
            assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
            _check_near([t[:rows].cpu() for t in got], plain[:rows], u[:rows], f)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_verify_hard_rows(dev, dtype, probs):
    """Drafted tokens among equal ones at a cut, in masked rows, and of values whose number passes 16 bits."""
    v = 70000
    _, x = _hard(v, dtype)
    cu = list(range(0, 21, 3)) + [MANY]
    tokens, q = _drafts(x.float().clamp(-100, 100).nan_to_num(-100.0), cu, 3, probs)
    g = torch.Generator().manual_seed(4)
    for i, f in enumerate((dict(top_k=1000), dict(top_k=30000, temperature=0.9), dict(min_p=0.3), dict())):
        for row in range(1, MANY):                    # one of the row's largest: kept or not by its index alone
            if row % 2 and not torch.isnan(x[row - 1]).all():
                best = torch.nonzero(x[row - 1] == x[row - 1][~torch.isnan(x[row - 1])].max())[:, 0]
                tokens[row] = best[torch.randint(0, len(best), (1,), generator=g)]
        _check_verify(dev, x, tokens, cu, _u(MANY, 5 + i), _u(len(cu) - 1, 15 + i), q, **f)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_ties_at_the_cut(dev, probs):
    """Each equal token around the one at which top-k ends, as the drafted one."""
    v, k = 20011, 50
    x = torch.zeros(2 * MANY, v)
    x[:, ::7] = 4.0
    x[:, 3::700] = 6.0
    x[:, 5] = float("nan")
    x = x.bfloat16()
    order = torch.argsort(-x[0].float().nan_to_num(-9e9), stable=True)
    cu = list(range(0, 2 * MANY + 1, 2))
    tokens = torch.zeros(2 * MANY, dtype=torch.int64)
    tokens[1::2] = order[k - MANY // 2 - 2:k + MANY // 2 - 1] if k > MANY // 2 + 2 else order[:MANY]
    q = torch.softmax(x.float().nan_to_num(-9e9), 1) if probs else None
    acc, _ = _check_verify(dev, x, tokens, cu, _u(2 * MANY, 1) * (0.1 if probs else 0.01), _u(MANY, 2), q, top_k=k)
    assert 0 < sum(acc) < MANY


@pytest.mark.parametrize("v", [17000, 90000])
def test_beams_hard_rows(dev, v):
    _, x = _hard(v, torch.bfloat16)
    x = torch.cat([x, x[:7]])
    for width, keep in ((4, 4), (1, 60), (8, 300)):
        _check_beams(dev, x, -_u(80, keep), width, keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [5, 150])
def test_sample_too_many_for_the_list(dev, dtype, rows):
    v = 70001
    x = (1.0 + 0.004 * torch.randn(rows, v, generator=torch.Generator().manual_seed(rows))).to(dtype)
    for i, f in enumerate((dict(), dict(top_k=40000), dict(top_p=0.6), dict(min_p=0.995), dict(top_k=60000, top_p=0.5, min_p=0.9))):
        if dtype != torch.float32 and "top_p" in f:
            f = {k: t for k, t in f.items() if k != "top_p"}
        _check_sample(dev, x[:5], _u(rows, i)[:5], given=x.to(dev)[:5], **f)
        want = sampling.sample(x[:5].to(dev), _u(rows, i)[:5].to(dev), **f)
        got = sampling.sample(x.to(dev), _u(rows, i).to(dev), **f)
        assert torch.equal(got[0][:5], want[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_sample_a_late_maximum(dev, dtype, rows):
    """The first logits say nothing of the largest, which comes last, or among them lie all of a chunk's."""
    v, low = 66003, -6e4 if dtype == torch.float16 else -3e38
    x = _logits(rows, v, 77, dtype)
    x[0, :1500] = low
    x[1, :v - 20] = low
    x[2, 1024:] -= 500.0
    x[2, v - 1] = 600.0
    for i, f in enumerate((dict(), dict(top_p=0.9, temperature=0.7), dict(top_k=30, min_p=0.01))):
        _check_sample(dev, x[:3], _u(3, i), **f)
        want = sampling.sample(x[:3].to(dev), _u(3, i).to(dev), **f)
        u = torch.cat([_u(3, i), _u(rows - 3, 5)])
        assert torch.equal(sampling.sample(x.to(dev), u.to(dev), **f)[0][:3], want[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, MANY])
def test_rows_anywhere_in_memory(dev, dtype, rows):
    """Rows that begin and end at any element, with what lies beside them larger than all of theirs."""
    v = 40003
    for off in (0, 1, 3, 7):
        wide = torch.full((rows, v + 24), 1000.0, dtype=dtype)
        wide[:, off:off + v] = _logits(rows, v, off, dtype)
        mine = wide.to(dev)[:, off:off + v]
        _check_sample(dev, wide[:, off:off + v], _u(rows, off), given=mine, top_p=0.9, top_k=2000)


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_calls_at_once(dev, dtype):
    """On two streams, each with its own workspace, over and over."""
    v = 66000
    x = [_logits(rows, v, rows, dtype).to(dev) for rows in (6, 90)]
    u = [_u(len(t), 8).to(dev) for t in x]
    want = [sampling.sample(t, r, top_p=0.9, temperature=0.8) for t, r in zip(x, u)]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sampling.sample(x[i], u[i], top_p=0.9, temperature=0.8))
    torch.cuda.synchronize()
    for i in range(2):
        for token, lp in got[i]:
            assert torch.equal(token, want[i][0]) and torch.equal(lp, want[i][1])


def test_many_rows_captured(dev):
    """Rows counted by value in a graph, with others' eager calls between its replays."""
    rows, v = 80, 40000
    x, u = _logits(rows, v, 1, torch.bfloat16).to(dev), _u(rows, 2).to(dev)
    out = torch.empty(rows, dtype=torch.int64, device=dev), torch.empty(rows, device=dev)
    sampling.sample(x, u, top_p=0.8, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampling.sample(x, u, top_p=0.8, out=out)
    for i in range(3):
        x.copy_(_logits(rows, v, 5 + i, torch.bfloat16))
        want = sampling.sample(x, u, top_p=0.8)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [20000, 99991])
def test_sample_runs_of_values(dev, v, dtype):
    """Runs of one value after another, of any length, between other tokens: counts of values change over within the row."""
    g = torch.Generator().manual_seed(v)
    x = _logits(MANY, v, v, dtype)
    values = torch.tensor([-float("inf"), 0.0, -0.0, 1.5, -2.0, 3.0, float("nan"), torch.finfo(dtype).min])
    for row in range(12):
        at = 0
        while at < v:
            n = int(2 ** (16 * torch.rand(1, generator=g)))
            if row % 2 == 0 or torch.rand(1, generator=g) < 0.5:
                x[row, at:at + n] = values[torch.randint(0, 8, (1,), generator=g)].to(dtype)
            at += n
    for row in range(12, 16):                         # some of each everywhere
        some = torch.rand(v, generator=g) < 0.2 * (row - 11)
        x[row, some] = values[torch.randint(0, 8, (int(some.sum()),), generator=g)].to(dtype)
    for i, f in enumerate((dict(), dict(top_k=500), dict(min_p=0.1), dict(temperature=0.5))):
        u = _u(MANY, v + i)
        print(f"{v} {dtype} {f}", flush=True)
        got = sampling.sample(x.to(dev), u.to(dev), **f)
        _check_near([t[:20].cpu() for t in got], x[:20], u[:20], f)
    _check_beams(dev, x[:16], -_u(16, 1), 4, 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [2, 150])
def test_sample_equal_logits_behind_a_mask(dev, dtype, rows):
    """All weights 1, and none among a row's first logits: borders that are hit exactly."""
    v, n = 46130, 15430
    x = torch.full((rows, v), -float("inf"))
    x[:, v - 2 * n::2] = -100.0
    x = x.to(dtype)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(3))
    u[0], u[1] = 0.5, 0.25
    for t in (1.7, 0.3, 1.0, 77.0):
        for f in (dict(top_p=0.5), dict(), dict(top_p=0.25, top_k=n // 2 * 2), dict(top_p=0.75, min_p=1.0), dict(top_k=8192)):
            _check_sample(dev, x[:2], u[:2], temperature=t, **f)
            if rows > 2:
                got = sampling.sample(x.to(dev), u.to(dev), temperature=t, **f)
                for i in range(0, rows, 7):
                    assert got[0][i].item() == R.sample(x[i].float().numpy(), u[i].item(), temperature=t, **f)[0]
