"""GPU: calls of ``mzoo_amd.sampling`` at the ends of what it documents -- tokens too light for the sums, temperatures
at the ends of float32, thousands of sequences, the longest rows, millions of rows -- each way a row is read."""

import numpy as np
import pytest
import torch

from mzoo_amd import sampling
from tests import sampling_ref as R
from tests.test_gpu_sampling import _u
from tests.test_gpu_sampling_rows import MANY, _check_near, _hard

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _in_chunks(rows, v, dtype):
    """Whether rows' chunks have workgroups of their own: such calls have a workspace, a workgroup a row has none."""
    return sampling.sample_workspace_bytes(rows, v, dtype) > 0


def _verify(logits, tokens, u, draw, probs=None, **filters):
    """One sequence, as ``R.verify``, also where probabilities are far below 2^-28.  A drafted token is accepted if u q W < w; w is off by at most
    2^-45 of itself (2^-51 of its power, 2^-52 of at most 1100 of its exponent), W by less than 2^-29 of itself: the
    comparison is sure unless u q and p are within 2^-28 of p.  What a refused token's row has above the draft is off by V 2^-52 of its units
    and by W's part of p: V 2^-51 of what is dropped and 512 roundings of V 2^-62 of it, V 2^-50 in all; V 2^-49 is below 2^-28 of their sum,
    where ``R.pick`` takes a border as near, if that is V 2^-20 or more."""
    n, v, clear = len(tokens), logits.shape[1], True
    for i in range(n):
        order, w, sure = R.kept(logits[i], **filters)
        clear &= sure
        if i == n - 1:
            break
        d = int(tokens[i + 1])
        at = np.flatnonzero(order == d) if 0 <= d < v else []
        p = w[at[0]] / w.sum() if len(at) else np.longdouble(0)
        q = 1.0 if probs is None or not 0 <= d < v else float(probs[i][d])
        a = np.longdouble(float(np.float32(u[i]))) * np.longdouble(q)
        if p < np.longdouble(2) ** -1100:             # below the numbers of 64 bits
            p = np.longdouble(0)
        clear &= not (0 < p < 2.0 ** -1000 and a < 2.0 ** -900) and not (p > 0 and abs(a - p) <= 2.0 ** -28 * p and not p == q == 1)
        if a < p:
            continue
        if probs is None:
            if p < 1:
                order, w = order[order != d], w[order != d]
        elif order.size:
            left = np.zeros(v, np.longdouble)
            left[order] = w / w.sum()
            left = np.maximum(left - np.asarray(probs[i], np.float64).astype(np.longdouble), 0)
            if left.sum() > 0:
                clear &= bool(left.sum() >= v * 2.0 ** -20)
                order, w = np.arange(v), left
        break
    token, sure = R.pick(order, w, draw)
    return i, token, clear and sure


# ---- tokens too light for the sums ------------------------------------------------------------

@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype,v,sequences,chunks", [
    (torch.float32, 64, 6, False), (torch.float32, 9001, 80, False), (torch.float32, 70001, 8, True),
    (torch.float16, 700, 6, False), (torch.float16, 70001, 8, True),
    (torch.bfloat16, 700, 6, False), (torch.bfloat16, 70001, 8, True),
    (torch.bfloat16, 20001, 80, False),               # counted by value
    (torch.bfloat16, 131072, 80, False)])             # and a value whose number passes 16 bits
def test_verify_top_k_ends_among_light_tokens(dev, dtype, v, sequences, chunks, probs):
    """3 tokens hold the sums, all others together less than 2^-80: which of them top-k keeps decides what is accepted
    at ``u`` (or a draft's probability) of next to nothing."""
    assert _in_chunks(2 * sequences, v, dtype) == chunks
    g = torch.Generator().manual_seed(v)
    heavy = torch.randperm(v, generator=g)[:3]
    x = torch.full((2 * sequences, v), -100.0)
    x[:, ::2] = -90.0                                 # before the others
    x[:, heavy] = 0.0
    x[1::2] = -float("inf")
    x[1::2, 5] = 1.0                                  # the token behind an accepted one
    order = np.argsort(-x[0].numpy(), kind="stable")
    k = torch.tensor([4, 5, 3 + v // 4, v // 2 + 9, v - 1, 0])[torch.arange(2 * sequences) // 2 % 6].int()
    at = torch.tensor([3, 5, 3 + v // 4, v // 2 + 8, v - 1, v - 1])[torch.arange(sequences) % 6]
    at -= torch.arange(sequences) // 6 % 2            # the place before: kept, if that one is not
    tokens = torch.zeros(2 * sequences, dtype=torch.int64)
    tokens[1::2] = torch.from_numpy(order)[at]
    cu = torch.arange(0, 2 * sequences + 1, 2)
    u = torch.full((2 * sequences,), 0.5 if probs else 0.0)
    draw = torch.rand(sequences, generator=g)
    q = torch.full((2 * sequences, v), 2.0 ** -149) if probs else None  # 2^-150 of u q: below p of 2^-130 and 2^-145
    acc, nxt = sampling.verify(x.to(dtype).to(dev), tokens.to(dev), cu.to(dev), u.to(dev), draw.to(dev),
                               draft_probs=None if q is None else q.to(dev), top_k=k.to(dev))
    acc, nxt = acc.tolist(), nxt.tolist()
    for b in range(sequences):
        if k[2 * b] == 0 or at[b] < k[2 * b]:
            assert (acc[b], nxt[b]) == (1, 5), f"sequence {b}: place {at[b]} of {k[2 * b]} kept ones: {acc[b]}, {nxt[b]}"
            continue
        among, w, clear = R.kept(x[2 * b].numpy(), top_k=int(k[2 * b]))
        if probs:
            left = np.zeros(v, np.longdouble)
            left[among] = w / w.sum()
            among, w = np.arange(v), np.maximum(left - 2.0 ** -149, 0)
            w[w < 0.25] = 0                           # units of 2^-52
        token, sure = R.pick(among, w, draw[b].item())
        assert clear and sure
        assert (acc[b], nxt[b]) == (0, token), f"sequence {b}: place {at[b]} of {k[2 * b]} kept ones: {acc[b]}, {nxt[b]}"


@pytest.mark.parametrize("dtype,v,sequences,chunks", [
    (torch.float32, 1000, 6, False), (torch.float32, 9001, 80, False), (torch.float32, 70001, 8, True), (torch.float16, 700, 6, False),
    (torch.float16, 70001, 8, True), (torch.bfloat16, 700, 6, False), (torch.bfloat16, 70001, 8, True), (torch.bfloat16, 20001, 80, False),
    (torch.bfloat16, 131072, 80, False)])
def test_verify_nothing_above_the_draft_but_light_tokens(dev, dtype, v, sequences, chunks):
    """One token holds the sum; the others are each 1 to 2 units of what a target has above a draft, and top-k keeps some of them, of which
    the draft is sure: what is left is nothing, and the next token is the one that holds the sum."""
    assert _in_chunks(2 * sequences, v, dtype) == chunks
    light = -35.5                                     # e^-35.5 = 1.72 2^-52: below what is counted, above 2^-52
    x = torch.full((2 * sequences, v), light)
    x[:, 7] = 0.0
    order = torch.argsort(-x[0], stable=True)
    k = torch.tensor([2, 3, 40, 500])[torch.arange(2 * sequences) // 2 % 4].int()
    q = torch.zeros(2 * sequences, v)
    for row in range(2 * sequences):
        q[row, order[:k[row]]] = 1.0
    tokens = torch.full((2 * sequences,), v)          # no token: refused
    cu = torch.arange(0, 2 * sequences + 1, 2)
    u, draw = torch.rand(2 * sequences, generator=torch.Generator().manual_seed(v)), torch.rand(sequences, generator=torch.Generator().manual_seed(v + 1))
    acc, nxt = sampling.verify(x.to(dtype).to(dev), tokens.to(dev), cu.to(dev), u.to(dev), draw.to(dev), draft_probs=q.to(dev), top_k=k.to(dev))
    assert acc.tolist() == [0] * sequences
    assert nxt.tolist() == [7] * sequences


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("probs", [False, True])
def test_verify_light_tokens_one_after_another(dev, dtype, probs):
    """Sequences of 150 tokens, each of which only its place says is kept: up to the first that is not, or is refused otherwise."""
    v, n, k = 3000, 150, 40
    g = torch.Generator().manual_seed(5)
    row = torch.full((v,), -60.0)
    row[torch.randperm(v, generator=g)[:2]] = 0.0
    order = np.argsort(-row.numpy(), kind="stable")
    x = row.expand(4 * n, v).to(dtype)
    tokens = torch.from_numpy(order)[torch.randint(2, k, (4 * n,), generator=g)]
    tokens[n + 71] = int(order[k])                    # behind top-k's end
    tokens[2 * n + 100], tokens[2 * n + 101] = v, int(order[k])  # no token, before that
    tokens[3 * n + 3] = int(order[-1])
    u = torch.full((4 * n,), 0.5 if probs else 0.0)
    q = torch.full((4 * n, v), 2.0 ** -140) if probs else None
    acc, nxt = sampling.verify(x.to(dev), tokens.to(dev), torch.arange(0, 4 * n + 1, n, device=dev), u.to(dev), torch.full((4,), 0.75, device=dev),
                               draft_probs=None if q is None else q.to(dev), top_k=k)
    assert acc.tolist() == [n - 1, 70, 99, 2]
    heavy = sorted(order[:2].tolist())
    assert nxt.tolist() == [heavy[1]] * 4             # by the order and by the index alike: equal ones


def test_verify_next_tokens_over_the_tokens(dev):
    """A call's next tokens may be written where its tokens were: 64 sequences of a drafted token that only its place says is kept,
    or not, over and over."""
    v, k, n = 5000, 20, 64
    x = torch.full((2 * n, v), -60.0)
    x[:, 7] = 0.0
    order = torch.argsort(-x[0], stable=True)
    tokens = order[torch.arange(2 * n) // 2 % (2 * k) + 1].to(dev)  # the places 1 .. 2 k of the order
    want = [1 if i % (2 * k) + 1 < k else 0 for i in range(n)]
    cu, zero = torch.arange(0, 2 * n + 1, 2, device=dev), torch.zeros(2 * n, device=dev)
    there, acc = x.to(dev), torch.empty(n, dtype=torch.int64, device=dev)
    for _ in range(20):
        mine = tokens.clone()
        sampling.verify(there, mine, cu, zero, zero[:n], top_k=k, out=(acc, mine[n // 2:n // 2 + n]))
        assert acc.tolist() == want
        assert mine[n // 2:n // 2 + n].tolist() == [7] * n


# ---- temperatures at the ends of float32 ------------------------------------------------------

ENDS = [1.401298464324817e-45, 1e-30, 1e-3, 0.01, 1e30, 3.4028234663852886e38, float("inf")]


def _sharp(rows, v, dtype, seed):
    """Rows whose largest logit lies low in its octave, high, at the ends of the type and below 0."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * 2.5
    top = torch.finfo(dtype).max
    for i, m in enumerate((40.0, 33.0, 63.5, 0.0, -17.0, top, 1e-4, -1e-4)):
        x[i] = torch.minimum(x[i], torch.tensor(min(m, 60000.0))) if m >= 0 else -x[i].abs() + m
        x[i, 7 + 1000 * i] = m
    x[8] = -float("inf")
    x[8, v - 3] = -top
    x[9, ::2] = float("nan")
    return x.to(dtype)


@pytest.mark.parametrize("dtype,rows,v,chunks", [(torch.bfloat16, 80, 17000, False), (torch.bfloat16, 80, 131072, False),
                                                 (torch.float16, 160, 17000, False), (torch.float32, 160, 17000, False),
                                                 (torch.bfloat16, 10, 131072, True), (torch.float16, 10, 131072, True),
                                                 (torch.float32, 10, 131072, True)])
def test_temperatures_at_the_ends(dev, dtype, rows, v, chunks):
    assert _in_chunks(rows, v, dtype) == chunks
    x = _sharp(rows, v, dtype, v)
    see, host = 10, x.float().numpy()
    u = torch.rand(rows, generator=torch.Generator().manual_seed(1))
    for t in ENDS:
        for f in (dict(), dict(top_k=20, top_p=0.9), dict(min_p=0.5)):
            print(f"{rows} rows of {v} {dtype} temperature {t} {f}", flush=True)
            token, lp = [r.tolist() for r in sampling.sample(x.to(dev), u.to(dev), temperature=t, **f)]
            for i in range(see):
                want, want_lp, clear = R.sample(host[i], u[i].item(), temperature=t, **f)
                assert clear, f"row {i}: a border is near"
                assert token[i] == want, f"row {i}: {token[i]}, expected {want}"
                assert abs(lp[i] - want_lp) <= 2.0 ** -24 * abs(want_lp) + 2.0 ** -29, f"row {i}: {lp[i]} {want_lp}"


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype,rows,v", [(torch.bfloat16, 80, 17000), (torch.float16, 12, 70000), (torch.float32, 12, 20000)])
def test_verify_at_the_ends_of_temperature(dev, dtype, rows, v, probs):
    x = _sharp(rows, v, dtype, v)
    cu = [0, 2, 4, 6, 8, 10, rows]
    tokens = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(2))
    tokens[1:10:4] = x.float().nan_to_num(-9e9).argmax(1)[0:9:4]
    q = torch.softmax(x.float().clamp(-1e4, 1e4).nan_to_num(-1e4), 1) if probs else None
    u, draw = torch.rand(rows, generator=torch.Generator().manual_seed(3)), torch.rand(6, generator=torch.Generator().manual_seed(4))
    for t in ENDS:
        print(f"verify {rows} rows of {v} {dtype} temperature {t} probs {probs}", flush=True)
        acc, nxt = sampling.verify(x.to(dev), tokens.to(dev), torch.tensor(cu, device=dev), u.to(dev), draw.to(dev),
                                   draft_probs=None if q is None else q.to(dev), temperature=t)
        for b in range(5):
            a, z = cu[b], cu[b + 1]
            n, token, clear = _verify(x[a:z].float().numpy(), tokens[a:z].tolist(), u[a:z].numpy(), draw[b].item(),
                                      None if q is None else q[a:z].numpy(), temperature=t)
            assert clear, f"sequence {b}: a border is near"
            assert (int(acc[b]), int(nxt[b])) == (n, token), f"sequence {b}: {int(acc[b])}, {int(nxt[b])}; expected {n}, {token}"


# ---- thousands of sequences ---------------------------------------------------------------------

def _best_us(f):
    f()
    torch.cuda.synchronize()
    best = float("inf")
    for _ in range(5):
        a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        z.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(z) * 1e3)
    return best


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("batch", [63, 64, 65, 4095, 4096, 4097, 9000])
def test_verify_thousands_of_sequences(dev, batch, probs):
    """Empty ones among them, at both ends and in runs longer than a wave."""
    v, g = 40, torch.Generator().manual_seed(batch)
    n = torch.randint(0, 4, (batch,), generator=g)
    n[:batch // 16] = 0
    n[batch // 2:batch // 2 + batch // 8] = 0
    n[-batch // 20:] = 0
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    rows = int(cu[-1]) + 5                            # five rows of no sequence
    x = torch.randn(rows, v, generator=g)
    tokens = x.argmax(1).roll(1)
    other = torch.rand(rows, generator=g) < 0.3
    tokens[other] = torch.randint(0, v, (int(other.sum()),), generator=g)
    q = torch.softmax(x + 0.3 * torch.randn(rows, v, generator=g), 1) if probs else None
    u, draw = torch.rand(rows, generator=g), torch.rand(batch, generator=g)
    acc, nxt = sampling.verify(x.to(dev), tokens.to(dev), cu.to(dev), u.to(dev), draw.to(dev), draft_probs=None if q is None else q.to(dev))
    acc, nxt = acc.tolist(), nxt.tolist()
    unclear = 0
    for b, (a, z) in enumerate(zip(cu.tolist(), cu[1:].tolist())):
        if a == z:
            assert (acc[b], nxt[b]) == (0, -1), f"sequence {b}"
            continue
        token, want, clear = _verify(x[a:z].numpy(), tokens[a:z].tolist(), u[a:z].numpy(), draw[b].item(), None if q is None else q[a:z].numpy())
        if not clear:                                 # (with the draft's probabilities: little is left above it)
            unclear += 1
            continue
        assert (acc[b], nxt[b]) == (token, want), f"sequence {b}: {acc[b]}, {nxt[b]}; expected {token}, {want}"
    assert unclear <= batch // 50
    assert set(acc) == {0, 1, 2} or batch < 100       # a sequence has at most two drafted tokens


def test_verify_finds_a_rows_sequence_in_few_steps(dev):
    """Of 65536 sequences.  (7.4 times the time of sampling the same rows, where each row walked through them.)"""
    rows, v = 65536, 64
    x, u = torch.randn(rows, v, device=dev), torch.rand(rows, device=dev)
    cu, tokens = torch.arange(rows + 1, device=dev), torch.zeros(rows, dtype=torch.int64, device=dev)
    verify = _best_us(lambda: sampling.verify(x, tokens, cu, u, u, top_p=0.9))
    sample = _best_us(lambda: sampling.sample(x, u, top_p=0.9))
    print(f"verify {verify:.0f} us, sample {sample:.0f} us", flush=True)
    assert verify < 3 * sample
    assert torch.equal(sampling.verify(x, tokens, cu, u, u, top_p=0.9)[1], sampling.sample(x, u, top_p=0.9)[0])


# ---- the most rows, the longest rows --------------------------------------------------------------

MOST = (1 << 22) - 1


def test_the_most_rows(dev):
    """2^22 - 1 rows of 3 logits; one more is refused."""
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(MOST, 3, device=dev, generator=g)
    u = torch.rand(MOST, device=dev, generator=g)
    tokens, lp = sampling.sample(x, u, temperature=0.7)
    w, order = (x.double() / float(np.float32(0.7))).softmax(1).sort(1, descending=True)
    sums = w.cumsum(1)
    at = (sums <= u.double()[:, None]).sum(1).clamp(max=2)
    clear = (sums[:, :2] - u.double()[:, None]).abs().amin(1) > 2.0 ** -28
    assert int(clear.sum()) > MOST - 20
    assert torch.equal(tokens[clear], order.gather(1, at[:, None])[:, 0][clear])
    want = w.gather(1, at[:, None])[:, 0].log()
    assert bool(((lp.double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -30)[clear].all())
    with pytest.raises(RuntimeError, match="too many rows"):
        sampling.sample(torch.zeros(MOST + 1, 3, device=dev), torch.zeros(MOST + 1, device=dev))

    # sequences of 3 rows, and beams, of all rows as of the second half alone
    drafted = torch.randint(0, 3, (MOST,), device=dev, generator=g)
    cu = torch.arange(0, MOST + 1, 3, device=dev)
    batch = cu.shape[0] - 1
    half = batch // 2
    draw = torch.rand(batch, device=dev, generator=g)
    q = torch.randn(MOST, 3, device=dev, generator=g).softmax(1)
    for probs in (None, q):
        acc, nxt = sampling.verify(x, drafted, cu, u, draw, draft_probs=probs)
        part = sampling.verify(x[3 * half:], drafted[3 * half:], cu[half:] - 3 * half, u[3 * half:], draw[half:],
                               draft_probs=None if probs is None else probs[3 * half:])
        assert torch.equal(acc[half:], part[0]) and torch.equal(nxt[half:], part[1])
        assert acc.unique().tolist() == [0, 1, 2] and nxt.unique().tolist() == [0, 1, 2]
    got = sampling.beams(x, -u, 3)
    part = sampling.beams(x[3 * half:], -u[3 * half:], 3)
    assert torch.equal(got[0][3 * half:], part[0] + 3 * half) and torch.equal(got[1][3 * half:], part[1]) and torch.equal(got[2][3 * half:], part[2])


@pytest.mark.parametrize("dtype,rows,chunks", [(torch.float32, 2, True), (torch.float32, 140, False), (torch.bfloat16, 2, True),
                                               (torch.bfloat16, 70, False), (torch.float16, 2, True), (torch.float16, 140, False)])
def test_the_longest_rows(dev, dtype, rows, chunks):
    """Of 2^20 logits, the last of which the largest; two rows of it are looked at, of which one begins masked."""
    v = 1 << 20
    assert _in_chunks(rows, v, dtype) == chunks
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(2, v, generator=g) * 2.0).to(dtype)
    x[1, :v // 2] = -float("inf")
    x[:, v - 1] = 17.0
    there = x[torch.arange(rows) % 2].to(dev)
    u = torch.rand(rows, generator=g)
    for f in (dict(top_p=0.9), dict(top_k=2000, temperature=1.4), dict(min_p=1e-4), dict()):
        print(f"{rows} rows of {v} {dtype} {f}", flush=True)
        token, lp = [r.tolist() for r in sampling.sample(there, u.to(dev), **f)]
        for i in range(2):
            want, want_lp, clear = R.sample(x[i].float().numpy(), u[i].item(), **f)
            assert clear, f"row {i}: a border is near"
            assert token[i] == want, f"row {i}: {token[i]}, expected {want}"
            # float32's half step, and the logarithm of W, which is off by less than 2^-29 of itself
            assert abs(lp[i] - want_lp) <= 2.0 ** -24 * abs(want_lp) + 2.0 ** -29, f"row {i}: {lp[i]} {want_lp}"
    with pytest.raises(RuntimeError, match="at most"):
        sampling.sample(torch.zeros(1, v + 1, device=dev), torch.zeros(1, device=dev))


# ---- hard rows, each way they are read ------------------------------------------------------------

EACH_WAY = [(torch.float32, 20000, 73, False), (torch.float32, 150000, 21, True), (torch.float32, 150000, 146, False),
            (torch.float16, 20000, 73, False), (torch.float16, 70000, 21, True), (torch.float16, 70000, 146, False),
            (torch.float16, 150000, 21, True), (torch.float16, 150000, 146, False),
            (torch.bfloat16, 16384, 73, False), (torch.bfloat16, 20000, 73, False), (torch.bfloat16, 150000, 21, True),
            (torch.bfloat16, 150000, 73, False)]


def _hard_filters(v):
    return dict(), dict(top_k=1000), dict(min_p=0.3), dict(temperature=0.0), dict(top_k=v - v // 20, temperature=1.5)


def _hard_case(v, dtype, rows):
    x, plain = _hard(v, dtype)
    of = torch.arange(rows) % MANY
    return x[of], plain[:21], _u(rows, v + 70)


@pytest.mark.parametrize("dtype,v,rows,chunks", EACH_WAY)
def test_hard_rows_each_way(dev, dtype, v, rows, chunks):
    """Masks, ties, the ends of the type, values whose number passes 16 bits: a workgroup a row, and in chunks, of each type."""
    assert _in_chunks(rows, v, dtype) == chunks
    x, plain, u = _hard_case(v, dtype, rows)
    for f in _hard_filters(v):
        print(f"{rows} rows of {v} {dtype} {f}", flush=True)
        token, lp = sampling.sample(x.to(dev), u.to(dev), **f)
        _check_near([token[:21].cpu(), lp[:21].cpu()], plain, u[:21], f)
