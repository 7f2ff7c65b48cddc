"""GPU: many calls of ``sample``, ``verify`` and ``beams`` of random sizes, types, ties, masks and settings against the restatements
of ``tests/sampling_ref.py``; rows that lie too near a border for those to decide are passed over and counted."""

import random

import numpy as np
import pytest
import torch

from mzoo_amd import sampling
from tests import sampling_ref as R
from tests.test_gpu_sampling import _check_beams
from tests.test_gpu_sampling_edges import _verify

pytestmark = pytest.mark.gpu
INF = float("inf")


def _rows(rng, rows, v, dtype):
    g = torch.Generator().manual_seed(rng.randrange(1 << 30))
    x = torch.randn(rows, v, generator=g) * rng.choice([0.0, 1e-3, 0.3, 2.5, 2.5, 8, 300])
    if rng.random() < 0.2:
        x = torch.round(x * rng.choice([1, 4, 0.25]))
    if rng.random() < 0.2:
        x = x + rng.choice([100.0, -100.0, 1e4, -3e4])
    if rng.random() < 0.4:                            # a mask
        x[torch.rand(rows, v, generator=g) < rng.choice([0.1, 0.5, 0.9, 0.999])] = rng.choice(
            [-INF, -INF, float("nan"), -1e4, 0.0, torch.finfo(dtype).min, -100.0])
    if rng.random() < 0.2:
        x[:, :max(1, v // 3)] = rng.choice([-INF, -1e4, torch.finfo(dtype).min])
    if rng.random() < 0.3:                            # a few tokens far above the others
        at = torch.randint(0, v, (rows, rng.choice([1, 2, 5])), generator=g)
        far = x.nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True) + rng.choice([10.0, 40.0, 50.0, 60.0])
        x.scatter_(1, at, far + torch.rand(at.shape, generator=g))
    return x.to(dtype), g


def _settings(rng, v):
    return dict(temperature=rng.choice([0.0, 1.0, 1.0, 0.3, 0.8, 1.7, 50.0, 1e-3, 1e-30, INF]), top_k=rng.choice([0, 0, 1, 5, 50, v // 2, v]),
                top_p=rng.choice([1.0, 1.0, 0.9, 0.5, 0.0, rng.random()]), min_p=rng.choice([0.0, 0.0, 0.05, rng.random(), 1.0, 1e-30]))


def _case(seed, most):
    rng = random.Random(seed)
    dtype = rng.choice([torch.float32, torch.bfloat16, torch.float16])
    while True:
        rows = rng.choice([1, 2, 3, 7, 20, 50, 75, 100, 150])
        v = int(2 ** (rng.random() * 17.2)) if rng.random() < 0.8 else rng.choice([16384, 16385, 65536, 65537, 131072])
        if rows * v <= most:
            return (rng, rows, v, dtype, *_rows(rng, rows, v, dtype))


@pytest.mark.parametrize("seed", range(6))
def test_sample(dev, seed):
    seen = near = 0
    for i in range(40):
        rng, rows, v, dtype, x, g = _case(1000 * seed + i, 6_000_000)
        f = _settings(rng, v)
        u = torch.rand(rows, generator=g)
        if rng.random() < 0.2:
            u[torch.rand(rows, generator=g) < 0.5] = rng.choice([0.0, 2.0 ** -24, 1 - 2.0 ** -24])
        off = rng.choice([0, 0, 1, 3])
        wide = torch.empty(rows, v + off + rng.choice([0, 5]), dtype=dtype, device=dev)
        wide[:, off:off + v] = x.to(dev)
        print(f"sample {seed} {i}: {rows} rows of {v} {dtype} at {off} {f}", flush=True)
        token, lp = [t.tolist() for t in sampling.sample(wide[:, off:off + v], u.to(dev), **f)]
        for row in rng.sample(range(rows), min(rows, max(2, 100000 // v))):
            want, want_lp, clear = R.sample(x[row].float().numpy(), u[row].item(), **f)
            seen += 1
            if not clear:
                near += 1
                continue
            assert token[row] == want, f"row {row}: {token[row]}, expected {want}"
            assert want < 0 or abs(lp[row] - want_lp) <= 2.0 ** -24 * abs(want_lp) + 2.0 ** -29, f"row {row}: {lp[row]} {want_lp}"
    assert near <= seen // 20, (seen, near)


@pytest.mark.parametrize("seed", range(6))
def test_verify(dev, seed):
    seen = near = 0
    for i in range(30):
        rng, rows, v, dtype, x, g = _case(1000 * seed + i + 500, 2_000_000)
        f = _settings(rng, v)
        cu = [0]
        while cu[-1] < rows and len(cu) < 200:
            cu.append(min(rows, cu[-1] + rng.choice([0, 1, 2, 5])))
        batch = len(cu) - 1
        q = torch.softmax(x.float().nan_to_num(-1e9, posinf=1e4, neginf=-1e9) / 1.5, 1) if rng.random() < 0.5 else None
        u, draw = torch.rand(rows, generator=g), torch.rand(batch, generator=g)
        if rng.random() < 0.3:
            u[torch.rand(rows, generator=g) < 0.5] = 0.0
        if q is not None and rng.random() < 0.3:
            q = q * 1e-25                             # a draft that is sure of other tokens
        tokens = torch.randint(0, v, (rows,), generator=g)
        likely = torch.rand(rows, generator=g) < rng.choice([0.7, 0.7, 0.1])
        tokens[likely] = x.float().nan_to_num(-INF).argmax(1).roll(1)[likely]
        print(f"verify {seed} {i}: {rows} rows of {v} {dtype}, {batch} sequences, probs {q is not None} {f}", flush=True)
        acc, nxt = [t.tolist() for t in sampling.verify(x.to(dev), tokens.to(dev), torch.tensor(cu, device=dev), u.to(dev), draw.to(dev),
                                                        draft_probs=None if q is None else q.to(dev), **f)]
        for b in rng.sample(range(batch), min(batch, max(2, 100000 // v))):
            a, z = cu[b], cu[b + 1]
            if a == z:
                assert (acc[b], nxt[b]) == (0, -1), f"sequence {b}"
                continue
            n, want, clear = _verify(x[a:z].float().numpy(), tokens[a:z].tolist(), u[a:z].numpy(), draw[b].item(),
                                     None if q is None else q[a:z].numpy(), **f)
            seen += 1
            if not clear:
                near += 1
                continue
            assert (acc[b], nxt[b]) == (n, want), f"sequence {b}: {acc[b]}, {nxt[b]}; expected {n}, {want}"
    assert near <= seen // 5, (seen, near)


@pytest.mark.parametrize("seed", range(2))
def test_beams(dev, seed):
    for i in range(12):
        rng, rows, v, dtype, x, g = _case(1000 * seed + i + 800, 1_000_000)
        width = rng.choice([d for d in (1, 2, 3, 5) if rows % d == 0])
        if width == 1 or not bool(((x == x[:, :1]).all(1)).any()):  # (beams of equal values: equal to more bits than a double has)
            _check_beams(dev, x, -5 * torch.rand(rows, generator=g), width, rng.choice([1, 4, 17]))


def test_the_restatements_differ(dev):
    """The comparison sees a token that is wrong: another u is another token."""
    x = torch.randn(40, 900, generator=torch.Generator().manual_seed(1))
    got = sampling.sample(x.to(dev), torch.full((40,), 0.3, device=dev))[0].tolist()
    assert sum(got[i] != R.sample(x[i].numpy(), 0.7)[0] for i in range(40)) > 30
    assert np.array_equal(got, [R.sample(x[i].numpy(), 0.3)[0] for i in range(40)])
