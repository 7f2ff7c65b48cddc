"""GPU: calls of ``mzoo_amd.sampling`` at the ends of what it documents -- tokens too light for the sums, temperatures
at the ends of float32, thousands of sequences, the longest rows, millions of rows -- each way a row is read."""

import numpy as np
import pytest
import torch

from mzoo_amd import sampling
from tests import sampling_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _in_chunks(rows, v, dtype):
    """Whether rows' chunks have workgroups of their own: such calls have a workspace, a workgroup a row has none."""
    return sampling.sample_workspace_bytes(rows, v, dtype) > 0


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
