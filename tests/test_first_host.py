"""CPU: what attention with first positions refuses, before anything reaches the GPU."""

import ctypes

import pytest
import torch

from mzoo_amd import _lib, csa2_attn, paged


@pytest.mark.parametrize("kw", [dict(first=4), dict(window=8, first=-1), dict(window=8, first=1 << 30), dict(window=8, first=2.0),
                                dict(window=8, first=None)])
def test_refusals(monkeypatch, kw):
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "call", lambda *a: pytest.fail("called"))
    t, n = torch.full((2, 4), -1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    pool = paged.new_pool(8, 16, 576, device="cpu")
    q = torch.zeros(2, 8, 576, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="first"):
        paged.attend(q, pool, t, n, **kw)
    with pytest.raises(ValueError, match="first"):
        csa2_attn.packed(q, q[:, :1].contiguous(), torch.tensor([0, 2]), **kw)


def test_a_list_takes_no_first(monkeypatch):
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    t, n = torch.full((2, 4), -1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="first|indices"):
        paged.attend(torch.zeros(2, 8, 576, dtype=torch.bfloat16), paged.new_pool(8, 16, 576, device="cpu"), t, n,
                     indices=torch.zeros(2, 5, dtype=torch.int32), first=3)


def test_entry_points_check_first():
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    n = ctypes.c_int64(0)
    for window, first in ((0, 3), (5, -1), (5, 1 << 30)):
        args = [p, 4, 128, 576, None, 4, 1, 512, p, 16, 64, p, 8, 8, p, None, 0, 0, window, first, None, p, 1 << 40, p, p, 0, None]
        assert lib.mzk_paged_attend_first(*args) < 0 and b"first positions" in lib.mzk_last_error()
        assert lib.mzk_packed_mqa_first(p, 10, 16, 576, p, 3, p, 576, 1, window, first, None, p, p, 0, None) < 0
        assert b"first positions" in lib.mzk_last_error()
        assert lib.mzk_paged_attend_first_workspace_bytes(4, 128, 576, 0, 4, 100, 64, window, first, -1, ctypes.byref(n)) < 0


def test_workspace_counts_the_first_positions():
    """A window of 12 tiles alone is not split (a token sees its own position in it); with first positions it is."""
    def need(first):
        n = ctypes.c_int64(0)
        _lib.call("mzk_paged_attend_first_workspace_bytes", 1, 128, 576, 0, 1, 10000, 64, 300, first, -1, ctypes.byref(n))
        return n.value
    assert need(0) == 0 and need(10) == 0 and need(1000) > 0
    assert paged.attend_workspace_bytes(1, 128, 576, 1, False, 10000, 64, 300, -1, 1000) == need(1000)
