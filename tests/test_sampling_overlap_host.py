"""CPU: what ``mzk_beams`` says of scores that are read and written in one launch."""

import ctypes

import pytest
import torch

from mzoo_amd import _lib, sampling


@pytest.mark.parametrize("width,keep,rows,shift,good", [(2, 2, 6, 0, True), (2, 2, 6, 8, False), (2, 2, 6, -8, False), (2, 2, 6, 24, True), (2, 2, 6, -24, True),
                                                        (4, 2, 8, 0, False), (4, 2, 8, 4 * 7, False), (4, 2, 8, 4 * 8, True), (4, 2, 8, -4 * 4, True),
                                                        (1, 3, 2, 0, False), (1, 3, 2, -4 * 6, True), (1, 3, 2, -4 * 5, False), (1, 1, 1, 0, True)])
def test_beams_scores_overlap(width, keep, rows, shift, good):
    """A group's new scores may lie where its old ones were, and no group's where another's are: a call that passes this check
    goes on to the next, which refuses it for its workspace."""
    lib = _lib.load()
    p = ctypes.c_void_p(4096)
    assert lib.mzk_beams(p, 0, rows, 1000, 1000, ctypes.c_void_p(4096), width, keep, p, p, ctypes.c_void_p(4096 + shift), p, 0, None) < 0
    text = lib.mzk_last_error().decode()
    assert ("workspace needs" if good else "out scores") in text, text


def test_beams_scores_overlap_of_tensors(monkeypatch):
    """From the public call, as an error of its arguments."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    x, buf = torch.zeros(8, 9), torch.zeros(12)
    ints = lambda n: (torch.zeros(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int64))  # noqa: E731
    monkeypatch.setattr(sampling, "_bytes", lambda *a: 64)
    monkeypatch.setattr(sampling, "_call", lambda *a: None)
    sampling.beams(x, buf[:8], 4, out=(*ints(8), buf[:8]))
    for keep, n, at in ((4, 8, 2), (2, 4, 0), (2, 4, 4)):
        with pytest.raises(ValueError, match="out scores"):
            sampling.beams(x, buf[:8], 4, keep, out=(*ints(n), buf[at:at + n]))
