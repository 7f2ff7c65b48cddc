"""CPU: what ``mzoo_amd.sampling`` refuses before anything reaches the GPU, and its restatement against closed forms."""

import ctypes

import numpy as np
import pytest
import torch

from mzoo_amd import _lib, sampling
from tests import sampling_ref as R


@pytest.fixture
def fake_gpu(monkeypatch):
    """The argument checks on CPU tensors; a call that passes them must not go further."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)

    def call(name, *args):
        raise AssertionError(f"{name} was called")
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(sampling, "_bytes", lambda *a: 64)


def test_cpu_tensors_are_refused():
    x, u = torch.zeros(4, 9), torch.zeros(4)
    cu = torch.tensor([0, 4])
    for f in (lambda: sampling.sample(x, u), lambda: sampling.verify(x, cu.new_zeros(4), cu, u, u[:1]), lambda: sampling.beams(x, u, 2)):
        with pytest.raises(RuntimeError, match="GPU only"):
            f()


def test_sample_refusals(fake_gpu):
    x, u = torch.zeros(4, 9), torch.zeros(4)
    nan = float("nan")
    for args, kw, what in (((x[0], u), {}, r"\[rows, V\]"), ((x[:, :0], u), {}, r"\[rows, V\]"), ((x, u[:3]), {}, "u must"), ((x, u.double()), {}, "u must"),
                           ((x, u), dict(temperature=-0.1), "temperature"), ((x, u), dict(temperature=nan), "temperature"),
                           ((x, u), dict(temperature=u.double()), "temperature"), ((x, u), dict(temperature=u[:2]), "temperature"),
                           ((x, u), dict(top_k=-1), "top_k"), ((x, u), dict(top_k=2.0), "top_k"), ((x, u), dict(top_k=1 << 31), "top_k"),
                           ((x, u), dict(top_k=torch.zeros(4, dtype=torch.int64)), "top_k"), ((x, u), dict(top_p=1.1), "top_p"),
                           ((x, u), dict(top_p="0.9"), "top_p"), ((x, u), dict(min_p=-0.5), "min_p"), ((x, u), dict(min_p=nan), "min_p"),
                           ((x, u), dict(out=(u,)), "out must be"), ((x, u), dict(out=(u, u)), "out tokens"),
                           ((x, u), dict(out=(torch.zeros(4, dtype=torch.int64), u.double())), "out logprobs"),
                           ((x, u), dict(workspace=torch.zeros(3, dtype=torch.uint8)), "workspace"),
                           ((x, u), dict(workspace=torch.zeros(64)), "workspace"),
                           ((x, torch.zeros(8)[::2]), {}, "strided")):
        with pytest.raises(ValueError, match=what):
            sampling.sample(*args, **kw)
    with pytest.raises(TypeError, match="dtype"):
        sampling.sample(x.double(), u)


def test_verify_refusals(fake_gpu):
    x, u, t, cu, d = torch.zeros(6, 9), torch.zeros(6), torch.zeros(6, dtype=torch.int64), torch.tensor([0, 2, 6]), torch.zeros(2)
    for args, kw, what in (((x, t[:5], cu, u, d), {}, "tokens"), ((x, t.int(), cu, u, d), {}, "tokens"), ((x, t, cu.int(), u, d), {}, "cu"),
                           ((x, t, cu[:0], u, d), {}, "cu"), ((x, t, cu[None], u, d), {}, "cu"), ((x, t, cu, u[:2], d), {}, "u must"),
                           ((x, t, cu, u, u), {}, "draw"), ((x, t, cu, u, d), dict(draft_probs=x[:5]), "draft_probs"),
                           ((x, t, cu, u, d), dict(draft_probs=x.bfloat16()), "draft_probs"), ((x, t, cu, u, d), dict(top_p=d), "top_p"),
                           ((x, t, cu, u, d), dict(out=(t[:2], d)), "out next"), ((x, t, cu, u, d), dict(workspace=t), "workspace")):
        with pytest.raises(ValueError, match=what):
            sampling.verify(*args, **kw)


def test_beams_refusals(fake_gpu):
    x, s = torch.zeros(6, 9), torch.zeros(6)
    for args, kw, what in (((x, s, 4), {}, "no groups"), ((x, s, 0), {}, "no groups"), ((x, s, 2.0), {}, "no groups"), ((x, s, 2, 0), {}, "keep"),
                           ((x, s, 3, 2000), {}, "keep"), ((x, s[:5], 2), {}, "scores"), ((x, s.double(), 2), {}, "scores"),
                           ((x, s, 2), dict(out=(s, s, s)), "out parents"), ((x, s, 2), dict(out=(s,)), "out must be")):
        with pytest.raises(ValueError, match=what):
            sampling.beams(*args, **kw)


def test_entry_points_check_their_arguments():
    """The C entries refuse before any HIP call."""
    lib = _lib.load()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)
    n = ctypes.c_int64(0)

    def refuse(name, args, text):
        assert getattr(lib, name)(*args) < 0
        assert text in lib.mzk_last_error().decode(), lib.mzk_last_error()

    big = 1 << 40
    sm = [p, 0, 4, 100000, 100000, p, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, p, big, None]
    for i, v, text in ((0, None, "null"), (0, odd, "misaligned"), (1, 7, "dtype"), (2, -1, "bad sizes"), (2, 1 << 22, "too many rows"), (3, 0, "bad sizes"),
                       (3, (1 << 20) + 1, "at most"), (4, 99999, "overlap"), (5, None, "null"), (14, None, "null"), (15, None, "null"), (16, None, "workspace needs"),
                       (16, ctypes.c_void_p(264), "misaligned"), (17, 8, "workspace needs")):
        refuse("mzk_sample", sm[:i] + [v] + sm[i + 1:], text)
    assert lib.mzk_sample(None, 0, 0, 1000, 1000, *sm[5:14], None, None, None, 0, None) == 0   # no rows
    vf = [p, 0, 6, 1000, 1000, p, p, 2, p, p, None, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, p, p, p, big, None]
    for i, v, text in ((0, None, "null"), (5, None, "null"), (6, None, "null"), (7, -1, "bad sizes"), (7, 1 << 22, "bad sizes"), (8, None, "null"),
                       (9, None, "null"), (20, None, "null"), (23, 8, "workspace needs"), (2, -2, "bad sizes")):
        refuse("mzk_verify", vf[:i] + [v] + vf[i + 1:], text)
    refuse("mzk_verify", vf[:10] + [p, 999] + vf[12:], "overlap")
    bm = [p, 0, 6, 1000, 1000, p, 2, 2, p, p, p, p, big, None]
    for i, v, text in ((6, 4, "no groups"), (6, 0, "at least 1"), (7, 0, "at least 1"), (7, 4096, "at most"), (5, None, "null"), (8, None, "null"),
                       (12, 8, "workspace needs"), (1, 3, "dtype")):
        refuse("mzk_beams", bm[:i] + [v] + bm[i + 1:], text)
    for f, args in (("sample", (4, 100000, 0)), ("verify", (4, 2, 100000, 0, 1)), ("beams", (4, 100000, 0, 2))):
        assert getattr(lib, f"mzk_{f}_workspace_bytes")(*args, ctypes.byref(n)) == 0 and n.value > 0
        assert getattr(lib, f"mzk_{f}_workspace_bytes")(*args, None) < 0
        assert getattr(lib, f"mzk_{f}_workspace_bytes")(4, *args[1:-2], 1 << 30, *args[-1:], ctypes.byref(n)) < 0


def test_restatement():
    """Probabilities that are known: 1/2, 1/4, 1/8, 1/8."""
    x = np.log(np.array([1.0, 4.0, 2.0, 1.0]))
    draws = lambda **f: [R.sample(x, u, **f)[0] for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 0.99)]  # noqa: E731
    assert draws() == [1, 1, 2, 2, 0, 0, 3, 3]
    assert draws(top_k=2) == [1, 1, 1, 2, 2, 2, 2, 2] and draws(temperature=0.0) == [1] * 8
    assert draws(top_p=0.6) == draws(top_k=2) and draws(top_p=0.8) == draws(top_k=3) and draws(top_p=0.0) == [1] * 8
    assert draws(min_p=0.3) == draws(top_k=2) and draws(min_p=0.2) == draws()
    assert abs(R.sample(x, 0.7)[1] - np.log(0.25)) < 1e-15
    rows = np.stack([x, x])
    assert R.verify(rows, [9, 2], [0.2, 0], 0.6)[:2] == (1, 2) and R.verify(rows, [9, 2], [0.3, 0], 0.6)[:2] == (0, 1)
    q = np.array([[0.0, 0.0, 1.0, 0.0]] * 2)
    assert R.verify(rows, [9, 2], [0.3, 0], 0.6, q)[:2] == (0, 1) and R.verify(rows, [9, 2], [0.3, 0], 0.1, q)[:2] == (0, 0)
    p, t, s = R.beams(rows, np.array([0.0, -0.5]), 2, 3)
    assert p.tolist() == [0, 1, 0] and t.tolist() == [1, 1, 2] and np.allclose(s, [np.log(0.5), np.log(0.5) - 0.5, np.log(0.25)])
