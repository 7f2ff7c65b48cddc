"""CPU: what the paged cache and packed attention refuse, before anything reaches the GPU."""

import ctypes

import pytest
import torch

from mzoo_amd import _lib, csa2_attn, paged


@pytest.fixture
def fake_gpu(monkeypatch):
    """The argument checks on CPU tensors; a call that passes them must not go further."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)

    def call(name, *args):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(paged, "attend_workspace_bytes", lambda *a: 64)
    monkeypatch.setattr(paged, "workspace_bytes", lambda *a: 64)


def _state(b=2, width=4, pages=8):
    return (torch.full((b, width), -1, dtype=torch.int32), torch.zeros(b, dtype=torch.int64),
            torch.zeros(pages, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    t, n, r = _state()
    pool = paged.new_pool(8, 16, 576, "bf16", device="cpu")
    q = torch.zeros(2, 8, 576, dtype=torch.bfloat16)
    for f in (lambda: paged.append(pool, t, n, q[:, 0]), lambda: paged.attend(q, pool, t, n),
              lambda: paged.grow(t, n, r, n, 16), lambda: paged.fork(t, n, r, torch.zeros(2, dtype=torch.int32), 16),
              lambda: paged.compact(t, r), lambda: csa2_attn.packed(q, q[:, :1], torch.tensor([0, 2]))):
        with pytest.raises(RuntimeError, match="GPU only"):
            f()


def test_new_pool():
    assert paged.new_pool(3, 16, 576, device="cpu").shape == (3, 16, 656)
    assert paged.new_pool(3, 16, 160, rope=32, device="cpu").shape == (3, 16, 196)
    assert paged.new_pool(3, 16, 96, "bf16", device="cpu").dtype == torch.bfloat16
    for bad in (dict(fmt="fp4"), dict(dim=96), dict(dim=200)):
        with pytest.raises(ValueError, match="new_pool"):
            paged.new_pool(3, 16, **{"dim": 576, "fmt": "fp8", "device": "cpu", **bad})


def test_append_refusals(fake_gpu):
    t, n, _ = _state()
    pool = paged.new_pool(8, 16, 576, device="cpu")
    x = torch.zeros(2, 576)
    for args, kw, what in (((pool, t.long(), n, x), {}, "tables"), ((pool, t, n.int(), x), {}, "lens"),
                           ((pool, t, n, torch.zeros(3, 576)), {}, "need cu"), ((pool, t, n, x[0]), {}, r"\[T, D\]"),
                           ((pool, t, n, torch.zeros(2, 160)), {}, "pool"), ((pool[:, :, :600], t, n, x), {}, "pool"),
                           ((pool, t, n, x), dict(cu=torch.zeros(4, dtype=torch.int64)), "cu"),
                           ((pool, t, n, x), dict(cu=torch.zeros(3, dtype=torch.int32)), "cu")):
        with pytest.raises(ValueError, match=what):
            paged.append(*args, **kw)


def test_attend_refusals(fake_gpu):
    t, n, _ = _state()
    pool = paged.new_pool(8, 16, 576, device="cpu")
    q = torch.zeros(2, 8, 576, dtype=torch.bfloat16)
    idx = torch.zeros(2, 5, dtype=torch.int32)
    out, lse = torch.zeros_like(q), torch.zeros(2, 8)
    for args, kw, what in (((q.float(), pool, t, n), {}, "q must be"), ((q[0], pool, t, n), {}, r"\[T, H, D\]"),
                           ((torch.zeros(3, 8, 576, dtype=torch.bfloat16), pool, t, n), {}, "need cu"),
                           ((q, pool, t, n), dict(window=0), "window"), ((q, pool, t, n), dict(window=2.5), "window"),
                           ((q, pool, t, n), dict(indices=idx, window=3), "indices"),
                           ((q, pool, t, n), dict(indices=idx[:1]), "indices"), ((q, pool, t, n), dict(indices=idx.long()), "indices"),
                           ((q, pool, t, n), dict(indices=idx, cu=torch.zeros(3, dtype=torch.int64)), "indices"),
                           ((q, pool, t, n), dict(sinks=torch.zeros(7)), "sinks"), ((q, pool, t, n), dict(out=out), "go together"),
                           ((q, pool, t, n), dict(out=out.float(), lse=lse), "out"), ((q, pool, t, n), dict(out=out, lse=lse[:1]), "lse"),
                           ((q, pool, t, n), dict(workspace=torch.zeros(3, dtype=torch.uint8)), "workspace"),
                           ((q.transpose(0, 1).contiguous().transpose(0, 1), pool, t, n), {}, "strided")):
        with pytest.raises(ValueError, match=what):
            paged.attend(*args, **kw)


def test_pages_refusals(fake_gpu):
    t, n, r = _state()
    par = torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(8, 16, 4)
    for f, what in ((lambda: paged.grow(t, n, r, n.int(), 16), "tokens"), (lambda: paged.grow(t, n, r.long(), n, 16), "refs"),
                    (lambda: paged.grow(t, n, r, n, 0), "page"), (lambda: paged.grow(t, n, r, n, 16, pools=[pool[:4]]), "pool 0"),
                    (lambda: paged.grow(t, n, r, n, 8, pools=[pool]), "pool 0"),
                    (lambda: paged.grow(t, n, r, n, 16, pools=[torch.zeros(8, 16, 3, dtype=torch.uint8)]), "multiple of 4"),
                    (lambda: paged.grow(t, n, r, n, 16, out=(t, n)), "out must be"),
                    (lambda: paged.grow(t, n, r, n, 16, out=(t[:1], n, r)), "out tables"),
                    (lambda: paged.grow(t, n, r, n, 16, missing=torch.zeros(2, dtype=torch.int64)), "missing"),
                    (lambda: paged.grow(t, n, r, n, 16, workspace=torch.zeros(3, dtype=torch.uint8)), "workspace"),
                    (lambda: paged.fork(t, n, r, par.long(), 16), "parents"), (lambda: paged.fork(t, n, r, par[None], 16), "parents"),
                    (lambda: paged.fork(t, n, r, torch.zeros(3, dtype=torch.int32), 16, out=(t, n, r)), "out tables"),
                    (lambda: paged.compact(t, r, pools=[pool[:4]]), "pool 0"), (lambda: paged.compact(t, r, out=(t, n, r)), "out must be")):
        with pytest.raises(ValueError, match=what):
            f()


def test_packed_refusals(fake_gpu):
    q = torch.zeros(5, 8, 160, dtype=torch.bfloat16)
    kv, cu = q[:, :2].contiguous(), torch.tensor([0, 5])
    for args, kw, what in (((q.float(), kv, cu), {}, "bf16"), ((q, kv.float(), cu), {}, "bf16"), ((q, kv[:4], cu), {}, "kv must be"),
                           ((q, q[:, :3].contiguous(), cu), {}, "kv must be"), ((q, kv, cu.int()), {}, "cu"), ((q, kv, cu[None]), {}, "cu"),
                           ((q, kv, cu), dict(window=0), "window"), ((q, kv, cu), dict(out=torch.zeros_like(q)), "go together"),
                           ((q, kv, cu), dict(sinks=torch.zeros(8, dtype=torch.float64)), "sinks")):
        with pytest.raises(ValueError, match=what):
            csa2_attn.packed(*args, **kw)


def test_entry_points_check_their_arguments():
    """The C entries refuse before any HIP call."""
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    odd = ctypes.c_void_p(264)

    def refuse(name, args, text):
        assert getattr(lib, name)(*args) < 0
        assert text in lib.mzk_last_error().decode(), lib.mzk_last_error()

    app = [p, 1, 4, 576, None, 4, p, 8, 8, p, 1, 576, 512, p, 16, 64, None]
    for i, v, text in ((3, 500, "strides"), (5, 3, "without cu"), (7, 4, "strides"), (10, 2, "fmt"), (11, 571, "multiple of 8"),
                       (12, 500, "multiple of 128"), (13, odd, "aligned"), (13, None, "null"), (15, 0, "one entry"), (14, -1, "bad sizes"),
                       (1, 9, "dtype")):
        refuse("mzk_paged_append", app[:i] + [v] + app[i + 1:], text)
    att = [p, 4, 128, 576, None, 4, 1, 512, p, 16, 64, p, 8, 8, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None]
    for i, v, text in ((3, 512, "unsupported latent"), (1, 5, "without cu"), (6, 7, "fmt"), (10, 0, "one entry"), (12, 7, "shorter"),
                       (18, -1, "negative"), (22, None, "null"), (22, odd, "aligned"), (2, 0, "bad sizes")):
        refuse("mzk_paged_attend", att[:i] + [v] + att[i + 1:], text)
    refuse("mzk_paged_attend", att[:15] + [p, 8, 8, 5] + att[19:], "no window")
    refuse("mzk_paged_attend", att[:3] + [80] + att[4:6] + [0] + att[7:], "unsupported head dim")
    pk = [p, 10, 16, 576, p, 3, p, 576, 1, 0, None, p, p, 0, None]
    for i, v, text in ((3, 80, "unsupported"), (8, 3, "divide"), (7, 570, "kv rows"), (9, -2, "window"), (6, None, "null"), (11, odd, "aligned")):
        refuse("mzk_packed_mqa", pk[:i] + [v] + pk[i + 1:], text)
    gr = [p, 8, 4, 8, p, p, 100, p, 16, None, None, 0, p, 8, p, p, p, p, 1 << 20, None]
    for i, v, text in ((1, 3, "strides"), (8, 0, "one entry"), (11, 2, "pool list"), (17, None, "workspace"), (18, 8, "workspace"), (5, None, "null")):
        refuse("mzk_paged_grow", gr[:i] + [v] + gr[i + 1:], text)
    fk = [p, 8, 4, 8, p, p, 100, p, 4, 16, p, 8, p, p, None, 0, None]
    refuse("mzk_paged_fork", fk, "in place")
    refuse("mzk_paged_fork", fk[:9] + [0] + fk[10:], "bad sizes")
    co = [p, 8, 4, 8, p, 100, 16, None, None, 0, p, 8, p, p, 1 << 20, None]
    refuse("mzk_paged_compact", co[:14] + [16] + co[15:], "workspace")
    refuse("mzk_paged_compact", co[:9] + [1] + co[10:], "pool list")


def test_sizes_past_a_launch_are_refused():
    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def refuse(name, args, text):
        assert getattr(lib, name)(*args) < 0
        assert text in lib.mzk_last_error().decode(), lib.mzk_last_error()

    refuse("mzk_paged_attend", [p, 1 << 30, 1, 576, p, 4, 1, 512, p, 16, 64, p, 8, 8, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None], "tokens")
    refuse("mzk_paged_attend", [p, 1 << 24, 128, 576, None, 1 << 24, 1, 512, p, 16, 64, p, 8, 8, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None],
           "too many rows")
    refuse("mzk_paged_attend", [p, 4, 8, 576, None, 4, 1, 512, p, 1 << 26, 64, p, 8, 8, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None], "less than 2^31")
    refuse("mzk_packed_mqa", [p, 1 << 30, 1, 576, p, 3, p, 576, 1, 0, None, p, p, 0, None], "tokens")
    refuse("mzk_packed_mqa", [p, 1 << 29, 1, 64, p, 3, p, 64, 1, 0, None, p, p, 0, None], "too many rows")
    refuse("mzk_paged_append", [p, 1, 1 << 27, 576, p, 4, p, 8, 8, p, 1, 576, 512, p, 16, 64, None], "too many tokens")
    refuse("mzk_paged_grow", [p, 8, 1 << 24, 8, p, p, 100, p, 16, None, None, 0, p, 8, p, p, p, p, 1 << 40, None], "bad sizes")
    refuse("mzk_paged_grow", [p, 8, 0, 8, p, p, 100, p, 16, None, None, 0, p, 8, p, p, p, p, 1 << 40, None], "at least one sequence")
    refuse("mzk_paged_fork", [p, 8, 4, 8, p, p, 100, p, 1 << 24, 16, p, 8, p, p, p, 1 << 40, None], "bad sizes")
    assert lib.mzk_paged_attend(p, 0, 128, 576, None, 0, 1, 512, p, 16, 64, p, 8, 8, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None) == 0


def test_attend_hands_over_an_empty_list(monkeypatch):
    """A list of no positions is a list: its pointer, which an empty tensor lacks, is not null."""
    got = {}
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(paged, "attend_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(paged, "_call", lambda dev, name, *args: got.update(args=args))
    t, n, _ = _state()
    pool = paged.new_pool(8, 16, 576, device="cpu")
    q = torch.zeros(2, 8, 576, dtype=torch.bfloat16)
    for idx, k in ((torch.empty(2, 0, dtype=torch.int32), 0), (torch.zeros(2, 3, dtype=torch.int32)[:, :0], 0),
                   (torch.zeros(2, 3, dtype=torch.int32), 3)):
        paged.attend(q, pool, t, n, indices=idx)
        assert got["args"][15] and got["args"][17] == k
    paged.attend(q, pool, t, n)
    assert not got["args"][15]


def test_room_for_the_new_tokens_positions():
    """Several tokens of a sequence over a table of nearly 2^31 entries would pass 32 bits: refused."""
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    att = [p, 100, 8, 576, p, 4, 1, 512, p, 16, 1, p, 0x7fffffff - 64 - 197, 0x7fffffff - 64 - 197, p, None, 0, 0, 0, None, p, 1 << 40, p, p, 0, None]
    assert lib.mzk_paged_attend(*att) < 0
    assert b"twice the new tokens" in lib.mzk_last_error()
    assert lib.mzk_paged_attend(*att[:12], 0x7fffffff, 0x7fffffff - 63, *att[14:]) < 0
    assert b"less than 2^31" in lib.mzk_last_error()


def test_compact_refuses_other_maps(fake_gpu):
    t, _, r = _state()
    for moved in (torch.zeros(8), torch.zeros(7, dtype=torch.int32), torch.zeros(16, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="moved"):
            paged.compact(t, r, moved=moved)


def test_workspace_of_calls_that_are_not_split():
    """Short tables, windows and lists take no workspace; a call that is split takes no more than any call may."""
    size = paged.attend_workspace_bytes
    most = size(400, 16, 576, 400, False)
    assert most > 100 << 20
    assert size(400, 16, 576, 400, False, 10, 16) == 0
    assert size(400, 16, 576, 400, False, 2000, 16) == most
    assert size(400, 16, 576, 400, False, 2000, 16, 128) == 0
    assert size(400, 16, 576, 400, False, 2000, 16, 0, 256) == 0
    assert size(8, 128, 576, 8, False, 2000, 16, 0, 2048) == size(8, 128, 576, 8, False)
    assert size(8, 128, 576, 8, False, 2000, 16, 0, 0) == 0
    assert size(0, 128, 576, 0, False) == size(8, 128, 576, 0, True, 2000, 16) == 0
    with pytest.raises(_lib.MzkError, match="bad sizes"):
        size(8, 128, 576, 8, False, -1, 16)
