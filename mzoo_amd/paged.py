"""The paged latent cache: many sequences of different lengths in one pool of pages.

The caches of ``mzoo_amd.decode`` give every row the same room; here a sequence holds pages of a
shared pool, and every count lives on the device, so a captured loop appends, grows and attends
without the host:

* ``pool``   ``new_pool(pages, page, dim, fmt)``: FP8-b128 entries, uint8 [P, page, bytes], or bf16
  [P, page, D] (K = V, one latent for all heads, as in ``mzoo_amd.csa2_attn``);
* ``tables`` int32 [B, max_pages]: a sequence's pages in order, -1 where there is none;
* ``lens``   int64 [B]: its tokens;
* ``refs``   int32 [P]: the table entries that name a page (0: free).  Several sequences may share
  pages; only whole tables are shared by ``fork``, and ``grow`` copies a shared last page before
  it is written.

``grow`` makes room and counts the new tokens, ``append`` writes their entries, ``attend`` attends
them; lowering ``lens`` takes refused tokens back; ``fork`` lets sequences begin as copies of others or
end; ``compact`` moves the used pages to the front.  One step of decoding::

    paged.grow(tables, lens, refs, ones, page, pools=pools, out=(tables, lens, refs), missing=missing)
    paged.append(pool, tables, lens, kv)
    o, lse = paged.attend(q, pool, tables, lens, sinks=sinks)

Pages for one layer serve all: ``tables``, ``lens`` and ``refs`` are shared and ``pools`` lists every
layer's.  Packed sequences (``cu``, int64 [B + 1]): rows ``cu[b] .. cu[b + 1] - 1`` are sequence b's.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib, quant
from .csa2_attn import FMT_BF16, FMT_FP8


def new_pool(pages: int, page: int, dim: int, fmt: str = "fp8", *, rope: int = quant.ENTRY_ROPE,
             device="cuda") -> torch.Tensor:
    """An empty pool of ``pages`` pages of ``page`` entries: ``fmt`` "fp8" (the last ``rope`` channels
    in bf16) or "bf16"."""
    if fmt not in ("fp8", "bf16"):
        raise ValueError(f"new_pool: fmt must be 'fp8' or 'bf16', got {fmt!r}")
    if fmt == "bf16":
        return torch.zeros(pages, page, dim, dtype=torch.bfloat16, device=device)
    if dim - rope < 128 or (dim - rope) % 128:
        raise ValueError(f"new_pool: FP8 entries need dim - rope, a multiple of 128, got {dim} - {rope}")
    return torch.zeros(pages, page, quant.entry_bytes(dim - rope, rope), dtype=torch.uint8, device=device)


def _refuse(what: str, name: str, t: torch.Tensor, dt: torch.dtype, shape=None):
    """A tensor is read through a raw pointer, so a wrong dtype or a strided view is rejected, not converted."""
    raise ValueError(f"{what}: {name} must be a contiguous {dt} tensor" + (f" of shape {list(shape)}" if shape is not None else "")
                     + f", got {t.dtype} {list(t.shape)}{'' if t.is_contiguous() else ' (strided)'}")


def _is(t: torch.Tensor, dt: torch.dtype, shape) -> bool:
    return t.dtype == dt and t.shape == shape and t.is_contiguous()


def _table(what: str, tables: torch.Tensor, name: str = "tables") -> tuple[int, int, int]:
    """(rows, pages per row, row stride) of a table, whose rows may be part of wider ones."""
    if tables.dtype != torch.int32 or tables.dim() != 2:
        raise ValueError(f"{what}: {name} must be int32 [B, max_pages], got {tables.dtype} {list(tables.shape)}")
    b, n = tables.shape
    stride, unit = tables.stride()
    if n > 1 and unit != 1 or b > 1 and stride < n:
        raise ValueError(f"{what}: {name} must have unit column stride and rows that do not overlap, got strides {(stride, unit)}")
    return b, n, stride if b > 1 else n


def _one_device(what: str, first: torch.Tensor, *rest) -> None:
    """All tensors on the GPU that holds the first."""
    _lib.require_gpu(first)
    dev = first.device
    for t in rest:
        if t is not None and t.device != dev:
            _lib.require_gpu(t)
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")


def _pool(what: str, pool: torch.Tensor, dim: int, rope: int) -> tuple[int, int, int, int]:
    """(format, nope, pages, entries per page)."""
    if pool.dim() == 3 and pool.is_contiguous():
        pages, page, size = pool.shape
        if page >= 1:
            if pool.dtype == torch.bfloat16 and size == dim:
                return FMT_BF16, dim, pages, page
            nope = dim - rope
            if pool.dtype == torch.uint8 and nope >= 128 and nope % 128 == 0 and rope >= 0 and size == quant.entry_bytes(nope, rope):
                return FMT_FP8, nope, pages, page
    raise ValueError(f"{what}: for {dim} channels ({rope} of them rope) the pool must be contiguous, bf16 [P, page, {dim}] or "
                     f"uint8 FP8-b128 entries, got {pool.dtype} {list(pool.shape)}")


def _call(device: torch.device, name: str, *args) -> None:
    """A call on the device of its tensors and its current stream (the last argument of every entry)."""
    stream = _lib.raw_stream(device)
    if torch.cuda.current_device() == device.index:
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, stream)


def append(pool: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, x: torch.Tensor, *,
           cu: torch.Tensor | None = None, rope: int = quant.ENTRY_ROPE) -> torch.Tensor:
    """The entries of new tokens into their sequences' pages.  x [T, D] (fp32, bf16 or fp16): one
    token per sequence (T == B), or with ``cu`` packed ones; sequence b's n rows become its last n
    entries, positions ``lens[b] - n .. lens[b] - 1`` (``lens`` counts them already).  Positions
    without a page are skipped.  Returns the pool."""
    _one_device("append", pool, tables, lens, x, cu)
    b, width, stride = _table("append", tables)
    if x.dim() != 2:
        raise ValueError(f"append: x must be [T, D], got {list(x.shape)}")
    t, d = x.shape
    fmt, nope, pages, page = _pool("append", pool, d, rope)
    if not _is(lens, torch.int64, (b,)):
        _refuse("append", "lens", lens, torch.int64, (b,))
    if cu is None:
        if t != b:
            raise ValueError(f"append: {t} tokens for {b} sequences; packed tokens need cu")
    elif not _is(cu, torch.int64, (b + 1,)):
        _refuse("append", "cu", cu, torch.int64, (b + 1,))
    row, unit = x.stride()
    if unit != 1 or row < d:
        x = x.contiguous()
        row = d
    _call(pool.device, "mzk_paged_append", x.data_ptr(), _lib.dtype_code(x.dtype), t, row if t > 1 else d, _lib.ptr(cu), b,
          tables.data_ptr(), stride, width, lens.data_ptr(), fmt, d, nope, pool.data_ptr(), pages, page)
    return pool


@functools.lru_cache(maxsize=1024)
def attend_workspace_bytes(tokens: int, heads: int, dim: int, batch: int, packed: bool, max_pages: int | None = None, page: int = 1,
                           window: int = 0, k: int = -1, first: int = 0) -> int:
    """What ``attend`` splits long sequences into: the partial results.  Without ``max_pages`` enough for any
    tables, windows and lists; with it what a call takes whose tables have so many columns (``window`` 0: none;
    ``k``: the positions of its lists, -1: none; ``first``: its first positions), 0 where no sequence is split."""
    n = ctypes.c_int64(0)
    if max_pages is None:
        _lib.call("mzk_paged_attend_workspace_bytes", tokens, heads, dim, int(packed), batch, ctypes.byref(n))
    else:
        _lib.call("mzk_paged_attend_first_workspace_bytes", tokens, heads, dim, int(packed), batch, max_pages, page, window,
                  first, k, ctypes.byref(n))
    return n.value


def attend(q: torch.Tensor, pool: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, *,
           cu: torch.Tensor | None = None, window: int | None = None, first: int = 0, indices: torch.Tensor | None = None,
           sinks: torch.Tensor | None = None, rope: int = quant.ENTRY_ROPE, workspace: torch.Tensor | None = None,
           out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
    """Attention of the newest tokens over their sequences' pages (their own entries appended).

    q bf16 [T, H, D]: one token per sequence, or with ``cu`` the last ``cu[b + 1] - cu[b]`` of each (drafted
    tokens, a chunk of a prompt), each at its own position and causal.  A token sees its sequence up
    to itself, the last ``window`` positions of that and beside them the ``first`` of the sequence, or -- one token per sequence -- the positions
    ``indices`` int32 [B, k] lists (outside the sequence: empty; k 0: none).  Positions on no page or
    past the table are empty.  ``sinks`` fp32 [H].  Returns (o bf16 [T, H, D], lse fp32 [T, H]); rows behind
    the last sequence are 0 (-inf), or as they were in a given ``out`` and ``lse``.  A token that sees
    nothing gets 0.  ``workspace``: uint8, of ``attend_workspace_bytes``, allocated per call if omitted;
    calls that overlap need their own."""
    _one_device("attend", q, pool, tables, lens, cu, indices, sinks, workspace, out, lse)
    if q.dim() != 3 or q.shape[1] < 1:
        raise ValueError(f"attend: q must be [T, H, D], got {list(q.shape)}")
    t, h, d = q.shape
    b, width, stride = _table("attend", tables)
    fmt, nope, pages, page = _pool("attend", pool, d, rope)
    if q.dtype != torch.bfloat16 or not q.is_contiguous():
        _refuse("attend", "q", q, torch.bfloat16)
    if not _is(lens, torch.int64, (b,)):
        _refuse("attend", "lens", lens, torch.int64, (b,))
    if cu is None:
        if t != b:
            raise ValueError(f"attend: {t} tokens for {b} sequences; packed tokens need cu")
    elif not _is(cu, torch.int64, (b + 1,)):
        _refuse("attend", "cu", cu, torch.int64, (b + 1,))
    if sinks is not None and not _is(sinks, torch.float32, (h,)):
        _refuse("attend", "sinks", sinks, torch.float32, (h,))
    if window is not None and (not isinstance(window, int) or window < 1):
        raise ValueError(f"attend: window must be a positive int or None, got {window!r}")
    if not isinstance(first, int) or not 0 <= first < 1 << 30 or first and window is None:
        raise ValueError(f"attend: first must be an int of at least 0, below 2^30, and goes with a window, got {first!r}")
    k = istride = idx = 0
    if indices is not None:
        if cu is not None or window is not None:
            raise ValueError("attend: indices go with one token per sequence and no window")
        rows, k, istride = _table("attend", indices, "indices")
        if rows != b:
            raise ValueError(f"attend: indices must be [{b}, k], got {list(indices.shape)}")
        # a list of no positions has no address either, and none means no list: any other that is never read
        idx = indices.data_ptr() or lens.data_ptr()
    given = out is not None
    if given != (lse is not None):
        raise ValueError("attend: out and lse go together")
    if given:
        if not _is(out, torch.bfloat16, (t, h, d)):
            _refuse("attend", "out", out, torch.bfloat16, (t, h, d))
        if not _is(lse, torch.float32, (t, h)):
            _refuse("attend", "lse", lse, torch.float32, (t, h))
    else:
        out = torch.empty_like(q)
        lse = torch.empty((t, h), dtype=torch.float32, device=q.device)
    wide = min(window or 0, (1 << 63) - 1)
    need = attend_workspace_bytes(t, h, d, b, cu is not None, width, page, wide, k if idx else -1, first)
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
            raise ValueError(f"attend: the workspace must be contiguous uint8 of at least {need} bytes")
    _call(q.device, "mzk_paged_attend_first", q.data_ptr(), t, h, d, _lib.ptr(cu), b, fmt, nope, pool.data_ptr(), pages, page,
          tables.data_ptr(), stride, width, lens.data_ptr(), idx, istride, k, wide, first, _lib.ptr(sinks),
          _lib.ptr(workspace) if need else None, need, out.data_ptr(), lse.data_ptr(), 0 if given else 1)
    return out, lse


# ---- the pages ----------------------------------------------------------------------------

@functools.lru_cache(maxsize=1024)
def workspace_bytes(batch: int, max_pages: int, pages: int) -> int:
    """The workspace of ``grow``, ``fork`` and ``compact``."""
    n = ctypes.c_int64(0)
    _lib.call("mzk_paged_workspace_bytes", batch, max_pages, pages, ctypes.byref(n))
    return n.value


def _workspace(what: str, workspace, need: int, device) -> torch.Tensor:
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"{what}: the workspace must be contiguous uint8 of at least {need} bytes")
    return workspace


def _pool_list(what: str, pools, pages: int, page: int):
    """The pools as C arrays of base pointers and entry bytes, and their number."""
    n = len(pools)
    if n == 0:
        return None, None, 0
    base, size = (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)()
    for i, t in enumerate(pools):
        if t.dim() < 2 or not t.is_contiguous() or t.shape[:2] != (pages, page) or t.numel() == 0:
            raise ValueError(f"{what}: pool {i} must be contiguous [{pages}, {page}, ...], got {list(t.shape)}")
        size[i] = t.stride(1) * t.element_size()
        if size[i] % 4:
            raise ValueError(f"{what}: pool {i} has entries of {size[i]} bytes, not a multiple of 4")
        base[i] = t.data_ptr()
    return base, size, n


def _book(what: str, tables, lens, refs) -> tuple[int, int, int, int]:
    """(sequences, pages per table row, row stride, pages) of a cache's tables, lengths and counts."""
    b, width, stride = _table(what, tables)
    if lens is not None and not _is(lens, torch.int64, (b,)):
        _refuse(what, "lens", lens, torch.int64, (b,))
    if refs.dim() != 1 or refs.dtype != torch.int32 or not refs.is_contiguous():
        _refuse(what, "refs", refs, torch.int32, ("pages",))
    if b == 0 or width == 0 or refs.shape[0] == 0:
        raise ValueError(f"{what}: a pool of no pages, or tables of no rows or width")
    return b, width, stride, refs.shape[0]


def _outs(what: str, out, rows: int, width: int, tables, refs, with_lens: bool):
    """(tables, lens or None, refs, table stride) to write, new ones unless given."""
    if out is None:
        dev = tables.device
        return (torch.empty((rows, width), dtype=torch.int32, device=dev),
                torch.empty(rows, dtype=torch.int64, device=dev) if with_lens else None, torch.empty_like(refs), width)
    got = tuple(out)
    if len(got) != 2 + with_lens:
        raise ValueError(f"{what}: out must be ({'tables, lens, refs' if with_lens else 'tables, refs'})")
    ot, ol, orf = got if with_lens else (got[0], None, got[1])
    _one_device(what, tables, *got)
    r, w, stride = _table(what, ot, "out tables")
    if (r, w) != (rows, width):
        raise ValueError(f"{what}: out tables must be [{rows}, {width}], got {list(ot.shape)}")
    if with_lens and not _is(ol, torch.int64, (rows,)):
        _refuse(what, "out lens", ol, torch.int64, (rows,))
    if not _is(orf, torch.int32, refs.shape):
        _refuse(what, "out refs", orf, torch.int32, refs.shape)
    return ot, ol, orf, stride


def grow(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, tokens: torch.Tensor, page: int, *, pools=(),
         out=None, missing: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """Room for ``tokens`` int64 [B] more tokens of each sequence: the lowest free pages, in the order
    of the sequences.  A partly filled last page that others hold too is replaced by a copy, in every
    one of ``pools`` ([P, page, ...]), for each of its holders that grows.  Either every sequence gets its pages or none
    does.  Returns (tables, lens + tokens, refs, missing): ``missing`` int64 [1] is 0, or the pages that lack, and then
    the rest is unchanged.  ``out=(tables, lens, refs)``, which may be the inputs themselves, is written
    instead of new tensors.

    ``lens`` may be lowered between calls, as for drafted tokens that were refused: the pages behind a
    sequence's tokens stay its own, and the next ``grow`` uses them first (those that others hold too
    it gives up); ``fork`` of a sequence to itself gives them back."""
    _one_device("grow", tables, lens, refs, tokens, missing, workspace, *pools)
    b, width, stride, pages = _book("grow", tables, lens, refs)
    if not _is(tokens, torch.int64, (b,)):
        _refuse("grow", "tokens", tokens, torch.int64, (b,))
    if page < 1:
        raise ValueError(f"grow: page must be at least 1, got {page}")
    if missing is None:
        missing = torch.empty(1, dtype=torch.int64, device=refs.device)
    elif not _is(missing, torch.int64, (1,)):
        _refuse("grow", "missing", missing, torch.int64, (1,))
    base, size, n = _pool_list("grow", pools, pages, page)
    ot, ol, orf, ostride = _outs("grow", out, b, width, tables, refs, True)
    need = workspace_bytes(b, width, pages)
    ws = _workspace("grow", workspace, need, refs.device)
    _call(refs.device, "mzk_paged_grow", tables.data_ptr(), stride, b, width, lens.data_ptr(), refs.data_ptr(), pages,
          tokens.data_ptr(), page, base, size, n, ot.data_ptr(), ostride, ol.data_ptr(), orf.data_ptr(), missing.data_ptr(),
          ws.data_ptr(), need)
    return ot, ol, orf, missing


def fork(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, page: int, *, out=None,
         workspace: torch.Tensor | None = None):
    """Sequences that go on from others' tokens: new sequence i holds the pages of sequence ``parents[i]``
    (int32 [R]; -1: it is empty), and the present ones hold theirs no longer.  Covers beams (any
    parent, any number of times), repeated prompts (R > B), sequences that end (-1).  Returns (tables
    [R, max_pages], lens [R], refs); ``out`` as in ``grow`` (the inputs themselves if R == B)."""
    _one_device("fork", tables, lens, refs, parents, workspace)
    b, width, stride, pages = _book("fork", tables, lens, refs)
    r = parents.shape[0] if parents.dim() == 1 else 0
    if r < 1 or parents.dtype != torch.int32 or not parents.is_contiguous():
        _refuse("fork", "parents", parents, torch.int32, ("R",))
    if page < 1:
        raise ValueError(f"fork: page must be at least 1, got {page}")
    ot, ol, orf, ostride = _outs("fork", out, r, width, tables, refs, True)
    ws, need = None, 0
    if out is not None:
        need = workspace_bytes(b, width, pages)
        ws = _workspace("fork", workspace, need, refs.device)
    _call(refs.device, "mzk_paged_fork", tables.data_ptr(), stride, b, width, lens.data_ptr(), refs.data_ptr(), pages,
          parents.data_ptr(), r, page, ot.data_ptr(), ostride, ol.data_ptr(), orf.data_ptr(), _lib.ptr(ws), need)
    return ot, ol, orf


def compact(tables: torch.Tensor, refs: torch.Tensor, *, pools=(), moved: torch.Tensor | None = None, out=None,
            workspace: torch.Tensor | None = None):
    """The used pages moved to the front of the pools ([P, page, ...]): of U used ones, those behind
    page U - 1, in order, into the free ones before it.  ``moved`` int32 [P] takes where each page's entries are
    now, for what else than ``tables`` holds pages (``moved[p]`` is p where page p stayed).  Returns (tables,
    refs); ``out=(tables, refs)`` may be the inputs."""
    _one_device("compact", tables, refs, moved, workspace, *pools)
    b, width, stride, pages = _book("compact", tables, None, refs)
    page = pools[0].shape[1] if pools and pools[0].dim() >= 2 else 1
    base, size, n = _pool_list("compact", pools, pages, page)
    if moved is not None and not _is(moved, torch.int32, (pages,)):
        _refuse("compact", "moved", moved, torch.int32, (pages,))
    ot, _, orf, ostride = _outs("compact", out, b, width, tables, refs, False)
    need = workspace_bytes(b, width, pages)
    ws = _workspace("compact", workspace, need, refs.device)
    _call(refs.device, "mzk_paged_compact_map", tables.data_ptr(), stride, b, width, refs.data_ptr(), pages, page, base, size, n,
          ot.data_ptr(), ostride, orf.data_ptr(), _lib.ptr(moved), ws.data_ptr(), need)
    return ot, orf
