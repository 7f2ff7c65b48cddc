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
them; ``fork`` lets sequences begin as copies of others or end; ``compact`` moves the used pages to
the front.  One step of decoding::

    paged.grow(tables, lens, refs, ones, page, pools=pools, out=(tables, lens, refs), missing=missing)
    paged.append(pool, tables, lens, kv)
    o, lse = paged.attend(q, pool, tables, lens, sinks=sinks)

Pages for one layer serve all: ``tables``, ``lens`` and ``refs`` are shared and ``pools`` lists every
layer's.  Packed sequences (``cu``, int64 [B + 1]): rows ``cu[b] .. cu[b + 1] - 1`` are sequence b's.
"""

from __future__ import annotations

import ctypes

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


def _check(what: str, *tensors) -> None:
    """(name, tensor, dtype, shape) of contiguous tensors: read through raw pointers, so a wrong dtype or
    a strided view is rejected, not converted."""
    for name, t, dt, shape in tensors:
        if t is None:
            continue
        if t.dtype != dt or not t.is_contiguous() or (shape is not None and tuple(t.shape) != tuple(shape)):
            raise ValueError(f"{what}: {name} must be a contiguous {dt} tensor"
                             + (f" of shape {list(shape)}" if shape is not None else "")
                             + f", got {t.dtype} {list(t.shape)}{'' if t.is_contiguous() else ' (strided)'}")


def _tables(what: str, tables: torch.Tensor, name: str = "tables") -> tuple[int, int, int]:
    """(rows, pages per row, row stride) of a table, whose rows may be part of wider ones."""
    if tables.dim() != 2 or tables.dtype != torch.int32 or (tables.shape[1] > 1 and tables.stride(1) != 1):
        raise ValueError(f"{what}: {name} must be int32 [B, max_pages] with unit column stride, got {tables.dtype} "
                         f"{list(tables.shape)}")
    b, n = tables.shape
    return b, n, max(tables.stride(0), n) if b > 1 else n


def _same_device(what: str, first: torch.Tensor, *rest) -> None:
    for t in rest:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _pool(what: str, pool: torch.Tensor, dim: int, rope: int) -> tuple[int, int, int, int]:
    """(format, nope, pages, entries per page)."""
    if pool.dim() != 3 or not pool.is_contiguous() or pool.shape[1] < 1:
        raise ValueError(f"{what}: the pool must be a contiguous [pages, page, entry] tensor, got {list(pool.shape)}")
    if pool.dtype == torch.bfloat16 and pool.shape[2] == dim:
        return FMT_BF16, dim, pool.shape[0], pool.shape[1]
    nope = dim - rope
    if pool.dtype == torch.uint8 and nope >= 128 and nope % 128 == 0 and pool.shape[2] == quant.entry_bytes(nope, rope):
        return FMT_FP8, nope, pool.shape[0], pool.shape[1]
    raise ValueError(f"{what}: for {dim} channels ({rope} of them rope) the pool must be bf16 [P, page, {dim}] or uint8 "
                     f"FP8-b128 entries, got {pool.dtype} {list(pool.shape)}")


def append(pool: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, x: torch.Tensor, *,
           cu: torch.Tensor | None = None, rope: int = quant.ENTRY_ROPE) -> torch.Tensor:
    """The entries of new tokens into their sequences' pages.  x [T, D] (fp32, bf16 or fp16): one
    token per sequence (T == B), or with ``cu`` packed ones; sequence b's n rows become its last n
    entries, positions ``lens[b] - n .. lens[b] - 1`` (``lens`` counts them already).  Positions
    without a page are skipped.  Returns the pool."""
    _lib.require_gpu(pool, tables, lens, x, cu)
    _same_device("append", pool, tables, lens, x, cu)
    b, width, stride = _tables("append", tables)
    if x.dim() != 2:
        raise ValueError(f"append: x must be [T, D], got {list(x.shape)}")
    t, d = x.shape
    fmt, nope, pages, page = _pool("append", pool, d, rope)
    _check("append", ("lens", lens, torch.int64, (b,)), ("cu", cu, torch.int64, (b + 1,)))
    if cu is None and t != b:
        raise ValueError(f"append: {t} tokens for {b} sequences; packed tokens need cu")
    if x.stride(1) != 1 or x.stride(0) < d:
        x = x.contiguous()
    with torch.cuda.device(pool.device):
        _lib.call("mzk_paged_append", x.data_ptr(), _lib.dtype_code(x.dtype), t, x.stride(0) if t > 1 else d,
                  _lib.ptr(cu), b, tables.data_ptr(), stride, width, lens.data_ptr(), fmt, d, nope, pool.data_ptr(),
                  pages, page, _lib.stream_of(pool))
    return pool


def attend_workspace_bytes(tokens: int, heads: int, dim: int, batch: int, packed: bool) -> int:
    """What ``attend`` splits long sequences into: the partial results (``mzk_paged_attend_workspace_bytes``)."""
    n = ctypes.c_int64(0)
    _lib.call("mzk_paged_attend_workspace_bytes", tokens, heads, dim, int(packed), batch, ctypes.byref(n))
    return n.value


def attend(q: torch.Tensor, pool: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, *,
           cu: torch.Tensor | None = None, window: int | None = None, indices: torch.Tensor | None = None,
           sinks: torch.Tensor | None = None, rope: int = quant.ENTRY_ROPE, workspace: torch.Tensor | None = None,
           out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
    """Attention of the newest tokens over their sequences' pages (their own entries appended).

    q bf16 [T, H, D]: one token per sequence, or with ``cu`` the last ``cu[b + 1] - cu[b]`` of each (drafted
    tokens, a chunk of a prompt), each at its own position and causal.  A token sees its sequence up
    to itself, the last ``window`` positions of that, or -- one token per sequence -- the positions
    ``indices`` int32 [B, k] lists (outside the sequence: empty).  ``sinks`` fp32 [H].  Returns (o bf16
    [T, H, D], lse fp32 [T, H]); rows behind the last sequence are 0 (-inf), or as they were in a
    given ``out`` and ``lse``.  A token that sees nothing gets 0.  ``workspace``: uint8, of
    ``attend_workspace_bytes``, allocated per call if omitted; calls that overlap need their own."""
    _lib.require_gpu(q, pool, tables, lens, cu, indices, sinks, workspace, out, lse)
    _same_device("attend", q, pool, tables, lens, cu, indices, sinks, workspace, out, lse)
    if q.dim() != 3 or q.shape[1] < 1:
        raise ValueError(f"attend: q must be [T, H, D], got {list(q.shape)}")
    t, h, d = q.shape
    b, width, stride = _tables("attend", tables)
    fmt, nope, pages, page = _pool("attend", pool, d, rope)
    _check("attend", ("q", q, torch.bfloat16, None), ("lens", lens, torch.int64, (b,)), ("cu", cu, torch.int64, (b + 1,)),
           ("sinks", sinks, torch.float32, (h,)), ("out", out, torch.bfloat16, (t, h, d)),
           ("lse", lse, torch.float32, (t, h)), ("workspace", workspace, torch.uint8, None))
    if cu is None and t != b:
        raise ValueError(f"attend: {t} tokens for {b} sequences; packed tokens need cu")
    if (out is None) != (lse is None):
        raise ValueError("attend: out and lse go together")
    if window is not None and (not isinstance(window, int) or window < 1):
        raise ValueError(f"attend: window must be a positive int or None, got {window!r}")
    k = istride = 0
    if indices is not None:
        if cu is not None or window is not None:
            raise ValueError("attend: indices go with one token per sequence and no window")
        rows, k, istride = _tables("attend", indices, "indices")
        if rows != b:
            raise ValueError(f"attend: indices must be [{b}, k], got {list(indices.shape)}")
    given = out is not None
    if not given:
        out = torch.empty_like(q)
        lse = torch.empty(t, h, dtype=torch.float32, device=q.device)
    need = attend_workspace_bytes(t, h, d, b, cu is not None)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    if need and workspace.numel() < need:
        raise ValueError(f"attend: the workspace needs {need} bytes, got {workspace.numel()}")
    if t and not b:  # rows of no sequence
        return (out, lse) if given else (out.zero_(), lse.fill_(float("-inf")))
    with torch.cuda.device(q.device):
        _lib.call("mzk_paged_attend", q.data_ptr(), t, h, d, _lib.ptr(cu), b, fmt, nope, pool.data_ptr(), pages, page,
                  tables.data_ptr(), stride, width, lens.data_ptr(), _lib.ptr(indices), istride, k, window or 0,
                  _lib.ptr(sinks), _lib.ptr(workspace), need, out.data_ptr(), lse.data_ptr(), int(not given),
                  _lib.stream_of(q))
    return out, lse


# ---- the pages ----------------------------------------------------------------------------

def workspace_bytes(batch: int, max_pages: int, pages: int) -> int:
    """The workspace of ``grow``, ``fork`` and ``compact``."""
    n = ctypes.c_int64(0)
    _lib.call("mzk_paged_workspace_bytes", batch, max_pages, pages, ctypes.byref(n))
    return n.value


def _workspace(what: str, workspace, batch: int, max_pages: int, refs: torch.Tensor) -> tuple[torch.Tensor, int]:
    need = workspace_bytes(batch, max_pages, refs.numel())
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=refs.device), need
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"{what}: the workspace must be contiguous uint8 of at least {need} bytes")
    return workspace, need


def _pool_list(what: str, pools, refs: torch.Tensor, page: int):
    """The pools as C arrays of base pointers and entry bytes."""
    n = len(pools)
    base, size = (ctypes.c_void_p * max(n, 1))(), (ctypes.c_int64 * max(n, 1))()
    for i, t in enumerate(pools):
        if t.dim() < 2 or not t.is_contiguous() or tuple(t.shape[:2]) != (refs.numel(), page):
            raise ValueError(f"{what}: pool {i} must be contiguous [{refs.numel()}, {page}, ...], got {list(t.shape)}")
        size[i] = t[0, 0].numel() * t.element_size() if t.numel() else 4
        if size[i] % 4:
            raise ValueError(f"{what}: pool {i} has entries of {size[i]} bytes, not a multiple of 4")
        base[i] = t.data_ptr() if t.numel() else None
    return base, size, n if refs.numel() else 0


def _state(what: str, tables, lens, refs, page: int, pools=()) -> tuple[int, int, int]:
    _lib.require_gpu(tables, lens, refs, *pools)
    _same_device(what, tables, lens, refs, *pools)
    b, width, stride = _tables(what, tables)
    _check(what, ("lens", lens, torch.int64, (b,)), ("refs", refs, torch.int32, None))
    if refs.dim() != 1 or page < 1:
        raise ValueError(f"{what}: refs must be [pages] and page at least 1")
    return b, width, stride


def _outs(what: str, out, rows: int, width: int, tables, refs, with_lens: bool):
    """(tables, lens or None, refs) to write, new ones unless given."""
    if out is None:
        new = (torch.empty(rows, width, dtype=torch.int32, device=tables.device),
               torch.empty(rows, dtype=torch.int64, device=tables.device) if with_lens else None, torch.empty_like(refs))
        return (*new, width)
    got = tuple(out)
    if len(got) != 2 + with_lens:
        raise ValueError(f"{what}: out must be ({'tables, lens, refs' if with_lens else 'tables, refs'})")
    ot, ol, orf = got if with_lens else (got[0], None, got[1])
    _lib.require_gpu(*got)
    _same_device(what, tables, *got)
    r, w, stride = _tables(what, ot, "out tables")
    if (r, w) != (rows, width):
        raise ValueError(f"{what}: out tables must be [{rows}, {width}], got {list(ot.shape)}")
    _check(what, ("out lens", ol, torch.int64, (rows,)), ("out refs", orf, torch.int32, tuple(refs.shape)))
    return ot, ol, orf, stride


def grow(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, tokens: torch.Tensor, page: int, *, pools=(),
         out=None, missing: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """Room for ``tokens`` int64 [B] more tokens of each sequence: the lowest free pages, in the order
    of the sequences.  A partly filled last page that others hold too is replaced by a copy, in every
    one of ``pools`` ([P, page, ...]).  Either every sequence gets its pages or none does.  Returns (tables, lens + tokens,
    refs, missing): ``missing`` int64 [1] is 0, or the pages that lack, and then the rest is
    unchanged.  ``out=(tables, lens, refs)``, which may be the inputs themselves, is written instead
    of new tensors."""
    b, width, stride = _state("grow", tables, lens, refs, page, pools)
    _lib.require_gpu(tokens, missing, workspace)
    _same_device("grow", tables, tokens, missing, workspace)
    _check("grow", ("tokens", tokens, torch.int64, (b,)), ("missing", missing, torch.int64, (1,)))
    ot, ol, orf, ostride = _outs("grow", out, b, width, tables, refs, True)
    base, size, n = _pool_list("grow", pools, refs, page)
    ws, need = _workspace("grow", workspace, b, width, refs)
    if missing is None:
        missing = torch.empty(1, dtype=torch.int64, device=refs.device)
    if b == 0:
        missing.zero_()
        if orf is not refs:
            orf.copy_(refs)
        return ot, ol, orf, missing
    if refs.numel() == 0 or width == 0:
        raise ValueError("grow: a pool of no pages, or tables of no width")
    with torch.cuda.device(refs.device):
        _lib.call("mzk_paged_grow", tables.data_ptr(), stride, b, width, lens.data_ptr(), refs.data_ptr(), refs.numel(),
                  tokens.data_ptr(), page, base, size, n, ot.data_ptr(), ostride, ol.data_ptr(), orf.data_ptr(),
                  missing.data_ptr(), ws.data_ptr(), need, _lib.stream_of(refs))
    return ot, ol, orf, missing


def fork(tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, page: int, *, out=None,
         workspace: torch.Tensor | None = None):
    """Sequences that go on from others' tokens: new sequence i holds the pages of sequence ``parents[i]``
    (int32 [R]; -1: it is empty), and the present ones hold theirs no longer.  Covers beams (any
    parent, any number of times), repeated prompts (R > B), sequences that end (-1).  Returns (tables
    [R, max_pages], lens [R], refs); ``out`` as in ``grow`` (the inputs themselves if R == B)."""
    b, width, stride = _state("fork", tables, lens, refs, page)
    _lib.require_gpu(parents, workspace)
    _same_device("fork", tables, parents, workspace)
    if parents.dim() != 1:
        raise ValueError(f"fork: parents must be [R], got {list(parents.shape)}")
    _check("fork", ("parents", parents, torch.int32, None))
    r = parents.shape[0]
    ot, ol, orf, ostride = _outs("fork", out, r, width, tables, refs, True)
    ws = need = None
    if out is not None:
        ws, need = _workspace("fork", workspace, b, width, refs)
    if refs.numel() == 0 or width == 0 or max(b, r) == 0:
        raise ValueError("fork: a pool of no pages, or tables of no rows or width")
    # an empty tensor has no address; nothing of it is read
    some = refs.data_ptr()
    with torch.cuda.device(refs.device):
        _lib.call("mzk_paged_fork", tables.data_ptr() or some, stride, b, width, lens.data_ptr() or some, refs.data_ptr(),
                  refs.numel(), parents.data_ptr() or some, r, page, ot.data_ptr() or some, ostride, ol.data_ptr() or some,
                  orf.data_ptr(), _lib.ptr(ws), need or 0, _lib.stream_of(refs))
    return ot, ol, orf


def compact(tables: torch.Tensor, refs: torch.Tensor, *, pools=(), out=None, workspace: torch.Tensor | None = None):
    """The used pages moved to the front of the pools ([P, page, ...]): of U used ones, those behind
    page U - 1, in order, into the free ones before it.  Returns (tables, refs); ``out=(tables, refs)``
    may be the inputs."""
    _lib.require_gpu(tables, refs, workspace, *pools)
    _same_device("compact", tables, refs, workspace, *pools)
    b, width, stride = _tables("compact", tables)
    _check("compact", ("refs", refs, torch.int32, None))
    if refs.dim() != 1:
        raise ValueError("compact: refs must be [pages]")
    page = pools[0].shape[1] if pools and pools[0].dim() >= 2 else 1
    ot, _, orf, ostride = _outs("compact", out, b, width, tables, refs, False)
    base, size, n = _pool_list("compact", pools, refs, page)
    ws, need = _workspace("compact", workspace, b, width, refs)
    if refs.numel() == 0 or width == 0 or b == 0:
        raise ValueError("compact: a pool of no pages, or tables of no rows or width")
    with torch.cuda.device(refs.device):
        _lib.call("mzk_paged_compact", tables.data_ptr(), stride, b, width, refs.data_ptr(), refs.numel(), page, base, size,
                  n, ot.data_ptr(), ostride, orf.data_ptr(), ws.data_ptr(), need, _lib.stream_of(refs))
    return ot, orf
