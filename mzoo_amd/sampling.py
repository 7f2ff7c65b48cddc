"""From a model's logits to the next tokens: draws, the verification of drafted tokens, beams.

What stands between a step of ``mzoo_amd.paged`` and the next one:

* ``sample``  tokens drawn behind temperature, top-k, top-p and min-p: the next ``append``'s;
* ``verify``  how many drafted tokens of each sequence stay (``lens`` is lowered by the others) and the
  token behind them;
* ``beams``   which continuations a beam search keeps: ``fork``'s parents, and their tokens.

Random numbers are inputs, and so everything is reproducible: the same call gives the same bits.  The same row gives the
same token in any batch, unless its random number times the sum is within 2^-29 of the sum (bf16 rows of more than 2^17
logits: 2^-27) from a border between two tokens: how many rows there are decides how weights are summed.  Calls read
lengths and settings on the device and never synchronise, so a step is captured once::

    o, lse = paged.attend(q, pool, tables, lens, cu=cu)          # the newest tokens, drafted ones among them
    accepted, token = sampling.verify(head(o), tokens, cu, u, draw, temperature=0.8, top_p=0.95)
    lens -= cu[1:] - cu[:-1] - 1 - accepted                      # refused tokens are taken back

A row's tokens stand in the order of falling logits, equal ones by rising index.  ``temperature`` divides the
logits; ``top_k`` keeps the first k tokens of the order; ``top_p`` the fewest of those that hold that share of
their probability; ``min_p`` those of at least that share of the first one's.  Each is a number for all
rows, a tensor of one for each row (float32; ``top_k`` int32), or None: off.  Temperature 0 takes the
first token of the order.  NaN and -inf are no tokens; +inf counts as the largest finite number of its type.

Logits are fp32, bf16 or fp16 [rows, V], V at most 2^20, rows of wider tensors among them.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .paged import _call, _is, _one_device, _refuse, _workspace


def _logits(what: str, logits: torch.Tensor):
    """(logits, rows, vocabulary, row stride)."""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{what}: logits must be [rows, V], got {list(logits.shape)}")
    _lib.dtype_code(logits.dtype)
    rows, v = logits.shape
    stride, unit = logits.stride()
    if v > 1 and unit != 1 or rows > 1 and stride < v:
        logits = logits.contiguous()
        stride = v
    return logits, rows, v, stride if rows > 1 else v


def _filter(what: str, name: str, f, rows: int, off, most):
    """(tensor or None, its pointer, number for all rows)."""
    dt = torch.int32 if name == "top_k" else torch.float32
    if torch.is_tensor(f):
        if not _is(f, dt, (rows,)):
            _refuse(what, name, f, dt, (rows,))
        return f, f.data_ptr(), off
    if f is None:
        return None, None, off
    if name == "top_k":
        good = isinstance(f, int) and 0 <= f < 1 << 31
    else:
        good = isinstance(f, (int, float)) and 0 <= f <= most
    if not good:
        raise ValueError(f"{what}: {name} must be None, a tensor of {dt} [{rows}] or " + (
            "an int of at least 0" if name == "top_k" else f"a number from 0 to {most}") + f", got {f!r}")
    return None, None, f


def _filters(what: str, rows: int, temperature, top_k, top_p, min_p):
    """The tensors among them, and the arguments of a call."""
    tensors, args = [], []
    for name, f, off, most in (("temperature", temperature, 1.0, float("inf")), ("top_k", top_k, 0, None),
                               ("top_p", top_p, 1.0, 1.0), ("min_p", min_p, 0.0, 1.0)):
        t, p, x = _filter(what, name, f, rows, off, most)
        tensors.append(t)
        args += [p, x]
    return tensors, args


def _out(what: str, out, names, shapes_dtypes, device):
    """The given outputs, checked, or new ones."""
    if out is None:
        return tuple(torch.empty(shape, dtype=dt, device=device) for shape, dt in shapes_dtypes)
    got = tuple(out)
    if len(got) != len(names):
        raise ValueError(f"{what}: out must be ({', '.join(names)})")
    for name, t, (shape, dt) in zip(names, got, shapes_dtypes):
        if not _is(t, dt, shape):
            _refuse(what, f"out {name}", t, dt, shape)
    _one_device(what, *got)
    if got[0].device != device:
        raise ValueError(f"{what}: tensors on {device} and {got[0].device}")
    return got


@functools.lru_cache(maxsize=1024)
def _bytes(entry: str, *args) -> int:
    n = ctypes.c_int64(0)
    _lib.call(entry, *args, ctypes.byref(n))
    return n.value


def sample_workspace_bytes(rows: int, vocab: int, dtype: torch.dtype = torch.float32) -> int:
    """The workspace of ``sample``."""
    return _bytes("mzk_sample_workspace_bytes", rows, vocab, _lib.dtype_code(dtype))


def verify_workspace_bytes(rows: int, batch: int, vocab: int, dtype: torch.dtype = torch.float32, probs: bool = False) -> int:
    """The workspace of ``verify``, with or without ``draft_probs``."""
    return _bytes("mzk_verify_workspace_bytes", rows, batch, vocab, _lib.dtype_code(dtype), int(probs))


def beams_workspace_bytes(rows: int, vocab: int, keep: int, dtype: torch.dtype = torch.float32) -> int:
    """The workspace of ``beams``."""
    return _bytes("mzk_beams_workspace_bytes", rows, vocab, _lib.dtype_code(dtype), keep)


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=None, top_k=None, top_p=None, min_p=None,
           workspace: torch.Tensor | None = None, out=None):
    """A token for each row of ``logits`` [B, V], drawn with ``u`` fp32 [B], random numbers of [0, 1): the
    first of the tokens that the filters leave, in their order, at which the running sum of their
    probabilities exceeds ``u``.  Returns (tokens int64 [B], logprobs fp32 [B]), the logarithm of the token's
    probability among those left; -1 and -inf for a row of no token.  ``out=(tokens, logprobs)`` is written
    instead of new tensors.  ``workspace``: uint8, of ``sample_workspace_bytes``, allocated per call if
    omitted; calls that overlap need their own."""
    _one_device("sample", logits, u, workspace)
    logits, rows, v, stride = _logits("sample", logits)
    if not _is(u, torch.float32, (rows,)):
        _refuse("sample", "u", u, torch.float32, (rows,))
    tensors, filters = _filters("sample", rows, temperature, top_k, top_p, min_p)
    _one_device("sample", logits, *tensors)
    tokens, logprobs = _out("sample", out, ("tokens", "logprobs"), (((rows,), torch.int64), ((rows,), torch.float32)), logits.device)
    if rows:
        need = sample_workspace_bytes(rows, v, logits.dtype)
        ws = _workspace("sample", workspace, need, logits.device)
        _call(logits.device, "mzk_sample", logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, v, stride, u.data_ptr(), *filters,
              tokens.data_ptr(), logprobs.data_ptr(), ws.data_ptr(), need)
    return tokens, logprobs


def verify(logits: torch.Tensor, tokens: torch.Tensor, cu: torch.Tensor, u: torch.Tensor, draw: torch.Tensor, *,
           draft_probs: torch.Tensor | None = None, temperature=None, top_k=None, top_p=None, min_p=None,
           workspace: torch.Tensor | None = None, out=None):
    """Which drafted tokens stay, so that what is accepted is distributed as if drawn from ``logits``.

    Rows ``cu[b] .. cu[b + 1] - 1`` (int64 [B + 1], as ``paged.attend`` takes it) are sequence b's newest tokens: the
    last certain one and the drafted ones behind it.  ``tokens`` int64 [T] are those, ``logits`` [T, V]
    follow each of them: row i judges token i + 1.  A drafted token of probability p behind the filters is accepted if
    ``u[i]`` (fp32 [T], of [0, 1)) times its probability in the draft is below p; the draft's probabilities
    ``draft_probs`` fp32 [T, V] stand in the same rows; without them the draft was certain.  Tokens outside
    the vocabulary are refused.  Returns (accepted int64 [B], next int64 [B]): the drafted tokens before the first
    refused one, and the token behind those, drawn with ``draw`` fp32 [B]: where none was refused from the
    last row as ``sample`` does; else from what the refused token's row has above the draft -- without
    ``draft_probs`` its other tokens, in their order, with them ``max(p - q, 0)`` by rising index, in units of 2^-52 (from p
    where that is nothing).  A sequence of no rows gives 0 and -1; rows behind the last sequence are not read.  Filters, ``out=(accepted,
    next)`` and ``workspace`` (``verify_workspace_bytes``) as in ``sample``."""
    _one_device("verify", logits, tokens, cu, u, draw, draft_probs, workspace)
    logits, rows, v, stride = _logits("verify", logits)
    if cu.dim() != 1 or cu.shape[0] < 1 or not _is(cu, torch.int64, cu.shape):
        _refuse("verify", "cu", cu, torch.int64, ("B + 1",))
    b = cu.shape[0] - 1
    for name, t, dt, shape in (("tokens", tokens, torch.int64, (rows,)), ("u", u, torch.float32, (rows,)),
                               ("draw", draw, torch.float32, (b,))):
        if not _is(t, dt, shape):
            _refuse("verify", name, t, dt, shape)
    qstride = 0
    if draft_probs is not None:
        if draft_probs.dtype != torch.float32 or draft_probs.shape != (rows, v):
            raise ValueError(f"verify: draft_probs must be float32 [{rows}, {v}], got {draft_probs.dtype} {list(draft_probs.shape)}")
        draft_probs, _, _, qstride = _logits("verify", draft_probs)
    tensors, filters = _filters("verify", rows, temperature, top_k, top_p, min_p)
    _one_device("verify", logits, *tensors)
    accepted, token = _out("verify", out, ("accepted", "next"), (((b,), torch.int64), ((b,), torch.int64)), logits.device)
    if b:
        need = verify_workspace_bytes(rows, b, v, logits.dtype, draft_probs is not None)
        ws = _workspace("verify", workspace, need, logits.device)
        _call(logits.device, "mzk_verify", logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, v, stride, tokens.data_ptr(),
              cu.data_ptr(), b, u.data_ptr(), draw.data_ptr(), _lib.ptr(draft_probs), qstride, *filters, accepted.data_ptr(),
              token.data_ptr(), ws.data_ptr(), need)
    return accepted, token


def beams(logits: torch.Tensor, scores: torch.Tensor, width: int, keep: int | None = None, *,
          workspace: torch.Tensor | None = None, out=None):
    """The step of a beam search.  Each ``width`` rows of ``logits`` [B, V] are a group's beams, ``scores`` fp32 [B]
    their log probabilities so far.  Of a group's continuations, valued ``scores[row] + log_softmax(logits[row])``, the
    ``keep`` best (``width`` if omitted; ``width * keep`` at most 4096), best first, equal ones by row and
    token.  Returns (parents int32, tokens int64, scores fp32), each [B / width * keep]: the rows that they
    continue -- ``paged.fork``'s parents --, their tokens and log probabilities; -1, -1 and -inf where a
    group has fewer.  A beam of score -inf or NaN has no continuation: a search starts with 0 and -inf.
    ``out=(parents, tokens, scores)`` and ``workspace`` (``beams_workspace_bytes``) as in ``sample``; the out scores may
    be ``scores`` itself, if as many, and overlap it no other way."""
    _one_device("beams", logits, scores, workspace)
    logits, rows, v, stride = _logits("beams", logits)
    if not isinstance(width, int) or width < 1 or rows % width:
        raise ValueError(f"beams: {rows} rows are no groups of {width!r}")
    keep = width if keep is None else keep
    if not isinstance(keep, int) or keep < 1 or width * keep > 4096:
        raise ValueError(f"beams: keep must be an int of at least 1, width * keep at most 4096, got {keep!r} of {width}")
    if not _is(scores, torch.float32, (rows,)):
        _refuse("beams", "scores", scores, torch.float32, (rows,))
    n = rows // width * keep
    parents, tokens, new = _out("beams", out, ("parents", "tokens", "scores"),
                                (((n,), torch.int32), ((n,), torch.int64), ((n,), torch.float32)), logits.device)
    at, to = scores.data_ptr(), new.data_ptr()
    if not (at == to and keep == width) and at < to + 4 * n and to < at + 4 * rows:
        raise ValueError("beams: the out scores are the scores themselves, as many, or overlap none of them")
    if rows:
        need = beams_workspace_bytes(rows, v, keep, logits.dtype)
        ws = _workspace("beams", workspace, need, logits.device)
        _call(logits.device, "mzk_beams", logits.data_ptr(), _lib.dtype_code(logits.dtype), rows, v, stride, scores.data_ptr(), width,
              keep, parents.data_ptr(), tokens.data_ptr(), new.data_ptr(), ws.data_ptr(), need)
    return parents, tokens, new
