"""Sparse rows of ids against dense matrices: lookups, their gradients, and the winners of dense scores.

Rows are given as tensors: ``ids`` [n] -- one id a row (the tokens of a sequence), ``ids`` [n, k] -- k ids a row (the result of
:func:`winners`), or ``ids`` [elements] with ``offsets`` [n + 1] -- ragged rows; the same operators are methods of
:class:`~sdr_amd.SDRBatch` for rows that a batch holds.  Ids are int32 or int64 and need be neither ascending nor distinct; an
id outside the dense matrix (a padded place holds -1) contributes nothing.  ``weights`` are float32, one an id.

Matrices are float32, float16 or bfloat16, with adjacent elements in a row and any row stride.  Sums are kept in binary32 and
rounded once to the output's type, in an order that the shapes and offsets fix: calls repeat bit for bit.  ``out``, where it is
given, may not overlap an input.  None of the functions is an autograd operator: a result carries no gradient function, whatever the
inputs require; a training step calls the gradients itself.

Everything is enqueued on ``stream`` (a torch stream or a handle; the current stream of the tensors' device by default), outputs
and scratch are allocated on that stream, and nothing waits for the GPU, so the calls can be captured into a graph.  An output that
is used on a further stream than ``stream`` and the current one needs torch's ``record_stream``.  All computation happens in
``libsdr_amd.so``; torch is used only to allocate and to name streams.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import Dense, Rows, WinnersSpec, check
from .batch import _empty as _batch_empty, _stream_handle

_SCORES = {"softmax": 0, "sigmoid": 1}
_types = {}
_raw_stream = None


def _torch():
    import torch  # plumbing only: device buffers and streams
    if not _types:
        global _raw_stream
        # the current stream's handle without making a stream object, where this torch offers it
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)
        _types.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return torch


def _device_of(t) -> int:
    device = t.get_device()
    if device < 0:
        raise ValueError("tensors must be on a GPU")
    return device


def _matrix(name, t, device) -> Dense:
    code = _types.get(t.dtype)
    if code is None or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-d float32, float16 or bfloat16 tensor")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device} like the other tensors")
    n, m = t.shape
    ld, inner = t.stride()
    if n <= 1:
        ld = m
    if (m > 1 and inner != 1) or ld < m:
        raise ValueError(f"{name} must have adjacent elements in a row and rows that do not overlap (call .contiguous())")
    return Dense(t.data_ptr(), n, m, ld, code)


def _vector(name, t, dtype, device, shape=None):
    if t.dtype != dtype or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor" + ("" if shape is None else f" of shape {tuple(shape)}"))
    if t.get_device() != device:
        raise ValueError(f"{name} must be on cuda:{device} like the other tensors")
    return t.data_ptr()


def _rows(torch, ids, weights, offsets) -> Rows:
    device = _device_of(ids)
    wide = ids.dtype == torch.int64
    if not (wide or ids.dtype == torch.int32) or not ids.is_contiguous() or ids.dim() not in (1, 2):
        raise ValueError("ids must be a contiguous 1-d or 2-d int32 or int64 tensor")
    off = None
    if offsets is not None:
        if ids.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets ([rows + 1]) go with 1-d ids")
        off = _vector("offsets", offsets, torch.int32, device)
        n = offsets.numel() - 1
    else:
        n = ids.shape[0]
    w = None if weights is None else _vector("weights", weights, torch.float32, device, ids.shape)
    return Rows(n, ids.numel(), off, ids.data_ptr(), w, 64 if wide else 32)


def _empty(torch, shape, dtype, like, stream):
    return like.new_empty(shape, dtype=dtype) if stream is None else _batch_empty(shape, dtype, like.get_device(), stream)


def _result(torch, out, n, m, dtype, like, stream):
    """(tensor, its description) of a result [n, m]: ``out``, or a new tensor"""
    if out is None:
        code = _types.get(dtype)
        if code is None:
            raise ValueError("results are float32, float16 or bfloat16")
        out = _empty(torch, (n, m), dtype, like, stream)
        return out, Dense(out.data_ptr(), n, m, m, code)
    if tuple(out.shape) != (n, m) or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out must have shape {(n, m)}" + ("" if dtype is None else f" and type {dtype}"))
    return out, _matrix("out", out, like.get_device())


def _scratch(torch, size, like, stream):
    if size == 0:
        return None, 0, None
    t = like.new_empty(size, dtype=torch.uint8) if stream is None else _batch_empty(size, torch.uint8, like.get_device(), stream, result=False)
    return t, size, t.data_ptr()


def _handle(device, stream) -> int:
    return _raw_stream(device) if stream is None else _stream_handle(device, stream)


def _lookup(lib, rows, device, table, scale, dtype, out, stream):
    torch = _torch()
    t = _matrix("table", table, device)
    out, o = _result(torch, out, rows.n_rows, t.n_cols, dtype if out is not None else dtype or table.dtype, table, stream)
    keep, size, at = None, 0, None
    if rows.row_offsets or rows.n_elems > 64 * rows.n_rows:   # (rows of equal length need none up to 64 ids)
        need = C.c_size_t()
        check(lib.sdrb_lookup_scratch(rows, t.n_cols, need))
        keep, size, at = _scratch(torch, need.value, table, stream)
    check(lib.sdrb_lookup(device, rows, t, scale, o, at, size, _handle(device, stream)))
    return out


def _lookup_grad_table(lib, rows, device, grad, n_table_rows, scale, dtype, out, accumulate, stream):
    torch = _torch()
    g = _matrix("grad", grad, device)
    if accumulate and out is None:
        raise ValueError("accumulate needs the tensor to add to as out")
    if n_table_rows is None:
        n_table_rows = out.shape[0]
    if n_table_rows < 0:
        raise ValueError("n_table_rows must not be negative")
    out, o = _result(torch, out, n_table_rows, g.n_cols, dtype if out is not None else dtype or torch.float32, grad, stream)
    need = C.c_size_t()
    check(lib.sdrb_lookup_grad_table_scratch(rows, n_table_rows, g.n_cols, need))
    keep, size, at = _scratch(torch, need.value, grad, stream)
    check(lib.sdrb_lookup_grad_table(device, rows, g, scale, int(accumulate), o, at, size, _handle(device, stream)))
    return out


def _lookup_grad_weights(lib, rows, device, grad, table, scale, shape, out, stream):
    torch = _torch()
    g, t = _matrix("grad", grad, device), _matrix("table", table, device)
    if out is None:
        out = _empty(torch, shape, torch.float32, grad, stream)
    check(lib.sdrb_lookup_grad_weights(device, rows, g, t, scale, _vector("out", out, torch.float32, device, torch.Size(shape)),
                                       _handle(device, stream)))
    return out


def lookup(ids, table, weights=None, *, offsets=None, scale: float = 1.0, dtype=None, out=None, stream=None):
    """``out[r] = scale * sum of weight * table[id]`` over the ids of row r, in their order: [rows, table columns], of the
    table's type unless ``dtype`` (or ``out``) says otherwise.  An embedding lookup where rows hold one id; a row without
    ids, or with none inside the table, yields zeros."""
    rows = _rows(_torch(), ids, weights, offsets)
    return _lookup(_lib.load(), rows, ids.get_device(), table, scale, dtype, out, stream)


def lookup_grad_table(ids, grad, n_table_rows=None, weights=None, *, offsets=None, scale: float = 1.0, dtype=None, out=None,
                      accumulate: bool = False, stream=None):
    """The gradient of :func:`lookup` to its table, from the gradient ``grad`` [rows, columns] of its result:
    ``out[v] = scale * sum over the elements with id v of weight * grad[their row]``, [n_table_rows, columns], float32 unless
    ``dtype`` (or ``out``) says otherwise; zeros where no row names v.  ``accumulate``: the sums are added to ``out``, and its rows
    that no id names are not touched.  The elements are sorted by id on the way; no atomic addition is used."""
    rows = _rows(_torch(), ids, weights, offsets)
    if n_table_rows is None and out is None:
        raise ValueError("give n_table_rows or out")
    return _lookup_grad_table(_lib.load(), rows, ids.get_device(), grad, n_table_rows, scale, dtype, out, accumulate, stream)


def lookup_grad_weights(ids, grad, table, *, offsets=None, scale: float = 1.0, out=None, stream=None):
    """The gradient of :func:`lookup` to its weights: ``scale * <grad[row], table[id]>`` an id, float32 in the shape of
    ``ids``; 0 for an id outside the table."""
    rows = _rows(_torch(), ids, None, offsets)
    return _lookup_grad_weights(_lib.load(), rows, ids.get_device(), grad, table, scale, ids.shape, out, stream)


def _spec(torch, k, score, renormalise, scale, device, bias=None, groups=1, top_groups=None, group_top=1, n_ids=0) -> WinnersSpec:
    if score not in _SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    if min(groups, group_top, 1 if top_groups is None else top_groups) < 1:
        raise ValueError("groups, top_groups and group_top must be positive")
    b = None if bias is None else _vector("bias", bias, torch.float32, device, torch.Size((n_ids,)))
    return WinnersSpec(k, _SCORES[score], int(renormalise), groups, groups if top_groups is None else top_groups, group_top, scale, b)


def winners(scores, k: int, *, score: str = "softmax", bias=None, groups: int = 1, top_groups=None, group_top: int = 1,
            renormalise: bool = False, scale: float = 1.0, stream=None):
    """The ``k`` winning ids of every row of ``scores`` [rows, ids], ascending, and their weights: ``(ids, weights)``, int32 and
    float32 [rows, k], -1 and 0 in the last places of a row with fewer candidates.  Routing of tokens to experts, or dense
    activations made into sparse codes (:meth:`SDRBatch.from_winners`).

    An id's share is the ``score`` -- "softmax" over the row, or "sigmoid" -- and its key the share plus ``bias`` (float32 [ids],
    which balances the choice and does not enter the weights).  With ``groups`` > 1 only ids of the ``top_groups`` groups win
    whose ``group_top`` (1 or 2) largest keys have the largest sums.  The largest keys win, equal ones by the lowest id; scores
    of -inf or NaN never do.  Weights are ``scale`` times the shares, or with ``renormalise`` the shares' parts of their sum."""
    torch = _torch()
    device = _device_of(scores)
    s = _matrix("scores", scores, device)
    if not 1 <= k <= s.n_cols:
        raise ValueError("k must be 1 .. ids")
    spec = _spec(torch, k, score, renormalise, scale, device, bias, groups, top_groups, group_top, s.n_cols)
    ids = _empty(torch, (s.n_rows, k), torch.int32, scores, stream)
    weights = _empty(torch, (s.n_rows, k), torch.float32, scores, stream)
    check(_lib.load().sdrb_winners(device, s, spec, ids.data_ptr(), weights.data_ptr(), _handle(device, stream)))
    return ids, weights


def winners_grad(scores, ids, grad_weights, *, score: str = "softmax", renormalise: bool = False, scale: float = 1.0, dtype=None,
                 out=None, stream=None):
    """The gradient of :func:`winners`' weights to ``scores``: [rows, ids], of the scores' type unless ``dtype`` (or ``out``) says
    otherwise, from the ``ids`` [rows, k] it chose (distinct in a row; their choice is constant) and the gradient ``grad_weights``
    of the weights.  ``score``, ``renormalise`` and ``scale`` as in the forward call; a bias and groups have no part in it."""
    torch = _torch()
    device = _device_of(scores)
    s = _matrix("scores", scores, device)
    if ids.dim() != 2 or ids.shape[0] != s.n_rows:
        raise ValueError("ids must be [rows, k]")
    i = _vector("ids", ids, torch.int32, device)
    g = _vector("grad_weights", grad_weights, torch.float32, device, ids.shape)
    spec = _spec(torch, ids.shape[1], score, renormalise, scale, device)
    out, o = _result(torch, out, s.n_rows, s.n_cols, dtype if out is not None else dtype or scores.dtype, scores, stream)
    check(_lib.load().sdrb_winners_grad(device, s, spec, i, g, o, _handle(device, stream)))
    return out
