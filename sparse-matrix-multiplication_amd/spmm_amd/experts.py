"""Mixture-of-experts routing and products, and low-rank adapters, over
libspmm_amd.so.

The routing of T tokens to E experts, k of them a token, is a sparse T x E
matrix with k entries a row.  ``route`` finds it and the order of its entries
by expert, ``dispatch`` and ``combine`` multiply by it (tokens into expert
order and back, weighted).  ``grouped_mm`` is the block-diagonal product of the
rows in expert order with their experts' weights.  Every one of these has its
gradient beside it.  ``adapter_mm`` is a shared projection with each row's own
low-rank adapter.

Operands are contiguous cuda tensors on the current device; outputs are
allocated where none is given, on the stream that the launch goes to (`stream`
or the current one).  An output given must not share memory with an operand.
Nothing synchronises.  Results carry no autograd graph, whatever the operands
require: a training step calls the gradients, or takes ``ExpertLayer``
(expert_layer.py), which does so under autograd.
"""
from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Any

import torch

from . import SPMM_INVALID, SPMM_UNSUPPORTED, SpmmError, _check, lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_OVER = {"chosen": 0, "all": 1}
_INT = (torch.int32,)
_FLOAT = (torch.float32,)


def _operand(t, name: str, dtypes, shape, device=None) -> None:
    """One contiguous operand of the given types and shape (a tuple, or the number
    of dimensions) on `device`, or on the current device where that is not given."""
    try:
        got = t.shape
        if (got == shape or len(got) == shape) and t.dtype in dtypes and t.is_contiguous():
            where = t.device
            if where == device or (device is None and where.type == "cuda"
                                   and where.index == torch.cuda.current_device()):
                return
    except (AttributeError, TypeError):
        pass
    _refuse(t, name, dtypes, shape, device)


def _refuse(t, name: str, dtypes, shape, device) -> None:
    """What is wrong with an operand, as an SpmmError."""
    if not isinstance(t, torch.Tensor):
        raise SpmmError(SPMM_INVALID, f"{name}: expected a torch tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise SpmmError(SPMM_INVALID, f"{name}: must be a cuda tensor (got {t.device})")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if t.device != device:
        raise SpmmError(SPMM_INVALID, f"{name}: on {t.device}, expected {device}")
    if t.dtype not in dtypes:
        want = " or ".join(str(d) for d in dtypes)
        raise SpmmError(SPMM_INVALID, f"{name}: dtype {t.dtype}, expected {want}")
    if not t.is_contiguous():
        raise SpmmError(SPMM_INVALID, f"{name}: must be contiguous (row-major)")
    want = f"{shape} dimensions" if isinstance(shape, int) else f"shape {tuple(shape)}"
    raise SpmmError(SPMM_INVALID, f"{name}: shape {tuple(t.shape)}, expected {want}")


def _out(t, name: str, dtype, shape, device):
    """The output given, checked, or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _operand(t, name, (dtype,), shape, device)
    return t


def _rows(t, name: str, rows: int) -> None:
    if t.shape[0] != rows:
        raise SpmmError(SPMM_INVALID, f"{name}: {t.shape[0]} rows, expected {rows}")


def _counts(*sizes) -> None:
    """Sizes go to the library as 32-bit integers, which would cut larger ones off."""
    if max(sizes) > 0x7fffffff:
        raise SpmmError(SPMM_UNSUPPORTED, f"sizes {sizes}: over 2^31 - 1")


_here = contextlib.nullcontext()


def _on(stream, device):
    """Allocations inside belong to the stream that the launch goes to, so that
    freeing them needs no wait of another stream's."""
    if stream is None:
        return _here
    if getattr(stream, "device", None) != device:
        raise SpmmError(SPMM_INVALID, f"stream: {stream!r}, expected a torch stream on {device}")
    return torch.cuda.stream(stream)


def _stream(device) -> int:
    # the handle alone: torch.cuda.current_stream builds a Stream object around it
    return torch._C._cuda_getCurrentRawStream(device.index)


@dataclass
class Routing:
    """Tokens' experts and the order of the (token, choice) entries by expert.

    experts  int32 [T, k]   chosen experts, -1 for none
    weights  fp32  [T, k]   their softmax weights, 0 for none
    offsets  int32 [E + 1]  each expert's first row in expert order
    entries  int32 [T * k]  the entry t * k + j in each row, -1 behind the last
    slots    int32 [T, k]   the row of each entry, -1 for none
    over     "chosen" or "all": what the softmax runs over
    """
    experts: Any
    weights: Any
    offsets: Any
    entries: Any
    slots: Any
    over: str = "chosen"

    def _sizes(self):
        """(tokens, k, experts), after a look at the fields that every call reads."""
        if not isinstance(self.slots, torch.Tensor) or self.slots.dim() != 2 \
                or not isinstance(self.offsets, torch.Tensor) or self.offsets.dim() != 1 \
                or self.offsets.shape[0] < 2:
            raise SpmmError(SPMM_INVALID, "routing: slots [T, k] and offsets [E + 1] are needed")
        T, k = self.slots.shape
        if k < 1:
            raise SpmmError(SPMM_INVALID, "routing: no choice a token")
        return T, k, self.offsets.shape[0] - 1


def _over_id(over) -> int:
    if over not in _OVER:
        raise SpmmError(SPMM_INVALID, f"over: {over!r}, expected 'chosen' or 'all'")
    return _OVER[over]


def route(logits, k: int, over: str = "chosen", stream=None) -> Routing:
    """The k largest of each token's logits [T, E] (float32, float16 or
    bfloat16), their softmax weights over the chosen experts or over "all", and
    the entries' order by expert.  Ties go to the lowest expert; -inf is never
    chosen; a NaN is above all numbers and makes its token's weights NaN."""
    over_id = _over_id(over)
    _operand(logits, "logits", _TYPES, 2)
    T, E = logits.shape
    k = int(k)
    if not 1 <= k <= E:
        raise SpmmError(SPMM_INVALID, f"k: {k}, expected 1 to {E} experts")
    _counts(T, E)
    L = lib()
    device = logits.device
    with _on(stream, device):
        experts = torch.empty((T, k), dtype=torch.int32, device=device)
        slots = torch.empty((T, k), dtype=torch.int32, device=device)
        entries = torch.empty(T * k, dtype=torch.int32, device=device)
        offsets = torch.empty(E + 1, dtype=torch.int32, device=device)
        weights = torch.empty((T, k), dtype=torch.float32, device=device)
        room = L.spmm_c_route_workspace(T, E, k)
        work = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        _check(L.spmm_c_route(logits.data_ptr(), _TYPES[logits.dtype], T, E, k, over_id,
                              experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(),
                              entries.data_ptr(), slots.data_ptr(),
                              work.data_ptr() if room else None, _stream(device)))
    return Routing(experts, weights, offsets, entries, slots, over)


def route_backward(logits, routing: Routing, dweights, out=None, stream=None):
    """The gradient of ``route``'s weights with respect to the logits, of the
    logits' type: [T, E]."""
    over_id = _over_id(routing.over)
    _operand(logits, "logits", _TYPES, 2)
    T, E = logits.shape
    device = logits.device
    _operand(routing.weights, "routing.weights", _FLOAT, 2, device)
    k = routing.weights.shape[1]
    if routing.weights.shape[0] != T or not 1 <= k <= E:
        raise SpmmError(SPMM_INVALID, f"routing: of {tuple(routing.weights.shape)} choices, "
                                      f"logits are {tuple(logits.shape)}")
    _counts(T, E)
    _operand(routing.experts, "routing.experts", _INT, (T, k), device)
    _operand(dweights, "dweights", _FLOAT, (T, k), device)
    with _on(stream, device):
        out = _out(out, "out", logits.dtype, (T, E), device)
        _check(lib().spmm_c_route_backward(
            logits.data_ptr(), _TYPES[logits.dtype], T, E, k, over_id, routing.experts.data_ptr(),
            routing.weights.data_ptr(), dweights.data_ptr(), out.data_ptr(), _stream(device)))
    return out


def group_entries(ids, groups: int, stream=None):
    """The stable order of entries by group, for ids int32 of any shape: (offsets
    [groups + 1], entries [n], slots like ids).  An id outside [0, groups) has no
    place: slot -1, and -1 fills the entries behind the last group."""
    if not isinstance(ids, torch.Tensor):
        raise SpmmError(SPMM_INVALID, f"ids: expected a torch tensor, got {type(ids).__name__}")
    _operand(ids, "ids", _INT, ids.shape)
    n, device = ids.numel(), ids.device
    groups = int(groups)
    if groups < 1:
        raise SpmmError(SPMM_INVALID, f"groups: {groups}, expected at least 1")
    _counts(n, groups)
    L = lib()
    with _on(stream, device):
        offsets = torch.empty(groups + 1, dtype=torch.int32, device=device)
        entries = torch.empty(n, dtype=torch.int32, device=device)
        slots = torch.empty_like(ids)
        room = L.spmm_c_group_workspace(n, groups)
        work = torch.empty(room, dtype=torch.uint8, device=device) if room else None
        _check(L.spmm_c_group_entries(ids.data_ptr(), n, groups, offsets.data_ptr(),
                                      entries.data_ptr(), slots.data_ptr(),
                                      work.data_ptr() if room else None, _stream(device)))
    return offsets, entries, slots


def dispatch(x, routing: Routing, out=None, stream=None):
    """Rows of x [T, D] into expert order: [T * k, D]; rows without an entry are zero."""
    T, k, E = routing._sizes()
    _operand(x, "x", _TYPES, 2)
    _rows(x, "x", T)
    D, device = x.shape[1], x.device
    _counts(T, k, D, E)
    _operand(routing.slots, "routing.slots", _INT, (T, k), device)
    _operand(routing.offsets, "routing.offsets", _INT, (E + 1,), device)
    with _on(stream, device):
        out = _out(out, "out", x.dtype, (T * k, D), device)
        _check(lib().spmm_c_dispatch(x.data_ptr(), _TYPES[x.dtype], T, k, D,
                                     routing.slots.data_ptr(), routing.offsets.data_ptr(), E,
                                     out.data_ptr(), _stream(device)))
    return out


def _gather(ys, name: str, routing: Routing, weighted: bool, out, stream):
    T, k, _ = routing._sizes()
    _operand(ys, name, _TYPES, 2)
    _rows(ys, name, T * k)
    D, device = ys.shape[1], ys.device
    _counts(T, k, D)
    _operand(routing.slots, "routing.slots", _INT, (T, k), device)
    if weighted:
        _operand(routing.weights, "routing.weights", _FLOAT, (T, k), device)
    with _on(stream, device):
        out = _out(out, "out", ys.dtype, (T, D), device)
        _check(lib().spmm_c_combine(ys.data_ptr(), _TYPES[ys.dtype], T, k, D,
                                    routing.slots.data_ptr(),
                                    routing.weights.data_ptr() if weighted else None,
                                    out.data_ptr(), _stream(device)))
    return out


def dispatch_backward(dxs, routing: Routing, out=None, stream=None):
    """The gradient of ``dispatch``: each token's rows of dxs [T * k, D] added up: [T, D]."""
    return _gather(dxs, "dxs", routing, False, out, stream)


def combine(ys, routing: Routing, out=None, stream=None):
    """Each token's rows of ys [T * k, D] in expert order, weighted and added up: [T, D]."""
    return _gather(ys, "ys", routing, True, out, stream)


def combine_backward(dy, ys, routing: Routing, stream=None):
    """The gradients of ``combine`` for dy [T, D]: (dys [T * k, D], dweights fp32 [T, k])."""
    T, k, E = routing._sizes()
    _operand(ys, "ys", _TYPES, 2)
    _rows(ys, "ys", T * k)
    D, device = ys.shape[1], ys.device
    _counts(T, k, D, E)
    _operand(dy, "dy", (ys.dtype,), (T, D), device)
    _operand(routing.slots, "routing.slots", _INT, (T, k), device)
    _operand(routing.weights, "routing.weights", _FLOAT, (T, k), device)
    _operand(routing.offsets, "routing.offsets", _INT, (E + 1,), device)
    with _on(stream, device):
        dys = torch.empty_like(ys)
        dweights = torch.empty((T, k), dtype=torch.float32, device=device)
        _check(lib().spmm_c_combine_backward(
            dy.data_ptr(), ys.data_ptr(), _TYPES[ys.dtype], T, k, D, routing.slots.data_ptr(),
            routing.weights.data_ptr(), routing.offsets.data_ptr(), E, dys.data_ptr(),
            dweights.data_ptr(), _stream(device)))
    return dys, dweights


_HALF = (torch.float16, torch.bfloat16)


def _half(t, name: str) -> None:
    if isinstance(t, torch.Tensor) and t.dtype == torch.float32:
        raise SpmmError(SPMM_UNSUPPORTED, f"{name}: float16 or bfloat16 (matrix cores)")
    _operand(t, name, _HALF, 2)


def _weights(w, dtype, K: int, w_in_rows: bool, device):
    """(G, N) of weights [G, N, K], or [G, K, N] with w_in_rows."""
    _operand(w, "w", (dtype,), 3, device)
    G, n, k = w.shape
    if w_in_rows:
        n, k = k, n
    if k != K:
        raise SpmmError(SPMM_INVALID, f"w: shape {tuple(w.shape)} for rows of {K} elements")
    _counts(G, n, k)
    return G, n


def grouped_mm(x, w, offsets, w_in_rows: bool = False, out=None, stream=None):
    """Rows of x [S, K] times their group's weights: [S, N].  Group g has rows
    offsets[g] to offsets[g + 1] (int32 [G + 1]); w is [G, N, K], or [G, K, N] with
    w_in_rows.  Rows in no group are zero."""
    _half(x, "x")
    S, K = x.shape
    device = x.device
    G, N = _weights(w, x.dtype, K, w_in_rows, device)
    _operand(offsets, "offsets", _INT, (G + 1,), device)
    _counts(S, N)
    with _on(stream, device):
        out = _out(out, "out", x.dtype, (S, N), device)
        _check(lib().spmm_c_grouped_mm(x.data_ptr(), w.data_ptr(), _TYPES[x.dtype],
                                       offsets.data_ptr(), G, S, N, K, int(bool(w_in_rows)),
                                       out.data_ptr(), _stream(device)))
    return out


def grouped_mm_backward(dy, x, w, offsets, w_in_rows: bool = False, stream=None, rows: bool = True,
                        weights: bool = True):
    """The gradients of ``grouped_mm`` for dy [S, N]: (dx [S, K], dw like w).  One that is
    not asked for (rows=False, weights=False) is not computed and None."""
    _half(x, "x")
    S, K = x.shape
    device = x.device
    G, N = _weights(w, x.dtype, K, w_in_rows, device)
    _operand(dy, "dy", (x.dtype,), (S, N), device)
    _operand(offsets, "offsets", _INT, (G + 1,), device)
    _counts(S, N)
    p, q, height, width = (x, dy, K, N) if w_in_rows else (dy, x, N, K)
    with _on(stream, device):
        dw = torch.empty_like(w) if weights else None
        dx = torch.empty_like(x) if rows else None
        L, s = lib(), _stream(device)
        if rows:
            _check(L.spmm_c_grouped_mm(dy.data_ptr(), w.data_ptr(), _TYPES[x.dtype],
                                       offsets.data_ptr(), G, S, K, N, int(not w_in_rows),
                                       dx.data_ptr(), s))
        if weights:
            _check(L.spmm_c_grouped_outer(p.data_ptr(), q.data_ptr(), _TYPES[x.dtype],
                                          offsets.data_ptr(), G, S, height, width, dw.data_ptr(), s))
    return dx, dw


def adapter_mm(x, w, a, b, ids, scale=None, out=None, stream=None):
    """A shared projection with low-rank adapters of many requests at once: row s of
    the result is x[s] w^T + scale[i] (x[s] a[i]^T) b[i]^T with i = ids[s], the
    projection alone where ids[s] is outside [0, L).

    x [T, K], w [N, K], a [L, R, K], b [L, N, R], float16 or bfloat16; ids int32
    [T]; scale float32 [L], 1 when None.  Adapters of a smaller rank are padded
    with zeros."""
    _half(x, "x")
    T, K = x.shape
    device = x.device
    _operand(w, "w", (x.dtype,), 2, device)
    N = w.shape[0]
    _operand(w, "w", (x.dtype,), (N, K), device)
    _operand(a, "a", (x.dtype,), 3, device)
    L, R = a.shape[:2]
    _operand(a, "a", (x.dtype,), (L, R, K), device)
    _operand(b, "b", (x.dtype,), (L, N, R), device)
    _operand(ids, "ids", _INT, (T,), device)
    _counts(T, N, K, L, R)
    if scale is not None:
        _operand(scale, "scale", _FLOAT, (L,), device)
    library = lib()
    with _on(stream, device):
        out = _out(out, "out", x.dtype, (T, N), device)
        work = torch.empty(library.spmm_c_adapter_workspace(T, R), dtype=torch.uint8,
                           device=device)
        _check(library.spmm_c_adapter_mm(
            x.data_ptr(), w.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(),
            None if scale is None else scale.data_ptr(), _TYPES[x.dtype], T, N, K, L, R,
            out.data_ptr(), work.data_ptr(), _stream(device)))
    return out
