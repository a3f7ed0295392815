"""Gated feed-forward blocks, activations kept in 8 bits for their backward pass, and
products in 8-bit integers, over libspmm_amd.so.

``gated_mm`` is act(x Wg^T) * (x Wu^T) in one kernel, for one pair of weights or with a
pair for each group of rows (``grouped_mm``'s), and ``gated_mm_backward`` its gradients.
``pack8`` and ``unpack8`` hold activations in 8 bits in between, which
``gated_mm_backward`` takes as they are.  ``quantize_rows`` and ``int8_mm`` are the
products in 8-bit integers with a scale a token and a channel; ``gated_mm`` takes
quantised rows too.

Operands, outputs, streams and errors are as in experts.py: contiguous cuda tensors on the
current device, outputs allocated where none is given, nothing synchronises, results carry
no autograd graph.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch

from . import SPMM_INVALID, SPMM_UNSUPPORTED, SpmmError, _check, lib
from .experts import (_FLOAT, _INT, _TYPES, _counts, _half, _on, _operand, _out, _refuse,
                      _stream)

_ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
_BYTES = (torch.int8,)
_SCALES = (torch.uint8,)
BLOCK = 32  # values that share a scale
_WIDEST_GRADIENT = 1 << 21  # columns: both projections' gradients are a product's row of 2^22


@dataclass
class Packed8:
    """Values in 8 bits: q * 2^(scale - 133), a scale for each 32 along the last dimension.

    values  int8  [..., K]
    scales  uint8 [..., ceil(K / 32)]
    """
    values: Any
    scales: Any

    def _checked(self, name: str, shape=None, device=None):
        v = self.values
        if not isinstance(v, torch.Tensor) or v.dim() < 1:
            _refuse(v, f"{name}.values", _BYTES, shape or 2, device)
        _operand(v, f"{name}.values", _BYTES, tuple(v.shape) if shape is None else shape, device)
        _operand(self.scales, f"{name}.scales", _SCALES,
                 tuple(v.shape[:-1]) + ((v.shape[-1] + BLOCK - 1) // BLOCK,), v.device)
        return v


@dataclass
class Rows8:
    """Rows of 8-bit integers with a scale each: values[..., :width] * scales[..., None].

    values  int8 [..., width rounded up to a multiple of 16], zero past width
    scales  fp32 [...]
    """
    values: Any
    scales: Any
    width: int

    def _checked(self, name: str, dims: int, device=None):
        _operand(self.values, f"{name}.values", _BYTES, dims, device)
        shape = tuple(self.values.shape)
        if isinstance(self.width, bool) or not isinstance(self.width, int) or self.width < 1 \
                or shape[-1] != _padded(self.width):
            raise SpmmError(SPMM_INVALID, f"{name}: rows of {shape[-1]} for a width of {self.width!r}")
        _operand(self.scales, f"{name}.scales", _FLOAT, shape[:-1], self.values.device)
        return self.values


def _padded(width: int) -> int:
    return (width + 15) // 16 * 16


def _act_id(act) -> int:
    if not isinstance(act, str) or act not in _ACTS:
        raise SpmmError(SPMM_INVALID, f"act: {act!r}, expected one of {sorted(_ACTS)}")
    return _ACTS[act]


def _flat(t, name: str):
    """(rows, width) of a tensor whose last dimension is a row."""
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        _refuse(t, name, _TYPES, 2, None)
    _operand(t, name, _TYPES, t.shape)
    width = t.shape[-1]
    if width < 1:
        raise SpmmError(SPMM_INVALID, f"{name}: shape {tuple(t.shape)} has empty rows")
    _counts(width)
    return t.numel() // width, width


def pack8(x, stream=None) -> Packed8:
    """x [..., K] (float32, float16 or bfloat16) in 8 bits: blocks of 32 along the last
    dimension with the power of two of their largest value.  A value is off by at most half
    a step, 2^-7 of the power of two at or below that largest value (a whole one next to it).
    A block with an infinity or a NaN is NaN."""
    rows, width = _flat(x, "x")
    device = x.device
    with _on(stream, device):
        values = torch.empty(x.shape, dtype=torch.int8, device=device)
        scales = torch.empty(x.shape[:-1] + ((width + BLOCK - 1) // BLOCK,), dtype=torch.uint8,
                             device=device)
        _check(lib().spmm_c_pack8(x.data_ptr(), _TYPES[x.dtype], rows, width, values.data_ptr(),
                                  scales.data_ptr(), _stream(device)))
    return Packed8(values, scales)


def unpack8(packed: Packed8, dtype=torch.bfloat16, out=None, stream=None):
    """The values that ``pack8`` holds, of the type asked for (exact in bfloat16 and float32)."""
    if dtype not in _TYPES:
        raise SpmmError(SPMM_INVALID, f"dtype: {dtype}, expected one of {list(_TYPES)}")
    if not isinstance(packed, Packed8):
        raise SpmmError(SPMM_INVALID, f"packed: expected Packed8, got {type(packed).__name__}")
    v = packed._checked("packed")
    width = v.shape[-1]
    if width < 1:
        raise SpmmError(SPMM_INVALID, f"packed: shape {tuple(v.shape)} has empty rows")
    _counts(width)
    with _on(stream, v.device):
        out = _out(out, "out", dtype, tuple(v.shape), v.device)
        _check(lib().spmm_c_unpack8(v.data_ptr(), packed.scales.data_ptr(), _TYPES[dtype],
                                    v.numel() // width, width, out.data_ptr(), _stream(v.device)))
    return out


def quantize_rows(x, stream=None) -> Rows8:
    """Rows of x [..., K] (float32, float16 or bfloat16) as 8-bit integers: scale = max|x| *
    (1 / 127), and the integers next to x * (1 / max|x| * 127), ties to even; these factors are
    rounded to float32 at each step, so they are up to two roundings from the quotients.  A
    largest value below 2^-100 is taken as that, so rows below 2^-108 are zeros.  A row with an
    infinity or a NaN has the scale NaN."""
    rows, width = _flat(x, "x")
    device = x.device
    with _on(stream, device):
        values = torch.empty(x.shape[:-1] + (_padded(width),), dtype=torch.int8, device=device)
        scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=device)
        _check(lib().spmm_c_quantize_rows(x.data_ptr(), _TYPES[x.dtype], rows, width,
                                          values.data_ptr(), scales.data_ptr(), _stream(device)))
    return Rows8(values, scales, width)


def _groups(offsets, w_shape, device):
    """(groups, pointer) of offsets, None for one group of all rows, whose weights then have
    no dimension for groups."""
    if offsets is None:
        return 1, None
    G = w_shape[0]
    _operand(offsets, "offsets", _INT, (G + 1,), device)
    if G < 1:
        raise SpmmError(SPMM_INVALID, "w: no group")
    return G, offsets.data_ptr()


def _int8(x, w, offsets, pair: bool, act: int, dtype, out, stream):
    if not isinstance(w, Rows8):
        raise SpmmError(SPMM_INVALID, f"w: expected Rows8, got {type(w).__name__}")
    if dtype is not None and dtype not in _TYPES:
        raise SpmmError(SPMM_INVALID, f"dtype: {dtype}, expected one of {list(_TYPES)}")
    # all is looked at before anything is launched
    wv = w._checked("w", 2 + pair + (offsets is not None))
    device = wv.device
    if pair and wv.shape[-3] != 2:
        raise SpmmError(SPMM_INVALID, f"w: shape {tuple(wv.shape)}, expected [..., 2, N, K]")
    quantised = isinstance(x, Rows8)
    if quantised:
        S, width = x._checked("x", 2, device).shape[0], x.width
    else:
        _operand(x, "x", _TYPES, 2, device)
        S, width = x.shape
    if width != w.width:
        raise SpmmError(SPMM_INVALID, f"w: rows of {w.width} for x of {width}")
    if dtype is None:
        dtype = torch.bfloat16 if quantised else x.dtype
    G, at = _groups(offsets, wv.shape, device)
    N, depth = wv.shape[-2:]
    _counts(S, N, depth, G)
    L = lib()
    with _on(stream, device):
        out = _out(out, "out", dtype, (S, N), device)
        s = _stream(device)
        if quantised:
            values, scales = x.values.data_ptr(), x.scales.data_ptr()
        else:
            # rows of integers and behind them their scales
            room = torch.empty(S * (depth + 4), dtype=torch.int8, device=device)
            values = room.data_ptr()
            scales = values + S * depth
            _check(L.spmm_c_quantize_rows(x.data_ptr(), _TYPES[x.dtype], S, width, values, scales, s))
        args = (values, scales, wv.data_ptr(), w.scales.data_ptr(), at, G, S, N, depth)
        if pair:
            _check(L.spmm_c_gated_int8_mm(*args, act, _TYPES[dtype], out.data_ptr(), s))
        else:
            _check(L.spmm_c_int8_mm(*args, _TYPES[dtype], out.data_ptr(), s))
    return out


def int8_mm(x, w: Rows8, offsets=None, dtype=None, out=None, stream=None):
    """x [S, K] w^T in 8-bit integers: [S, N].  x is Rows8, or a tensor that is quantised a
    row at a time; w is Rows8 of [N, K], or of [G, N, K] with offsets (``grouped_mm``'s;
    rows in no group are zero).  The integers' sums are exact.  dtype: float32, float16 or
    bfloat16; x's where it is a tensor, else bfloat16.  K up to 131056."""
    return _int8(x, w, offsets, False, 0, dtype, out, stream)


def gated_mm(x, w, offsets=None, act: str = "silu", keep=None, dtype=None, out=None, stream=None):
    """act(g) * u with g = x w[0]^T and u = x w[1]^T: [S, N].

    x [S, K], w [2, N, K], or [G, 2, N, K] with offsets (``grouped_mm``'s; rows in no group
    are zero), float16 or bfloat16.  act: "silu", "gelu" or "gelu_tanh".  keep: "full" returns
    g and u [S, 2, N] of x's type too, for ``gated_mm_backward``, "8bit" the same as Packed8.
    x and w may be quantised rows (``int8_mm``'s operands: x a tensor or Rows8, w Rows8), with
    ``int8_mm``'s dtype; nothing can be kept then."""
    act_id = _act_id(act)
    if keep not in (None, "full", "8bit"):
        raise SpmmError(SPMM_INVALID, f"keep: {keep!r}, expected None, 'full' or '8bit'")
    if isinstance(w, Rows8):
        if keep is not None:
            raise SpmmError(SPMM_UNSUPPORTED, "keep: products in 8-bit integers have no gradients")
        return _int8(x, w, offsets, True, act_id, dtype, out, stream)
    if isinstance(x, Rows8):
        raise SpmmError(SPMM_INVALID, "w: expected Rows8 next to x of Rows8")
    _half(x, "x")
    if dtype not in (None, x.dtype):
        raise SpmmError(SPMM_INVALID, f"dtype: {dtype}, expected {x.dtype}, x's")
    S, K = x.shape
    device = x.device
    G, N, at = _pairs(w, x.dtype, K, offsets, device)
    _counts(S, K)
    with _on(stream, device):
        out = _out(out, "out", x.dtype, (S, N), device)
        kept = values = scales = None
        if keep == "full":
            kept = values = torch.empty((S, 2, N), dtype=x.dtype, device=device)
        elif keep == "8bit":
            values = torch.empty((S, 2, N), dtype=torch.int8, device=device)
            scales = torch.empty((S, 2, (N + BLOCK - 1) // BLOCK), dtype=torch.uint8, device=device)
            kept = Packed8(values, scales)
        _check(lib().spmm_c_gated_mm(x.data_ptr(), w.data_ptr(), _TYPES[x.dtype], at, G, S, N, K,
                                     act_id, out.data_ptr(),
                                     None if values is None else values.data_ptr(),
                                     None if scales is None else scales.data_ptr(),
                                     _stream(device)))
    return out if keep is None else (out, kept)


def _pairs(w, dtype, K: int, offsets, device):
    """(groups, N, offsets' pointer) of weights [2, N, K], or [G, 2, N, K] with offsets."""
    _operand(w, "w", (dtype,), 3 + (offsets is not None), device)
    if w.shape[-3] != 2 or w.shape[-1] != K:
        raise SpmmError(SPMM_INVALID, f"w: shape {tuple(w.shape)}, expected [..., 2, N, {K}]")
    G, at = _groups(offsets, w.shape, device)
    N = w.shape[-2]
    _counts(G, 2 * N)
    return G, N, at


def gated_mm_backward(dh, x, w, kept, offsets=None, act: str = "silu", stream=None,
                      rows: bool = True, weights: bool = True, hidden: bool = False):
    """The gradients of ``gated_mm`` for dh [S, N]: (dx [S, K], dw like w), and with hidden
    the product act(g) * u again [S, N], for the gradient of what it was multiplied by.

    The gradients of g and u go into the products in dh's type, which rounds them once; in
    float16 a row's are multiplied by a power of two on their way, so that products of dh, u and
    act'(g) past float16's range at either end do not matter.
    kept is what ``gated_mm`` kept, in full or packed; x the operand, or packed by ``pack8``
    (only needed for weights).  N goes up to 2^21, ``gated_mm``'s to 2^22.  A gradient that is not asked for (rows=False,
    weights=False) is not computed and None."""
    act_id = _act_id(act)
    _half(dh, "dh")
    S, N = dh.shape
    device, dtype = dh.device, dh.dtype
    if not isinstance(w, torch.Tensor) or w.dim() < 1:
        _refuse(w, "w", (dtype,), 3, device)
    K = w.shape[-1]
    G, n, at = _pairs(w, dtype, K, offsets, device)
    if n != N:
        raise SpmmError(SPMM_INVALID, f"dh: shape {tuple(dh.shape)} for weights {tuple(w.shape)}")
    packed = isinstance(kept, Packed8)
    if packed:
        values = kept._checked("kept", (S, 2, N), device)
    else:
        _operand(kept, "kept", (dtype,), (S, 2, N), device)
        values = kept
    if weights:
        if isinstance(x, Packed8):
            x._checked("x", (S, K), device)
        else:
            _operand(x, "x", (dtype,), (S, K), device)
    _counts(S, K, 2 * N)
    if (rows or weights) and (N > _WIDEST_GRADIENT or K > 2 * _WIDEST_GRADIENT):
        raise SpmmError(SPMM_UNSUPPORTED, f"gradients for weights {tuple(w.shape)}: N over 2^21, whose "
                        "rows hold both projections', or K over 2^22")
    with _on(stream, device):
        L, s = lib(), _stream(device)
        h = torch.empty((S, N), dtype=dtype, device=device) if hidden else None
        dkept = torch.empty((S, 2, N), dtype=dtype, device=device)
        held = values.data_ptr(), kept.scales.data_ptr() if packed else None
        again = None if h is None else h.data_ptr()
        # float16's range: rows times a power of two each, and behind those the groups'
        scales = None
        if dtype == torch.float16:
            scales = torch.empty(S + G, dtype=torch.float32, device=device)
            _check(L.spmm_c_gated_grad_scaled(dh.data_ptr(), *held, S, N, act_id, dkept.data_ptr(),
                                              scales.data_ptr(), again, s))
        else:
            _check(L.spmm_c_gated_grad(dh.data_ptr(), _TYPES[dtype], *held, S, N, act_id,
                                       dkept.data_ptr(), again, s))
        dx = torch.empty((S, K), dtype=dtype, device=device) if rows else None
        dw = torch.empty_like(w) if weights else None
        if weights and isinstance(x, Packed8):
            x = unpack8(x, dtype)
        if rows or weights:
            operands = x.data_ptr() if weights else None, w.data_ptr()
            results = dx.data_ptr() if rows else None, dw.data_ptr() if weights else None
            if scales is None:
                _check(L.spmm_c_gated_mm_backward(dkept.data_ptr(), *operands, _TYPES[dtype], at, G, S, N,
                                                  K, *results, s))
            else:
                _check(L.spmm_c_gated_mm_backward_scaled(dkept.data_ptr(), scales.data_ptr(), *operands, at,
                                                         G, S, N, K, *results,
                                                         scales.data_ptr() + 4 * S, s))
    return (dx, dw, h) if hidden else (dx, dw)
