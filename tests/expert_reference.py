"""Plain 64-bit forms of the routing and product operators, on the CPU, and the
bounds that their tests use.

Unit roundoffs: fp32 2^-24, fp16 2^-11, bf16 2^-8.  A result held in fp32 over n
roundings and rounded once to its type is within u_type |r| + n 2^-24 sum|terms|
of the exact one (n 2^-24 sum|terms| bounds any order of a sum of n roundings).
"""
from __future__ import annotations

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def within(got: torch.Tensor, want: np.ndarray, scale: np.ndarray, roundings: int) -> None:
    """got against the 64-bit result; scale = the sum of the terms' magnitudes."""
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.shape
    assert np.array_equal(np.isfinite(g), np.isfinite(want))
    fine = np.isfinite(want)
    bound = (ROUNDOFF[got.dtype] * (np.abs(want) + roundings * 2.0 ** -24 * scale)
             + roundings * 2.0 ** -24 * scale + TINY[got.dtype])
    off = np.abs(np.where(fine, g, 0) - np.where(fine, want, 0))
    bad = (off > bound) & fine
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[0].tolist(),
                           float((off / bound)[fine].max()))


def route(logits: np.ndarray, k: int, over: str):
    """(experts, weights, offsets, entries, slots) in 64 bits, one token at a time."""
    T, E = logits.shape
    experts = np.full((T, k), -1, np.int64)
    weights = np.zeros((T, k))
    for t in range(T):
        row = logits[t].astype(np.float64)
        nan = np.isnan(row)
        order = sorted((e for e in range(E) if row[e] != -np.inf),
                       key=lambda e: (not nan[e], 0.0 if nan[e] else -row[e], e))[:k]
        experts[t, :len(order)] = order
        if order:
            with np.errstate(invalid="ignore", over="ignore"):
                m = row[order[0]]
                e = np.exp(row - m)
                weights[t, :len(order)] = e[order] / (e[order] if over == "chosen" else e).sum()
    return (experts, weights) + group(experts.reshape(-1), E, experts.shape)


def group(ids: np.ndarray, groups: int, shape):
    ids = np.asarray(ids).reshape(-1)
    inside = (ids >= 0) & (ids < groups)
    order = np.argsort(np.where(inside, ids, groups), kind="stable")
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids[inside], minlength=groups))])
    entries = np.full(ids.size, -1, np.int64)
    slots = np.full(ids.size, -1, np.int64)
    placed = order[:inside.sum()]
    entries[:placed.size] = placed
    slots[placed] = np.arange(placed.size)
    return offsets, entries, slots.reshape(shape)


def route_grad(logits, experts, weights, dweights, over):
    d = np.zeros(logits.shape)
    p = np.zeros(logits.shape)
    if over == "all":
        m = logits.max(1, keepdims=True)
        e = np.exp(logits - np.where(np.isfinite(m), m, 0.0))
        p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    for t in range(logits.shape[0]):
        on = experts[t] >= 0
        dot = (weights[t] * dweights[t])[on].sum()
        if over == "chosen":
            d[t, experts[t, on]] = (weights[t] * (dweights[t] - dot))[on]
        else:
            g = np.full(logits.shape[1], -dot)
            g[experts[t, on]] += dweights[t, on]
            d[t] = p[t] * g
    return d


def take(rows: np.ndarray, slots: np.ndarray) -> np.ndarray:
    """rows[slots], zeros where there is no slot."""
    out = np.zeros(slots.shape + rows.shape[1:])
    out[slots >= 0] = rows[slots[slots >= 0]]
    return out


def place(values: np.ndarray, slots: np.ndarray) -> np.ndarray:
    """values[t, j] into row slots[t, j], zeros elsewhere."""
    out = np.zeros((slots.size,) + values.shape[2:])
    out[slots[slots >= 0]] = values[slots >= 0]
    return out
