"""Plain 64-bit forms of gated products, packed activations and 8-bit integers, and the
bounds that their tests use (roundoffs as in expert_reference.py).

The activations are g p(g); the kernels' p is off by `share_error` of itself:
  silu, gelu_tanh  p = 1 / (1 + e^-t): the power of two's argument is t times a constant, off
                   by |t| of some 2^-24 (gelu_tanh's t has five more roundings, all of
                   factors or of sums of one sign); power, sum and reciprocal by a few
                   2^-24 each: (6 |t| + 8) 2^-24
  gelu             p = erfc(-g / sqrt 2) / 2: the argument is off by 2 2^-24 of itself, by
                   which p changes by at most (g^2 + 1) times as much; erfc itself by at
                   most 16 2^-24: (2 g^2 + 18) 2^-24
and by what underflows, 2^-126.  act' is p + g p' with p' off as p is, twice for p (1 - p)
(1 - p where it is small is off by 2^-23 beside p): 4 share_error |g p'| + 2^-22 |g| p beside p's.
"""
from __future__ import annotations

import math

import numpy as np
import torch

import expert_reference as R

ACTS = ("silu", "gelu", "gelu_tanh")
TINY = 2.0 ** -126


def share(g, act):
    """p(g), g p'(g) and p's error relative to it, in 64 bits."""
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        return p, g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi), (2 * g * g + 18) * 2.0 ** -24
    t = g if act == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    dt = torch.ones_like(g) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    p, q = torch.sigmoid(t), torch.sigmoid(-t)
    return p, g * p * q * dt, (6 * t.abs() + 8) * 2.0 ** -24


def value(g, act):
    return g * share(g, act)[0]


def close(got, want, bound):
    """got within `bound` (before its own rounding) and a rounding to its type."""
    u = R.ROUNDOFF[got.dtype]
    g = got.double()
    assert g.shape == want.shape
    assert torch.equal(torch.isfinite(g), torch.isfinite(want))
    allowed = u * want.abs() + (1 + u) * bound + R.TINY[got.dtype]
    over = torch.where(torch.isfinite(want), (g - want).abs() / allowed, 0.0)
    assert (over <= 1).all(), (float(over.max()), int((over > 1).sum()),
                               (over > 1).nonzero()[0].tolist())


def product_bound(g, u, eg, eu, act):
    """How far act(g) u is off when g and u are, by eg and eu, and with the kernel's p."""
    p, _, rel = share(g, act)
    a = g * p
    ea = 1.13 * eg + (rel + 2.0 ** -23) * a.abs() + TINY * g.abs()  # |act'| < 1.13
    return ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs()


def gradients(dh, g, u, act):
    """dg, du and their errors in fp32."""
    p, gp, rel = share(g, act)
    dg, du = dh * u * (p + gp), dh * g * p
    es = rel * p + 4 * rel * gp.abs() + 2.0 ** -22 * (g.abs() * p + gp.abs() + p) + TINY * (1 + g.abs())
    eg = (dh * u).abs() * es + 2.0 ** -22 * dg.abs()
    eu = dh.abs() * ((rel + 2.0 ** -22) * (g * p).abs() + TINY * g.abs())
    return dg, du, eg, eu


# ---------------------------------------------------------------------------
# values in eight bits, with numpy
# ---------------------------------------------------------------------------
def pack(x: np.ndarray):
    """(q int8, scale uint8) of fp32 values, blocks of 32 along the last dimension."""
    K = x.shape[-1]
    blocks = -(-K // 32)
    f = np.zeros(x.shape[:-1] + (blocks * 32,), np.float32)
    f[..., :K] = x
    f = f.reshape(x.shape[:-1] + (blocks, 32))
    bits = np.abs(f).view(np.uint32).max(-1)
    none = bits >= 0x7f800000
    scale = np.where(none, 255, np.maximum(bits >> 23, 7)).astype(np.int64)
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.rint(np.ldexp(f.astype(np.float64), (133 - scale)[..., None]))
        q = np.where(none[..., None], 0, np.clip(q, -127, 127))
    q = np.nan_to_num(q).astype(np.int8).reshape(x.shape[:-1] + (blocks * 32,))[..., :K]
    return q, scale.astype(np.uint8)


def unpack(q: np.ndarray, scale: np.ndarray) -> np.ndarray:
    s = np.repeat(scale.astype(np.int64), 32, -1)[..., :q.shape[-1]]
    return np.where(s == 255, np.nan, np.ldexp(q.astype(np.float64), s - 133))


def quantise(x: np.ndarray):
    """(q int8 padded to whole 16s, scale fp32) of rows of fp32 values."""
    K = x.shape[-1]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        most = np.abs(x).view(np.uint32).max(-1).view(np.float32)
        fine = np.isfinite(most)
        largest = np.maximum(most, np.float32(2.0 ** -100))
        up = np.where(fine, np.float32(1) / largest * np.float32(127), np.float32(0)).astype(np.float32)
        q = np.rint(x.astype(np.float64) * up.astype(np.float64)[..., None])
        scale = np.where(fine, np.where(most == 0, np.float32(0), largest * (np.float32(1) / np.float32(127))),
                         np.float32(np.nan)).astype(np.float32)
    q = np.where(fine[..., None], q, 0)
    out = np.zeros(x.shape[:-1] + (-(-K // 16) * 16,), np.int8)
    out[..., :K] = q
    return out, scale
