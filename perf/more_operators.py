"""The operators of gated feed-forward blocks, trained with activations kept in 16
or 8 bits and served in 8-bit integers: the plain forms and the framework's kernels
on the same inputs.

A case names an operator (`op`) and its sizes:

  gated            act(x Wg^T) * (x Wu^T), with or without what its backward pass needs
  gated_grad       its gradients
  checkpoint       a tensor packed into 8 bits and unpacked again
  checkpoint_grad  gated's gradients from packed operands, and the product again
  int8             tokens quantised and multiplied by weights in 8-bit integers

`groups` 0 is one pair of weights for all rows, others have rows in group order, with
`spare` rows behind the last group.  `width` names the 16-bit type of the operands.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "sparse-matrix-multiplication_amd")

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
ACTS = ["silu", "gelu", "gelu_tanh"]
BLOCK = 32  # elements that share a packed scale

# Bounds of a drawn case, by the largest listed one of its operator.
MOST_PRODUCT = 16384 * 8192 * 4096  # rows x n x k of a forward product
MOST_WEIGHTS = 2 * 8192 * 8192      # elements of all groups' weights
MOST_PACKED = 16384 * 8192          # elements


def listed():
    return [
        # A serving step of 16 requests: both weights are read once.
        {"name": "gated_step", "op": "gated", "rows": 16, "groups": 0, "spare": 0, "n": 8192,
         "k": 4096, "act": "silu", "keep": False, "width": "bfloat16"},
        # The forward pass of a training step; the projections are kept.
        {"name": "gated_train", "op": "gated", "rows": 16384, "groups": 0, "spare": 0, "n": 8192,
         "k": 4096, "act": "silu", "keep": True, "width": "bfloat16"},
        # A short prompt over a few experts, sizes that are multiples of nothing.
        {"name": "gated_ragged", "op": "gated", "rows": 701, "groups": 5, "spare": 3, "n": 1003,
         "k": 2001, "act": "gelu", "keep": False, "width": "float16"},
        # The backward pass of a training step.
        {"name": "gated_grad", "op": "gated_grad", "rows": 8192, "groups": 0, "spare": 0, "n": 8192,
         "k": 4096, "act": "silu", "width": "bfloat16"},
        # The same over experts with ragged rows each.
        {"name": "gated_grad_experts", "op": "gated_grad", "rows": 20011, "groups": 16, "spare": 0,
         "n": 1408, "k": 2048, "act": "gelu_tanh", "width": "float16"},
        # A few tokens' activations: launch latency.
        {"name": "checkpoint_small", "op": "checkpoint", "rows": 61, "k": 1000,
         "width": "float16"},
        # A training step's hidden activations into 8 bits and back.
        {"name": "checkpoint_large", "op": "checkpoint", "rows": 16384, "k": 8192,
         "width": "bfloat16"},
        # Gradients from activations in 8 bits; the product for the next gradient is made again.
        {"name": "checkpoint_grad", "op": "checkpoint_grad", "rows": 8192, "groups": 0, "spare": 0,
         "n": 5632, "k": 2048, "act": "silu", "width": "bfloat16"},
        # The same over experts, widths that end inside a block.
        {"name": "checkpoint_grad_ragged", "op": "checkpoint_grad", "rows": 3001, "groups": 7,
         "spare": 5, "n": 1001, "k": 1030, "act": "gelu_tanh", "width": "float16"},
        # A serving step of 16 requests in 8-bit integers.
        {"name": "int8_step", "op": "int8", "rows": 16, "groups": 0, "spare": 0, "n": 8192,
         "k": 8192, "width": "bfloat16"},
        # A long prompt.
        {"name": "int8_prompt", "op": "int8", "rows": 8192, "groups": 0, "spare": 0, "n": 8192,
         "k": 8192, "width": "bfloat16"},
        # Prompts over experts, ragged sizes.
        {"name": "int8_experts", "op": "int8", "rows": 1009, "groups": 12, "spare": 2, "n": 1408,
         "k": 2050, "width": "float16"},
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _size(rng, lo, hi):
    """A size between lo and hi: half of them multiples of 64, the others anything."""
    v = int(_log(rng, lo, hi + 1))
    return v if rng.random() < 0.5 or v < 64 else v // 64 * 64


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_grad", "checkpoint", "checkpoint_grad", "int8", "int8"])
    width = rng.choice(sorted(TYPES))
    if op == "checkpoint":
        k = _size(rng, 16, 16384)
        return {"op": op, "rows": max(1, min(_size(rng, 1, 65536), MOST_PACKED // k)), "k": k,
                "width": width}
    n, k = _size(rng, 64, 8192), _size(rng, 64, 8192)
    most = MOST_PRODUCT // (n * k) // {"gated": 1, "int8": 1}.get(op, 2)
    groups = rng.choice([0, 0, int(_log(rng, 1, 65))])
    groups = min(groups, max(1, MOST_WEIGHTS // (2 * n * k)))
    rows = max(1, min(_size(rng, 1, 32768), most))
    case = {"op": op, "rows": rows, "groups": groups, "n": n, "k": k, "width": width,
            "spare": rng.choice([0, 0, rng.randint(1, 40)]) if groups else 0}
    if op != "int8":
        case["act"] = rng.choice(ACTS)
    if op == "gated":
        case["keep"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# Inputs, from the seed alone
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, width, scale=1.0, loud=0.0):
    """Normal values of the named type, made in pieces so that no large fp32 copy is held;
    a `loud` share of the last dimension's places is eight times as large."""
    out = torch.empty(shape, dtype=TYPES[width], device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        piece = flat[at:at + (1 << 26)]
        piece.copy_(torch.randn(piece.numel(), generator=g, device="cuda").mul_(scale))
    if loud:
        out[..., torch.rand(shape[-1], generator=g, device="cuda") < loud] *= 8
    return out


def _offsets(case, g):
    """Rows of each group: every row picks a group, some groups twice as popular as others."""
    popular = 1.0 + torch.rand(case["groups"], generator=g, device="cuda")
    ids = torch.multinomial(popular, case["rows"], replacement=True, generator=g)
    offsets = torch.zeros(case["groups"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(ids, minlength=case["groups"]).cumsum(0)
    return offsets


def prepare(case, seed):
    g, op, width = _generator(seed), case["op"], case["width"]
    k = case["k"]
    s = {"op": op, "type": TYPES[width]}
    if op == "checkpoint":
        # activations: some channels much larger than the rest, some tokens nearly silent
        x = _normal(g, (case["rows"], k), width, 1.0, 0.01)
        x[torch.rand(case["rows"], generator=g, device="cuda") < 0.02] *= 2.0 ** -8
        return s | {"x": x}
    rows, n, groups = case["rows"] + case["spare"], case["n"], case["groups"]
    s["offsets"] = _offsets(case, g) if groups else None
    x = _normal(g, (rows, k), width, 1.0, 0.005 if op == "int8" else 0.0)
    if op == "int8":
        # the weights are quantised once, when a program loads them
        w = _normal(g, (groups, n, k) if groups else (n, k), width, k ** -0.5)
        values, scales = _plain_quantise(w)
        padded = torch.zeros(values.shape[:-1] + ((k + 15) // 16 * 16,), dtype=torch.int8,
                             device="cuda")
        padded[..., :k] = values
        return s | {"x": x, "w": padded, "w_scales": scales}
    s["act"] = case["act"]
    s["w"] = _normal(g, (groups, 2, n, k) if groups else (2, n, k), width, k ** -0.5)
    if op == "gated":
        return s | {"x": x, "keep": case["keep"]}
    # what the forward pass kept: the projections' results are about as large as normal values
    kept = _normal(g, (rows, 2, n), width)
    s["dh"] = _normal(g, (rows, n), width)
    if op == "gated_grad":
        return s | {"x": x, "kept": kept}
    return s | {"x8": _plain_pack(x), "kept8": _plain_pack(kept)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
_fw = None


def _framework():
    global _fw
    if _fw is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import spmm_amd
        _fw = spmm_amd
    return _fw


def _run_own(s):
    S, op = _framework(), s["op"]
    if op == "gated":
        if not s["keep"]:
            return S.gated_mm(s["x"], s["w"], s["offsets"], act=s["act"])
        h, kept = S.gated_mm(s["x"], s["w"], s["offsets"], act=s["act"], keep="full")
        return {"h": h, "kept": kept}
    if op == "gated_grad":
        dx, dw = S.gated_mm_backward(s["dh"], s["x"], s["w"], s["kept"], s["offsets"],
                                     act=s["act"])
        return {"dx": dx, "dw": dw}
    if op == "checkpoint":
        return S.unpack8(S.pack8(s["x"]), s["type"])
    if op == "checkpoint_grad":
        dx, dw, h = S.gated_mm_backward(s["dh"], S.Packed8(*s["x8"]), s["w"],
                                        S.Packed8(*s["kept8"]), s["offsets"], act=s["act"],
                                        hidden=True)
        return {"dx": dx, "dw": dw, "h": h}
    return S.int8_mm(s["x"], S.Rows8(s["w"], s["w_scales"], s["x"].shape[1]), s["offsets"])


def _plain_act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = 2.0 * math.sqrt(2.0 / math.pi)
    p = 1.0 / (1.0 + torch.exp(-c * (g + 0.044715 * g * g * g)))
    return g * p, p + g * p * (1.0 - p) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain_pack(x):
    """(values int8 like x, scale bytes): blocks of 32 along the last dimension share the power
    of two of their largest value."""
    K = x.shape[-1]
    blocks = (K + BLOCK - 1) // BLOCK
    f = torch.zeros(x.shape[:-1] + (blocks * BLOCK,), device=x.device)
    f[..., :K] = x.float()
    f = f.view(x.shape[:-1] + (blocks, BLOCK))
    largest = f.abs().amax(-1)
    scale = (largest.view(torch.int32) >> 23).clamp(min=7)
    q = torch.round(f * (260 - scale << 23).view(torch.float32)[..., None]).clamp(-127, 127)
    return q.to(torch.int8).view(x.shape[:-1] + (-1,))[..., :K].contiguous(), scale.to(torch.uint8)


def _plain_unpack(packed):
    values, scale = packed
    step = (scale.int() - 6 << 23).view(torch.float32)
    return values.float() * step.repeat_interleave(BLOCK, -1)[..., :values.shape[-1]]


def _plain_quantise(x):
    """(values int8, scales fp32): the products with 127 / max, which is held in 32 bits, are
    formed in 64 bits, where they are exact, so that ties are ties."""
    largest = torch.amax(x.abs(), -1).float()
    there = largest > 0
    factor = torch.where(there, 127.0 / largest, 0.0)
    scales = torch.where(there, largest / 127.0, 0.0)
    values = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    flat, rows, by = values.view(-1, x.shape[-1]), x.reshape(-1, x.shape[-1]), factor.view(-1, 1)
    for at in range(0, rows.shape[0], 4096):
        piece = slice(at, at + 4096)
        flat[piece] = torch.round(rows[piece].double() * by[piece].double()).to(torch.int8)
    return values, scales


class _Groups:
    """Rows of each group from the first on, zeros to the longest group's length."""

    def __init__(self, offsets, rows):
        self.offsets, self.rows = offsets, rows
        if offsets is None:
            return
        counts = (offsets[1:] - offsets[:-1]).long()
        G, device = counts.numel(), offsets.device
        at = torch.arange(rows, device=device)
        # rows behind the last group go to a group of their own
        self.group = torch.bucketize(at, offsets[1:].long(), right=True)
        self.at = at - offsets.long()[self.group]
        self.shape = (G + 1, max(int(counts.max()), rows - int(offsets[-1])))

    def split(self, x):
        x = x.float()
        if self.offsets is None:
            return x
        padded = torch.zeros(self.shape + x.shape[1:], device=x.device)
        padded[self.group, self.at] = x
        return padded[:-1]

    def join(self, y):
        if self.offsets is None:
            return y
        return torch.cat([y, torch.zeros_like(y[:1])])[self.group, self.at]


def _run_plain(s):
    op = s["op"]
    if op == "checkpoint":
        return _plain_unpack(_plain_pack(s["x"])).to(s["type"])
    x = _plain_unpack(s["x8"]) if op == "checkpoint_grad" else s["x"]
    split = _Groups(s["offsets"], x.shape[0])
    if op == "int8":
        values, scales = _plain_quantise(x)
        k = x.shape[1]
        w = s["w"][..., :k].float() * s["w_scales"][..., None]
        y = split.join(split.split(values) @ w.transpose(-1, -2))
        return (y * scales[:, None]).to(s["type"])
    w = s["w"].float()
    wg, wu = w.unbind(-3)
    if op == "gated":
        rows = split.split(x)
        g, u = (split.join(rows @ m.transpose(-1, -2)) for m in (wg, wu))
        h = (_plain_act(g, s["act"])[0] * u).to(s["type"])
        return {"h": h, "kept": torch.stack([g, u], 1).to(s["type"])} if s["keep"] else h
    kept = _plain_unpack(s["kept8"]) if op == "checkpoint_grad" else s["kept"].float()
    g, u = kept.unbind(1)
    a, slope = _plain_act(g, s["act"])
    dh = s["dh"].float()
    dg, du = split.split(dh * u * slope), split.split(dh * a)
    rows = split.split(x)
    out = {"dx": split.join(dg @ wg + du @ wu).to(s["type"]),
           "dw": torch.stack([dg.transpose(-1, -2) @ rows, du.transpose(-1, -2) @ rows], -3).to(
               s["type"])}
    if op == "checkpoint_grad":
        out["h"] = (a * u).to(s["type"])
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without, and how exact it is
# ---------------------------------------------------------------------------
def work(case):
    op, k = case["op"], case["k"]
    packed = 1.0 + 1.0 / BLOCK
    if op == "checkpoint":
        return {"bytes": case["rows"] * k * 2 * (2 + packed), "flops": 0}
    S, n, G = case["rows"], case["n"], case["groups"]
    pairs = G * (1.0 - (1.0 - 1.0 / G) ** S) if G else 1.0  # weights of groups with rows
    rows = S + case["spare"]
    if op == "int8":
        return {"bytes": 2 * S * k + pairs * n * (k + 4) + 2 * rows * n, "flops": 2 * S * n * k}
    if op == "gated":
        return {"bytes": 2 * (S * k + 2 * pairs * n * k + rows * n * (3 if case["keep"] else 1)),
                "flops": 4 * S * n * k}
    held = 2 if op == "gated_grad" else packed
    weights = 2 * 2 * n * k * (pairs + max(G, 1))
    again = 2 * rows * n if op == "checkpoint_grad" else 0
    return {"bytes": held * S * (2 * n + k) + 2 * (S * n + rows * k) + weights + again,
            "flops": 8 * S * n * k}


def _exact_act(g, act):
    if act == "silu":
        a = g * torch.sigmoid(g)
        return a, torch.sigmoid(g) + a * torch.sigmoid(-g)
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g.square() / 2) / (2 * math.pi) ** 0.5
    t = (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
    slope = (2 / math.pi) ** 0.5 * (1 + 0.134145 * g ** 2)
    p = torch.sigmoid(2 * t)
    return g * p, p + 2 * g * p * torch.sigmoid(-2 * t) * slope


def _power(e):
    """2^e in 64 bits for whole e, from the bits: a power function may be off by its last bit."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_unpack(packed):
    values, scale = packed
    out = values.double()
    for at in range(scale.shape[-1]):
        part = out[..., at * BLOCK:(at + 1) * BLOCK]
        part *= _power(scale[..., at, None].long() - 133)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        x = s["x"].double()
        out = torch.empty_like(x)
        for at in range(0, x.shape[1], BLOCK):
            block = x[:, at:at + BLOCK]
            largest = block.abs().amax(1, keepdim=True)
            step = _power((torch.frexp(largest).exponent - 7).clamp(min=-126))
            out[:, at:at + BLOCK] = (block / step).round().clamp(-127, 127) * step
        return out
    x = _exact_unpack(s["x8"]) if op == "checkpoint_grad" else s["x"].double()
    rows, offsets = x.shape[0], s["offsets"]
    spans = [(0, rows)] if offsets is None else list(zip(offsets[:-1].tolist(), offsets[1:].tolist()))
    weights = s["w"][None] if offsets is None else s["w"]
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    if op == "int8":
        k = case["k"]
        by = torch.where(x.abs().amax(1) > 0, 127.0 / s["x"].float().abs().amax(1), 0.0)
        q = (x * by.double()[:, None]).round()
        back = (s["x"].float().abs().amax(1) / 127.0).double()
        scales = (s["w_scales"][None] if offsets is None else s["w_scales"]).double()
        y = zeros(rows, case["n"])
        for i, (lo, hi) in enumerate(spans):
            y[lo:hi] = q[lo:hi] @ weights[i, :, :k].double().t() * scales[i] * back[lo:hi, None]
        return y
    if op == "gated":
        h, kept = zeros(rows, case["n"]), zeros(rows, 2, case["n"])
        for i, (lo, hi) in enumerate(spans):
            for j in range(2):
                kept[lo:hi, j] = x[lo:hi] @ weights[i, j].double().t()
            h[lo:hi] = _exact_act(kept[lo:hi, 0], s["act"])[0] * kept[lo:hi, 1]
        return {"h": h, "kept": kept} if s["keep"] else h
    kept = _exact_unpack(s["kept8"]) if op == "checkpoint_grad" else s["kept"].double()
    a, slope = _exact_act(kept[:, 0], s["act"])
    dh = s["dh"].double()
    d = [dh * kept[:, 1] * slope, dh * a]
    dx, dw = zeros(rows, case["k"]), zeros(*weights.shape)
    for i, (lo, hi) in enumerate(spans):
        for j in range(2):
            dx[lo:hi] += d[j][lo:hi] @ weights[i, j].double()
            dw[i, j] = d[j][lo:hi].t() @ x[lo:hi]
    out = {"dx": dx, "dw": dw if offsets is not None else dw[0]}
    if op == "checkpoint_grad":
        out["h"] = a * kept[:, 1]
    return out
