"""A mixture-of-experts layer on the routing and product operators, trained and served.

    y[t] = sum_j weight[t, j] * W_out[e] silu(W_in[e] x[t]),   e = expert[t, j]

or with gated experts

    y[t] = sum_j weight[t, j] * W_out[e] (act(W_in[e, 0] x[t]) * (W_in[e, 1] x[t]))

``ExpertLayer`` is a torch module: its forward and backward run ``route``,
``dispatch``, ``grouped_mm`` (gated: ``gated_mm``) and ``combine`` and their gradients,
gated ones from activations kept in 16 or 8 bits.  ``serve`` runs the layer for the tokens
of many requests and then a shared projection with each request's own low-rank adapter
(``adapter_mm``).  ``Int8Experts`` is a layer's experts in 8-bit integers, to serve it.

Usage:
    python -m spmm_amd.expert_layer [--tokens 4096] [--experts 16] [--k 2] [--width 1024]
                                    [--hidden 2048] [--adapters 8] [--rank 16]
                                    [--dtype bf16] [--iters 20]
                                    [--gated {silu,gelu,gelu_tanh}] [--keep {full,8bit}] [--int8]
prints one ``expert_layer ...`` line a workload: a training step over the tokens,
one served step of a token for each of 16 requests, and with --int8 the same step with the
experts in 8-bit integers.
"""
from __future__ import annotations

import argparse

import torch

from . import SPMM_INVALID, SPMM_UNSUPPORTED, SpmmError
from .experts import (adapter_mm, combine, combine_backward, dispatch, dispatch_backward,
                      grouped_mm, grouped_mm_backward, route, route_backward)
from .gated import (_ACTS, Packed8, gated_mm, gated_mm_backward, int8_mm, pack8, quantize_rows,
                    unpack8)

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _forward(x, logits, w_in, w_out, k, over):
    r = route(logits, k, over)
    xs = dispatch(x, r)
    h = grouped_mm(xs, w_in, r.offsets)
    a = torch.nn.functional.silu(h)
    ys = grouped_mm(a, w_out, r.offsets)
    return combine(ys, r), (r, xs, h, a, ys)


class _Once(torch.autograd.Function):
    """Hands gradients on (the first n) that kernels computed without a graph from the rest:
    going back through them is refused, where it would count as zero otherwise."""

    @staticmethod
    def forward(ctx, n, *grads):
        return tuple(g if g is None else g.view_as(g) for g in grads[:n])

    @staticmethod
    def backward(ctx, *_):
        raise SpmmError(SPMM_UNSUPPORTED, "expert layer: differentiable once, no second derivative")


def _once(ctx, dy, gradients):
    """gradients(ctx, dy), to go back through once."""
    with torch.no_grad():
        grads = gradients(ctx, dy)
    if not torch.is_grad_enabled():
        return grads
    # under create_graph: what the gradients hang on besides dy (which is all that
    # torch's once_differentiable looks at) goes along
    return _Once.apply(len(grads), *grads, dy, *ctx.saved_tensors[:3])


class _Experts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, logits, w_in, w_out, k, over):
        y, (r, xs, h, a, ys) = _forward(x, logits, w_in, w_out, k, over)
        ctx.save_for_backward(logits, w_in, w_out, xs, h, a, ys)
        ctx.routing = r
        return y

    @staticmethod
    def backward(ctx, dy):
        return _once(ctx, dy, _Experts._gradients)

    @staticmethod
    def _gradients(ctx, dy):
        logits, w_in, w_out, xs, h, a, ys = ctx.saved_tensors
        r = ctx.routing
        of_x, of_logits, of_in, of_out = ctx.needs_input_grad[:4]
        dx = dlogits = dw_in = dw_out = None
        dys, dweights = combine_backward(dy.contiguous(), ys, r)
        if of_logits:
            dlogits = route_backward(logits, r, dweights)
        hidden = of_x or of_in
        if hidden or of_out:
            da, dw_out = grouped_mm_backward(dys, a, w_out, r.offsets, rows=hidden, weights=of_out)
        if hidden:
            dh = torch.ops.aten.silu_backward(da, h)
            dxs, dw_in = grouped_mm_backward(dh, xs, w_in, r.offsets, rows=of_x, weights=of_in)
        if of_x:
            dx = dispatch_backward(dxs, r)
        return dx, dlogits, dw_in, dw_out, None, None


class _GatedExperts(torch.autograd.Function):
    """Kept in 16 bits: the tokens in expert order, both projections, their product and the
    experts' results.  In 8: the tokens in their own order, which there are fewer of, both
    projections and the results; the product is made again."""

    @staticmethod
    def forward(ctx, x, logits, w_in, w_out, k, over, act, keep):
        r = route(logits, k, over)
        xs = dispatch(x, r)
        h, kept = gated_mm(xs, w_in, r.offsets, act=act, keep=keep)
        ys = grouped_mm(h, w_out, r.offsets)
        if keep == "full":
            ctx.save_for_backward(logits, w_in, w_out, xs, kept, h, ys)
        else:
            x8, ys8 = pack8(x), pack8(ys)
            ctx.save_for_backward(logits, w_in, w_out, x8.values, x8.scales, kept.values, kept.scales,
                                  ys8.values, ys8.scales)
        ctx.routing, ctx.act = r, act
        return combine(ys, r)

    @staticmethod
    def backward(ctx, dy):
        return _once(ctx, dy, _GatedExperts._gradients)

    @staticmethod
    def _gradients(ctx, dy):
        logits, w_in, w_out, *kept = ctx.saved_tensors
        r, act, eight = ctx.routing, ctx.act, len(kept) == 6
        of_x, of_logits, of_in, of_out = ctx.needs_input_grad[:4]
        dx = dlogits = dw_in = dw_out = h = None
        if eight:
            x8, kept, ys8 = (Packed8(*kept[i:i + 2]) for i in (0, 2, 4))
            ys = unpack8(ys8, w_in.dtype)
            xs = dispatch(unpack8(x8, w_in.dtype), r) if of_in else None
        else:
            xs, kept, h, ys = kept
        dys, dweights = combine_backward(dy.contiguous(), ys, r)
        if of_logits:
            dlogits = route_backward(logits, r, dweights)
        hidden = of_x or of_in
        again = eight and of_out  # the product, from what was kept of its factors
        if hidden or again:
            dh = grouped_mm(dys, w_out, r.offsets, w_in_rows=True)
            dxs, dw_in, *made = gated_mm_backward(dh, xs, w_in, kept, r.offsets, act=act, rows=of_x,
                                                  weights=of_in, hidden=again)
            h = made[0] if again else h
        if of_out:
            _, dw_out = grouped_mm_backward(dys, h, w_out, r.offsets, rows=False)
        if of_x:
            dx = dispatch_backward(dxs, r)
        return dx, dlogits, dw_in, dw_out, None, None, None, None


class ExpertLayer(torch.nn.Module):
    """`experts` two-layer networks of `width` and `hidden` units, `k` of them a token.
    The router's logits are held in float32; `over` is what its softmax runs over.
    Differentiable once; a second derivative raises.

    gated: None for silu between the layers, or the activation of gated experts ("silu",
    "gelu", "gelu_tanh"), whose w_in is [experts, 2, hidden, width].  keep: what gated
    experts keep for the backward pass, "full" or "8bit"."""

    def __init__(self, width: int, hidden: int, experts: int, k: int, over: str = "chosen",
                 dtype=torch.bfloat16, device="cuda", gated=None, keep: str = "full"):
        super().__init__()
        if gated is not None and (not isinstance(gated, str) or gated not in _ACTS):
            raise SpmmError(SPMM_INVALID, f"gated: {gated!r}, expected None or one of {sorted(_ACTS)}")
        if keep not in ("full", "8bit"):
            raise SpmmError(SPMM_INVALID, f"keep: {keep!r}, expected 'full' or '8bit'")
        if keep == "8bit" and gated is None:
            raise SpmmError(SPMM_UNSUPPORTED, "keep: 8 bits are gated experts'")
        make = lambda *s, d=dtype: torch.nn.Parameter(  # noqa: E731
            torch.randn(s, device=device).mul_(s[-1] ** -0.5).to(d))
        self.router = make(experts, width, d=torch.float32)
        self.w_in = make(*((experts,) if gated is None else (experts, 2)), hidden, width)
        self.w_out = make(experts, width, hidden)
        self.k, self.over, self.gated, self.keep = k, over, gated, keep

    def forward(self, x):
        """x [T, width], of any strides -> [T, width]"""
        x = x.contiguous()
        logits = x.float() @ self.router.t()
        if self.gated is None:
            return _Experts.apply(x, logits, self.w_in, self.w_out, self.k, self.over)
        if not torch.is_grad_enabled():
            return self._served(x, logits)
        return _GatedExperts.apply(x, logits, self.w_in, self.w_out, self.k, self.over, self.gated,
                                   self.keep)

    def _served(self, x, logits):
        if self.gated is None:
            return _forward(x, logits, self.w_in, self.w_out, self.k, self.over)[0]
        r = route(logits, self.k, self.over)
        h = gated_mm(dispatch(x, r), self.w_in, r.offsets, act=self.gated)
        return combine(grouped_mm(h, self.w_out, r.offsets), r)

    @torch.no_grad()
    def serve(self, x, w, a, b, ids, scale=None):
        """The layer and its residual for tokens x [T, width] of requests whose adapters
        are ids [T], then the projection w with each row's adapter: [T, N]."""
        x = x.contiguous()
        return adapter_mm(x + self._served(x, x.float() @ self.router.t()), w, a, b, ids, scale)


class Int8Experts:
    """A layer's experts in 8-bit integers with a scale a channel, made from it once: changing
    the layer later does not change them.  Tokens and what is between the layers get a scale a
    row.  The router stays in float32."""

    @torch.no_grad()
    def __init__(self, layer: ExpertLayer):
        self.router = layer.router.detach().clone()
        self.w_in = quantize_rows(layer.w_in.detach())
        self.w_out = quantize_rows(layer.w_out.detach())
        self.k, self.over, self.gated = layer.k, layer.over, layer.gated

    @torch.no_grad()
    def __call__(self, x):
        """x [T, width], of any strides -> [T, width]"""
        x = x.contiguous()
        r = route(x.float() @ self.router.t(), self.k, self.over)
        xs = dispatch(x, r)
        if self.gated is None:
            h = torch.nn.functional.silu(int8_mm(xs, self.w_in, r.offsets))
        else:
            h = gated_mm(xs, self.w_in, r.offsets, act=self.gated)
        return combine(int8_mm(h, self.w_out, r.offsets), r)

    @torch.no_grad()
    def serve(self, x, w, a, b, ids, scale=None):
        """As ``ExpertLayer.serve``."""
        x = x.contiguous()
        return adapter_mm(x + self(x), w, a, b, ids, scale)


def _microseconds(call, iters: int) -> float:
    for _ in range(3):
        call()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(iters):
        call()
    stop.record()
    stop.synchronize()
    return 1000 * start.elapsed_time(stop) / iters


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 4096), ("experts", 16), ("k", 2), ("width", 1024),
                        ("hidden", 2048), ("adapters", 8), ("rank", 16), ("iters", 20)):
        p.add_argument(f"--{name}", type=int, default=value)
    p.add_argument("--dtype", choices=sorted(_DTYPES), default="bf16")
    p.add_argument("--gated", choices=sorted(_ACTS))
    p.add_argument("--keep", choices=["full", "8bit"], default="full")
    p.add_argument("--int8", action="store_true")
    args = p.parse_args(argv)
    for name in ("tokens", "experts", "k", "width", "hidden", "adapters", "rank", "iters"):
        if getattr(args, name) < 1:
            p.error(f"--{name} must be at least 1")
    if args.k > args.experts:
        p.error("--k is larger than --experts")
    if args.keep == "8bit" and args.gated is None:
        p.error("--keep 8bit needs --gated")
    if not torch.cuda.is_available():
        p.error("a GPU is needed")
    torch.manual_seed(0)
    dtype, dev = _DTYPES[args.dtype], "cuda"
    layer = ExpertLayer(args.width, args.hidden, args.experts, args.k, dtype=dtype,
                        gated=args.gated, keep=args.keep)
    x = torch.randn(args.tokens, args.width, device=dev).to(dtype).requires_grad_()
    goal = torch.randn(args.tokens, args.width, device=dev)
    params = [x] + list(layer.parameters())

    def train():
        loss = (layer(x).float() - goal).square().mean()
        return loss, torch.autograd.grad(loss, params)

    loss, grads = train()
    finite = all(torch.isfinite(g).all().item() for g in grads)
    sizes = (f"experts={args.experts} k={args.k} width={args.width} hidden={args.hidden} "
             f"dtype={args.dtype}")
    if args.gated is not None:
        sizes += f" gated={args.gated} keep={args.keep}"
    print(f"expert_layer kind=train tokens={args.tokens} {sizes} "
          f"time_us={_microseconds(train, args.iters):.1f} loss={loss.item():.6f} "
          f"finite={'yes' if finite else 'no'}")

    T = 16
    w = torch.randn(args.width, args.width, device=dev).mul_(args.width ** -0.5).to(dtype)
    a = torch.randn(args.adapters, args.rank, args.width, device=dev).mul_(args.width ** -0.5)
    b = torch.randn(args.adapters, args.width, args.rank, device=dev).mul_(args.rank ** -0.5)
    ids = torch.arange(T, dtype=torch.int32, device=dev) % (args.adapters + 1) - 1
    xs = torch.randn(T, args.width, device=dev).to(dtype)
    a, b = a.to(dtype), b.to(dtype)
    served = [("serve", layer)] + ([("serve_int8", Int8Experts(layer))] if args.int8 else [])
    for kind, experts in served:
        out = experts.serve(xs, w, a, b, ids)
        finite &= torch.isfinite(out).all().item()
        print(f"expert_layer kind={kind} tokens={T} {sizes} adapters={args.adapters} rank={args.rank} "
              f"time_us={_microseconds(lambda: experts.serve(xs, w, a, b, ids), args.iters):.1f} "
              f"finite={'yes' if finite else 'no'}")
    return 0 if finite else 1


if __name__ == "__main__":
    raise SystemExit(main())
