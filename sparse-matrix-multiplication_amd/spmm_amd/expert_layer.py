"""A mixture-of-experts layer on the routing and product operators, trained and served.

    y[t] = sum_j weight[t, j] * W_out[e] silu(W_in[e] x[t]),   e = expert[t, j]

``ExpertLayer`` is a torch module: its forward and backward run ``route``,
``dispatch``, ``grouped_mm`` and ``combine`` and their gradients.  ``serve`` runs
the layer for the tokens of many requests and then a shared projection with each
request's own low-rank adapter (``adapter_mm``).

Usage:
    python -m spmm_amd.expert_layer [--tokens 4096] [--experts 16] [--k 2] [--width 1024]
                                    [--hidden 2048] [--adapters 8] [--rank 16]
                                    [--dtype bf16] [--iters 20]
prints one ``expert_layer ...`` line a workload: a training step over the tokens,
and one served step of a token for each of 16 requests.
"""
from __future__ import annotations

import argparse

import torch

from . import SPMM_UNSUPPORTED, SpmmError
from .experts import (adapter_mm, combine, combine_backward, dispatch, dispatch_backward,
                      grouped_mm, grouped_mm_backward, route, route_backward)

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


class _Experts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, logits, w_in, w_out, k, over):
        y, (r, xs, h, a, ys) = _forward(x, logits, w_in, w_out, k, over)
        ctx.save_for_backward(logits, w_in, w_out, xs, h, a, ys)
        ctx.routing = r
        return y

    @staticmethod
    def backward(ctx, dy):
        with torch.no_grad():
            grads = _Experts._gradients(ctx, dy)
        if not torch.is_grad_enabled():
            return grads
        # under create_graph: what the gradients hang on besides dy (which is all that
        # torch's once_differentiable looks at) goes along
        return _Once.apply(len(grads), *grads, dy, *ctx.saved_tensors[:3])

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


class ExpertLayer(torch.nn.Module):
    """`experts` two-layer networks of `width` and `hidden` units, `k` of them a token.
    The router's logits are held in float32; `over` is what its softmax runs over.
    Differentiable once; a second derivative raises."""

    def __init__(self, width: int, hidden: int, experts: int, k: int, over: str = "chosen",
                 dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        make = lambda *s, d=dtype: torch.nn.Parameter(  # noqa: E731
            torch.randn(s, device=device).mul_(s[-1] ** -0.5).to(d))
        self.router = make(experts, width, d=torch.float32)
        self.w_in = make(experts, hidden, width)
        self.w_out = make(experts, width, hidden)
        self.k, self.over = k, over

    def forward(self, x):
        """x [T, width], of any strides -> [T, width]"""
        x = x.contiguous()
        return _Experts.apply(x, x.float() @ self.router.t(), self.w_in, self.w_out, self.k,
                              self.over)

    @torch.no_grad()
    def serve(self, x, w, a, b, ids, scale=None):
        """The layer and its residual for tokens x [T, width] of requests whose adapters
        are ids [T], then the projection w with each row's adapter: [T, N]."""
        x = x.contiguous()
        y, _ = _forward(x, x.float() @ self.router.t(), self.w_in, self.w_out, self.k, self.over)
        return adapter_mm(x + y, w, a, b, ids, scale)


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
    args = p.parse_args(argv)
    for name in ("tokens", "experts", "k", "width", "hidden", "adapters", "rank", "iters"):
        if getattr(args, name) < 1:
            p.error(f"--{name} must be at least 1")
    if args.k > args.experts:
        p.error("--k is larger than --experts")
    if not torch.cuda.is_available():
        p.error("a GPU is needed")
    torch.manual_seed(0)
    dtype, dev = _DTYPES[args.dtype], "cuda"
    layer = ExpertLayer(args.width, args.hidden, args.experts, args.k, dtype=dtype)
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
    out = layer.serve(xs, w, a, b, ids)
    finite &= torch.isfinite(out).all().item()
    print(f"expert_layer kind=serve tokens={T} {sizes} adapters={args.adapters} rank={args.rank} "
          f"time_us={_microseconds(lambda: layer.serve(xs, w, a, b, ids), args.iters):.1f} "
          f"finite={'yes' if finite else 'no'}")
    return 0 if finite else 1


if __name__ == "__main__":
    raise SystemExit(main())
