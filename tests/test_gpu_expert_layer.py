"""The operators together, as a layer that is trained and served."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "sparse-matrix-multiplication_amd")


def _run(*args):
    return subprocess.run([sys.executable, "-m", "spmm_amd.expert_layer", *args],
                          env=dict(os.environ, PYTHONPATH=PKG), capture_output=True, text=True,
                          timeout=110)


def _plain(x, router, w_in, w_out, experts, over):
    """The layer in 64 bits for the experts chosen; differentiable."""
    logits = x @ router.t()
    if over == "all":
        weights = torch.softmax(logits, 1).gather(1, experts)
    else:
        weights = torch.softmax(logits.gather(1, experts), 1)
    rows = []
    for t in range(x.shape[0]):
        y = 0
        for j, e in enumerate(experts[t].tolist()):
            y = y + weights[t, j] * (w_out[e] @ torch.nn.functional.silu(w_in[e] @ x[t]))
        rows.append(y)
    return torch.stack(rows)


def _magnitudes(x, router, w_in, w_out, dy, weights, experts):
    """Bounds of the terms' magnitudes of the result and of each gradient: the formulas
    on absolute values, with |silu'| <= 1.1, |silu''| <= 0.5 and a softmax's derivative
    of at most 1 a weight (|w_j (d_j - sum w d)| <= 2 max |d|)."""
    x, router, w_in, w_out, dy = (v.abs() for v in (x, router, w_in, w_out, dy))
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dlogits = torch.zeros(x.shape[0], router.shape[0], dtype=torch.float64)
    dw_in, dw_out = torch.zeros_like(w_in), torch.zeros_like(w_out)
    for t in range(x.shape[0]):
        biggest = 0.0
        for j, e in enumerate(experts[t].tolist()):
            h = w_in[e] @ x[t]
            a = 1.1 * h
            ys = w_out[e] @ a
            y[t] += weights[t, j] * ys
            biggest = max(biggest, float(dy[t] @ ys))
            dys = weights[t, j] * dy[t]
            dw_out[e] += torch.outer(dys, a)
            dh = (w_out[e].t() @ dys) * (1.1 + 0.5 * h)
            dw_in[e] += torch.outer(dh, x[t])
            dx[t] += w_in[e].t() @ dh
        dlogits[t] = 2 * biggest
    return y, dx + dlogits @ router, dlogits.t() @ x, dw_in, dw_out


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,H,E,k,over", [(1, 8, 16, 2, 1, "chosen"), (33, 64, 96, 5, 2, "chosen"),
                                            (40, 50, 70, 4, 4, "all"), (64, 128, 64, 70, 3, "all")])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_layer_and_gradients(S, T, D, H, E, k, over, name):
    from spmm_amd.expert_layer import ExpertLayer
    torch.manual_seed(T)
    layer = ExpertLayer(D, H, E, k, over, R.TYPES[name])
    x = torch.randn(T, D).to(R.TYPES[name]).cuda().requires_grad_()
    dy = torch.randn(T, D).to(R.TYPES[name]).cuda()
    y = layer(x)
    y.backward(dy)
    experts = S.route(x.detach().float() @ layer.router.detach().t(), k, over).experts.long().cpu()
    wide = [v.detach().double().cpu().requires_grad_()
            for v in (x, layer.router, layer.w_in, layer.w_out)]
    want = _plain(*wide, experts, over)
    want.backward(dy.double().cpu())
    with torch.no_grad():
        logits = wide[0] @ wide[1].t()
        weights = (torch.softmax(logits, 1).gather(1, experts) if over == "all"
                   else torch.softmax(logits.gather(1, experts), 1))
        sizes = _magnitudes(*wide, dy.double().cpu(), weights, experts)
    # A result goes through at most 8 roundings to 16 bits (h, silu, ys, dys, da, dh,
    # dxs and itself), each at most the type's roundoff of its terms' magnitude and
    # passed on in proportion to the magnitudes; as many again cover the fp32 sums of up
    # to D, H or T terms and the products of two errors.
    got = [y, x.grad, layer.router.grad, layer.w_in.grad, layer.w_out.grad]
    exact = [want] + [v.grad for v in wide]
    for g, e, size in zip(got, exact, sizes):
        off = (g.detach().double().cpu() - e.detach()).abs()
        allowed = 16 * R.ROUNDOFF[R.TYPES[name]] * size + T * R.TINY[R.TYPES[name]]
        assert (off <= allowed).all(), float((off / allowed.clamp_min(1e-300)).max())


@pytest.mark.gpu
def test_serve(S):
    """One token a request: the layer's result goes into the adapters' projection."""
    from spmm_amd.expert_layer import ExpertLayer
    torch.manual_seed(1)
    layer = ExpertLayer(64, 128, 8, 2, dtype=torch.float16)
    x = torch.randn(5, 64).half().cuda()
    w, a, b = torch.randn(96, 64), torch.randn(3, 8, 64) / 8, torch.randn(3, 96, 8) / 3
    w, a, b = (t.half().cuda() for t in (w, a, b))
    ids = torch.tensor([2, -1, 0, 2, 1], dtype=torch.int32, device="cuda")
    got = layer.serve(x, w, a, b, ids)
    with torch.no_grad():
        z = (x + layer(x)).double()
    want = z @ w.double().t()
    size = z.abs() @ w.double().abs().t()
    low = torch.zeros_like(want)
    for t, i in enumerate(ids.tolist()):
        if i >= 0:
            h = a[i].double() @ z[t]
            want[t] += b[i].double() @ h
            low[t] = b[i].double().abs() @ (a[i].double().abs() @ z[t].abs())
    # h is rounded once to 16 bits; the fp32 sums have 64 and 8 terms more
    R.within(got, want.cpu().numpy(), (size + low * (1 + 2.0 ** -11 / (72 * 2.0 ** -24))).cpu().numpy(),
             72)


@pytest.mark.gpu
def test_command_line(S):
    out = _run("--tokens", "300", "--experts", "6", "--width", "128", "--hidden", "192", "--iters", "2")
    assert out.returncode == 0, out.stderr
    lines = out.stdout.splitlines()
    assert [line.split()[1] for line in lines] == ["kind=train", "kind=serve"]
    assert all("finite=yes" in line for line in lines)


def test_command_line_refuses():
    for bad in (["--k", "9", "--experts", "4"], ["--tokens", "0"], ["--dtype", "f64"]):
        out = _run(*bad)
        assert out.returncode == 2 and "error" in out.stderr
