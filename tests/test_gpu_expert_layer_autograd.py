"""What the layer's autograd gives, refuses and leaves out."""
import pytest

torch = pytest.importorskip("torch")


def _layer(T=40, D=64, H=96, E=5):
    from spmm_amd.expert_layer import ExpertLayer
    torch.manual_seed(T)
    layer = ExpertLayer(D, H, E, 2)
    x = torch.randn(T, D, device="cuda").bfloat16().requires_grad_()
    return layer, x, torch.randn(T, D, device="cuda").bfloat16()


@pytest.mark.gpu
def test_second_derivative_is_refused(S):
    """A gradient penalty through the layer raises; its terms are not left out in silence."""
    layer, x, dy = _layer()
    y = layer(x)
    g, = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(S.SpmmError) as e:
        (g.float().square().sum() + x.float().sum()).backward()
    assert e.value.code == S.SPMM_UNSUPPORTED
    # the same values as without a graph, and a loss that curves is no different
    y = layer(x)
    plain, = torch.autograd.grad(y, x, dy)
    assert torch.equal(plain, g)
    loss = layer(x).float().square().sum()
    g, = torch.autograd.grad(loss, layer.w_in, create_graph=True)
    with pytest.raises(S.SpmmError):
        torch.autograd.grad(g.float().sum(), x)


def _launches(monkeypatch):
    """Names of the products' gradients that are computed."""
    import spmm_amd.experts as X
    real, seen = X.lib(), []

    class Watched:
        def __getattr__(self, name):
            if name in ("spmm_c_grouped_mm", "spmm_c_grouped_outer"):
                seen.append(name)
            return getattr(real, name)

    monkeypatch.setattr(X, "lib", lambda: Watched())
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("frozen,products,outers", [
    ((), 2, 2), (("w_in", "w_out"), 2, 0), (("w_in",), 2, 1), (("w_out",), 2, 1), (("x",), 1, 2),
    (("x", "router", "w_in"), 0, 1), (("x", "w_in", "w_out"), 0, 0)])
def test_frozen_parts_cost_nothing(S, monkeypatch, frozen, products, outers):
    """What is not trained gets no gradient and no product for one; the rest is unchanged."""
    layer, x, dy = _layer()
    names = {"x": x, "router": layer.router, "w_in": layer.w_in, "w_out": layer.w_out}
    want = dict(zip(names, torch.autograd.grad(layer(x), list(names.values()), dy)))
    for n in frozen:
        names[n].requires_grad_(False)
    y = layer(x)
    seen = _launches(monkeypatch)
    y.backward(dy)
    assert (seen.count("spmm_c_grouped_mm"), seen.count("spmm_c_grouped_outer")) == (products, outers)
    for n, v in names.items():
        assert v.grad is None if n in frozen else torch.equal(v.grad, want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("w_in_rows", [False, True])
def test_one_gradient_of_a_product(S, w_in_rows):
    torch.manual_seed(0)
    x, dy = torch.randn(50, 24, device="cuda").half(), torch.randn(50, 40, device="cuda").half()
    w = torch.randn(3, *((24, 40) if w_in_rows else (40, 24)), device="cuda").half()
    offsets = torch.tensor([0, 20, 20, 45], dtype=torch.int32, device="cuda")
    dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows)
    only, none = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows, weights=False)
    assert none is None and torch.equal(only, dx)
    none, only = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows, rows=False)
    assert none is None and torch.equal(only, dw)


@pytest.mark.gpu
def test_rows_of_any_strides(S):
    """A transposed or sliced x gives what its copy gives, gradients included."""
    layer, x, dy = _layer(T=40, D=64)
    want = layer(x)
    want.backward(dy)
    wide = torch.zeros(40, 80, device="cuda", dtype=x.dtype)
    wide[:, 8:72] = x.detach()
    w, a, b = (torch.randn(s, device="cuda").bfloat16() for s in ((64, 64), (2, 8, 64), (2, 64, 8)))
    ids = (torch.arange(40, device="cuda", dtype=torch.int32) % 3) - 1
    served = layer.serve(x.detach(), w, a, b, ids)
    for base, view in ((wide, lambda t: t[:, 8:72]), (x.detach().t().contiguous(), lambda t: t.t())):
        base = base.clone().requires_grad_()
        assert not view(base).is_contiguous()
        y = layer(view(base))
        y.backward(dy)
        assert torch.equal(y, want) and torch.equal(view(base.grad), x.grad)
        assert torch.equal(layer.serve(view(base.detach()), w, a, b, ids), served)
