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
