"""A layer's experts in 8-bit integers are its experts as they were when they were made."""
import pytest

torch = pytest.importorskip("torch")


def test_router_is_a_copy(S, monkeypatch):
    from spmm_amd import expert_layer
    # quantising needs a GPU; what becomes of the router does not
    monkeypatch.setattr(expert_layer, "quantize_rows", lambda w: w.clone())
    layer = expert_layer.ExpertLayer(8, 16, 3, 1, device="cpu")
    experts = expert_layer.Int8Experts(layer)
    before = layer.router.detach().clone()
    with torch.no_grad():
        layer.router.add_(1.0)
    assert torch.equal(experts.router, before) and not experts.router.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "silu"])
def test_training_on_does_not_change_them(S, act):
    from spmm_amd.expert_layer import ExpertLayer, Int8Experts
    torch.manual_seed(0)
    layer = ExpertLayer(72, 100, 6, 2, gated=act)
    x = torch.randn(37, 72, device="cuda").bfloat16()
    experts = Int8Experts(layer)
    before = experts(x)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn_like(p))
    assert torch.equal(experts(x), before)
    layer.load_state_dict({n: torch.zeros_like(p) for n, p in layer.state_dict().items()})
    assert torch.equal(experts(x), before)
