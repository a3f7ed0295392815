"""The widest gated products: rows of 2^22 elements forth, and of 2^21 back, where a row holds both
projections' gradients."""
import pytest

torch = pytest.importorskip("torch")

import gated_reference as G  # noqa: E402
import kernel_names  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.gpu
def test_forward(S):
    N, K = 1 << 22, 8
    x, w = _values((1, K), torch.bfloat16, 1), _values((2, N, K), torch.bfloat16, 2)
    g, u = (x.double() @ m.double().t() for m in w)
    eg, eu = (K * 2.0 ** -24 * (x.double().abs() @ m.double().abs().t()) for m in w)
    G.close(S.gated_mm(x, w), G.value(g, "silu") * u, G.product_bound(g, u, eg, eu, "silu"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_wider_gradients_are_refused_before_anything_runs(S, dtype):
    N, K = (1 << 21) + 8, 8
    x, w, dh, kept = (torch.zeros(s, dtype=dtype, device="cuda") for s in ((1, K), (2, N, K), (1, N), (1, 2, N)))
    seen = []

    def call(**which):
        seen.append(which)
        with pytest.raises(S.SpmmError) as e:
            S.gated_mm_backward(dh, x, w, kept, **which)
        assert e.value.code == S.SPMM_UNSUPPORTED and "2^21" in str(e.value)

    for which in ({}, {"rows": False}, {"weights": False}, {"hidden": True}):
        assert kernel_names.launches(lambda: call(**which)) == []
    assert len(seen) == 8
    # the product alone is no product's row
    *none, h = S.gated_mm_backward(dh, x, w, kept, rows=False, weights=False, hidden=True)
    assert none == [None, None] and (h == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_widest_gradients(S, dtype):
    N, K = 1 << 21, 8
    x, w = _values((1, K), dtype, 1), _values((2, N, K), dtype, 2, 2.0 ** -12)
    dh, kept = _values((1, N), dtype, 3), _values((1, 2, N), dtype, 4)
    dx, dw = S.gated_mm_backward(dh, x, w, kept)
    g, u = kept.double().unbind(1)
    dg, du, eg, eu = G.gradients(dh.double(), g, u, "silu")
    r, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25
    d, e = torch.cat([dg, du], 1), torch.cat([eg, eu], 1)
    e = e * (1 + r) + r * d.abs() + tiny
    W = w.double().view(2 * N, K)
    # fp32 sums of 2 N terms: 2 N 2^-24 of their magnitudes bounds any order
    G.close(dx, d @ W, (e + 2 * N * 2.0 ** -24 * (d.abs() + e)) @ W.abs())
    X = x.double()
    G.close(dw.view(2 * N, K), d.t() @ X, (e + 2.0 ** -24 * (d.abs() + e)).t() @ X.abs())
