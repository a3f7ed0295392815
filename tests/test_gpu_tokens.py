"""Tokens into expert order and back against the 64-bit plain form."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402

SHAPES = [(1, 1, 1, 1), (1, 8, 2, 4096), (3, 5, 5, 7), (64, 64, 8, 129), (33, 4, 3, 2050),
          (4100, 6, 2, 40), (5000, 16, 1, 9), (2, 70, 64, 1000)]


def _routing(S, T, E, k, seed, masked=0.2):
    g = np.random.default_rng(seed)
    v = g.standard_normal((T, E))
    v[g.random((T, E)) < masked] = -np.inf
    v[g.random(T) < masked] = -np.inf
    return S.route(torch.from_numpy(v).float().cuda(), k)


def _values(shape, dtype, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape)).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,D", SHAPES)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_dispatch_and_back(S, T, E, k, D, name):
    dtype = R.TYPES[name]
    r = _routing(S, T, E, k, T + D)
    slots, weights = r.slots.cpu().numpy(), r.weights.double().cpu().numpy()
    x = _values((T, D), dtype, 1)
    xs = S.dispatch(x.cuda(), r)
    want = R.place(np.repeat(x.double().numpy()[:, None], k, 1), slots)
    assert np.array_equal(xs.double().cpu().numpy(), want)  # a copy: exact

    ys = _values((T * k, D), dtype, 2)
    # what no entry owns is never read
    ys_dev = ys.cuda()
    ys_dev[int(r.offsets[E]):] = float("nan")
    terms = weights[..., None] * R.take(ys.double().numpy(), slots)
    R.within(S.combine(ys_dev, r), terms.sum(1), np.abs(terms).sum(1), k)
    terms = R.take(ys.double().numpy(), slots)
    R.within(S.dispatch_backward(ys_dev, r), terms.sum(1), np.abs(terms).sum(1), k)

    dy = _values((T, D), dtype, 3)
    dys, dweights = S.combine_backward(dy.cuda(), ys_dev, r)
    g = dy.double().numpy()
    want = R.place(weights[..., None] * g[:, None], slots)
    R.within(dys, want, np.abs(want), 1)
    terms = R.take(ys.double().numpy(), slots) * g[:, None]
    assert dweights.dtype == torch.float32
    R.within(dweights, terms.sum(2), np.abs(terms).sum(2), D // 64 + 16)


@pytest.mark.gpu
def test_outputs_given_streams_and_unaligned_rows(S):
    T, E, k, D = 50, 6, 2, 37
    r = _routing(S, T, E, k, 9)
    base = _values((T * D + 1,), torch.bfloat16, 4).cuda()
    x = base[1:].view(T, D)  # 2-byte aligned
    assert x.data_ptr() % 4 == 2
    out = torch.empty((T * k, D), dtype=torch.bfloat16, device="cuda")
    assert S.dispatch(x, r, out=out) is out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    again = S.dispatch(x, r, stream=side)
    back = S.combine(again, r, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, again)
    # the weights of a token with an expert add up to one
    there = (r.slots >= 0).any(1)
    assert torch.allclose(back.float()[there], x.float()[there], rtol=2 ** -6, atol=0)
    assert (back[~there] == 0).all()


@pytest.mark.gpu
def test_no_tokens_and_no_features(S):
    r = S.route(torch.empty((0, 4), device="cuda"), 2)
    assert S.dispatch(torch.empty((0, 8), device="cuda"), r).shape == (0, 8)
    assert S.combine(torch.empty((0, 8), device="cuda"), r).shape == (0, 8)
    r = S.route(torch.zeros((3, 4), device="cuda"), 2)
    assert S.dispatch(torch.empty((3, 0), device="cuda"), r).shape == (6, 0)
    e = torch.empty((6, 0), device="cuda")
    dys, dw = S.combine_backward(torch.empty((3, 0), device="cuda"), e, r)
    assert dys.shape == (6, 0) and (dw == 0).all()


@pytest.mark.gpu
def test_gradients_against_differences(S):
    """combine and dispatch are linear in their rows: a step along the gradient moves the
    loss by the step times the gradient, within the roundings of the two sums."""
    T, E, k, D = 20, 5, 3, 24
    r = _routing(S, T, E, k, 3)
    ys, dy = _values((T * k, D), torch.float32, 5).cuda(), _values((T, D), torch.float32, 6).cuda()
    dys, dw = S.combine_backward(dy, ys, r)
    loss = lambda y: (y.double() * dy.double()).sum().item()  # noqa: E731
    base = loss(S.combine(ys, r))
    step = _values((T * k, D), torch.float32, 7).cuda()
    n = T * D * (k + 2) * 2.0 ** -24 * 40
    assert abs(loss(S.combine(ys + step, r)) - base - (dys.double() * step.double()).sum().item()) < n
    dr = _values((T, k), torch.float32, 8).cuda()
    moved = S.Routing(r.experts, r.weights + dr, r.offsets, r.entries, r.slots, r.over)
    assert abs(loss(S.combine(ys, moved)) - base - (dw.double() * dr.double()).sum().item()) < n
    x, dxs = _values((T, D), torch.float32, 9).cuda(), _values((T * k, D), torch.float32, 10).cuda()
    lhs = (S.dispatch(x, r).double() * dxs.double()).sum().item()
    rhs = (S.dispatch_backward(dxs, r).double() * x.double()).sum().item()
    assert abs(lhs - rhs) < n


@pytest.mark.gpu
def test_refusals(S):
    r = S.route(torch.zeros((4, 6), device="cuda"), 2)
    x = torch.zeros((4, 8), device="cuda")
    xs = torch.zeros((8, 8), device="cuda")
    wrong = S.Routing(r.experts, r.weights, r.offsets, r.entries, r.slots.long(), r.over)
    for bad in (lambda: S.dispatch(x[:3], r), lambda: S.dispatch(x.t(), r),
                lambda: S.dispatch(x.cpu(), r), lambda: S.dispatch(x.double(), r),
                lambda: S.dispatch(x, r, out=xs.half()), lambda: S.dispatch(x, r, out=xs[:7]),
                lambda: S.dispatch(x, wrong), lambda: S.combine(x, r), lambda: S.combine(xs.int(), r),
                lambda: S.combine(xs, r, out=x[:, :7]), lambda: S.dispatch_backward(x, r),
                lambda: S.combine_backward(x.half(), xs, r),
                lambda: S.combine_backward(x[:, :4].contiguous(), xs, r),
                lambda: S.dispatch(x, S.Routing(None, None, None, None, None))):
        with pytest.raises(S.SpmmError) as e:
            bad()
        assert e.value.code == S.SPMM_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,D,name", [(8200, 32, 8, 2050, "f32"), (2000, 40, 16, 2100, "f32"),
                                          (4100, 20, 8, 4099, "bf16"), (70000, 64, 8, 4000, "f16")])
def test_rows_beyond_the_caches(S, T, E, k, D, name):
    """256 MB and more in expert order; the last size has more than 2^31 elements there."""
    torch.manual_seed(T)
    r = S.route(torch.randn(T, E, device="cuda"), k)
    x = torch.randn(T, D, device="cuda").to(R.TYPES[name])
    xs = S.dispatch(x, r)
    assert torch.equal(xs, x[(r.entries // k).long()])  # copies: exact
    # a token's rows are all itself: k equal terms with weights that add up to one; the
    # weights carry 64 fp32 roundings, the sum k more
    y, back = S.combine(xs, r), S.dispatch_backward(xs, r)
    u = R.ROUNDOFF[x.dtype]
    off = (y.float() - x.float()).abs()
    assert (off <= (u + (64 + k) * 2.0 ** -24) * x.float().abs() + R.TINY[x.dtype]).all()
    off = (back.float() - k * x.float()).abs()
    assert (off <= (u + k * 2.0 ** -24) * k * x.float().abs() * (1 + u) + R.TINY[x.dtype]).all()
    dys, dw = S.combine_backward(x, xs, r)
    assert torch.equal(dys[-1], (x[r.entries[-1] // k].float() * r.weights.view(-1)[r.entries[-1]]).to(x.dtype))
    want = (x.double() ** 2).sum(1, keepdim=True)
    assert ((dw.double() - want).abs() <= (D // 64 + 16) * 2.0 ** -24 * want).all()
