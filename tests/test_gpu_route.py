"""Routing of tokens to experts against its 64-bit plain form: choices and order
exactly, weights and gradients within the bounds of their roundings."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402


def _logits(T, E, dtype, seed, masked=0.0, ties=False):
    g = np.random.default_rng(seed)
    v = g.uniform(-4.0, 4.0, (T, E))
    if ties:
        v = np.round(v)  # many equal logits, zeros of both signs among them
    if masked:
        v[g.random((T, E)) < masked] = -np.inf
        v[g.random(T) < masked] = -np.inf
    return torch.from_numpy(v).to(dtype)


def _check_order(r, want):
    experts, _, offsets, entries, slots = want
    for got, w in ((r.experts, experts), (r.offsets, offsets), (r.entries, entries),
                   (r.slots, slots)):
        assert np.array_equal(got.cpu().numpy(), w)


# |l - m| <= 8 after the subtraction: its rounding moves exp by 8 * 2^-24, expf by 2 * 2^-23, the
# sum of positive terms over 16 registers and 6 steps by 22 * 2^-24, the quotient by 2^-23.
WEIGHT = 64 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 6), (3, 65, 8), (17, 100, 4), (513, 128, 8),
                                   (2049, 7, 7), (300, 256, 2), (70, 1000, 33), (64, 1024, 64),
                                   (5000, 16, 1)])
@pytest.mark.parametrize("over", ["chosen", "all"])
def test_route(S, T, E, k, over):
    for n, (name, masked) in enumerate([("f32", 0.0), ("f16", 0.3), ("bf16", 0.05)]):
        logits = _logits(T, E, R.TYPES[name], T + E + n, masked, ties=n == 1)
        r = S.route(logits.cuda(), k, over=over)
        want = R.route(logits.double().numpy(), k, over)
        _check_order(r, want)
        assert np.abs(r.weights.cpu().numpy() - want[1]).max() <= WEIGHT
        assert r.over == over


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(1, 16, 16), (3, 129, 1), (66, 200, 9), (130, 255, 16),
                                   (4, 256, 16), (5, 256, 17), (1025, 65, 5), (7, 257, 3)])
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_route_16_bit(S, T, E, k, over, name):
    """Around the widths and choices where 16-bit logits are taken four tokens a wave."""
    for n, (masked, ties) in enumerate([(0.0, False), (0.5, False), (0.02, True)]):
        logits = _logits(T, E, R.TYPES[name], T * E + n, masked, ties)
        r = S.route(logits.cuda(), k, over=over)
        want = R.route(logits.double().numpy(), k, over)
        _check_order(r, want)
        assert np.abs(r.weights.cpu().numpy() - want[1]).max() <= WEIGHT


@pytest.mark.gpu
def test_route_masks_ties_and_nan_16_bit(S):
    inf, nan = float("inf"), float("nan")
    rows = [[-inf] * 5, [1, 1, 1, 1, 1], [-0.0, 0.0, -0.0, 0.0, -1.0], [nan, 1, 2, nan, 3],
            [1, nan, -inf, inf, 0], [-inf, -inf, -inf, -inf, 5], [0.0, -0.0, -inf, -0.0, 0.0]]
    for dtype in (torch.float16, torch.bfloat16):
        low = torch.finfo(dtype).min
        logits = torch.tensor(rows + [[low] * 5, [low, -inf, low, -inf, -inf]]).to(dtype)
        for over in ("chosen", "all"):
            r = S.route(logits.cuda(), 3, over=over)
            want = R.route(logits.double().numpy(), 3, over)
            _check_order(r, want)
            got = r.weights.cpu().numpy()
            assert np.array_equal(np.isnan(got), np.isnan(want[1]))
            fine = ~np.isnan(got)
            assert np.abs(got[fine] - want[1][fine]).max() <= WEIGHT


@pytest.mark.gpu
def test_route_masks_ties_and_nan(S):
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    rows = [[-inf] * 5, [low] * 5, [low, -inf, low, -inf, -inf], [1, 1, 1, 1, 1],
            [-0.0, 0.0, -0.0, 0.0, -1.0], [nan, 1, 2, nan, 3], [1, nan, -inf, inf, 0],
            [3, 2, 1, 0, -1], [-inf, -inf, -inf, -inf, 5]]
    logits = torch.tensor(rows, dtype=torch.float32)
    for over in ("chosen", "all"):
        r = S.route(logits.cuda(), 3, over=over)
        want = R.route(logits.double().numpy(), 3, over)
        _check_order(r, want)
        got = r.weights.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want[1]))
        fine = ~np.isnan(got)
        assert np.abs(got[fine] - want[1][fine]).max() <= WEIGHT
        assert np.array_equal(got[0], [0, 0, 0])


@pytest.mark.gpu
def test_route_of_no_tokens(S):
    r = S.route(torch.empty((0, 8), device="cuda"), 2)
    assert r.experts.shape == (0, 2) and r.entries.shape == (0,)
    assert r.offsets.cpu().tolist() == [0] * 9
    assert S.route_backward(torch.empty((0, 8), device="cuda"), r, r.weights).shape == (0, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("n,groups", [(0, 3), (1, 1), (63, 2), (64, 64), (513, 5), (4097, 200),
                                      (70001, 1024), (200000, 3)])
def test_group_entries(S, n, groups):
    g = np.random.default_rng(n)
    ids = g.integers(-2, groups + 2, n).astype(np.int32)  # some outside
    ids[: n // 3] = groups - 1                             # one group with many
    offsets, entries, slots = S.group_entries(torch.from_numpy(ids).cuda(), groups)
    want = R.group(ids, groups, ids.shape)
    for got, w in zip((offsets, entries, slots), want):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 6), (37, 100, 4), (513, 128, 8), (9, 1000, 64)])
@pytest.mark.parametrize("over", ["chosen", "all"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_route_backward(S, T, E, k, over, name):
    logits = _logits(T, E, R.TYPES[name], T * E, 0.1)
    r = S.route(logits.cuda(), k, over=over)
    dw = torch.from_numpy(np.random.default_rng(T).standard_normal((T, k))).float()
    d = S.route_backward(logits.cuda(), r, dw.cuda())
    assert d.dtype == logits.dtype
    experts, weights = r.experts.cpu().numpy(), r.weights.double().cpu().numpy()
    want = R.route_grad(logits.double().numpy(), experts, weights, dw.double().numpy(), over)
    # p (64 roundings of 2^-24) times a difference of dw and a sum of up to 64 products
    scale = np.abs(dw.numpy()).max(1, keepdims=True) * np.ones((1, E)) * 2
    R.within(d, want, scale, 64 + 64 + 8)


def test_route_gradient_formula_against_differences():
    """The 64-bit formula that the kernel is held to, against differences of the weights."""
    g = np.random.default_rng(5)
    logits = g.uniform(-2.0, 2.0, (4, 9))
    logits[1, 3:] = -np.inf
    dw = g.standard_normal((4, 4))
    for over in ("chosen", "all"):
        experts, weights = R.route(logits, 4, over)[:2]
        want = R.route_grad(logits, experts, weights, dw, over)
        for t in range(4):
            for e in range(9):
                if logits[t, e] == -np.inf:
                    assert want[t, e] == 0
                    continue
                h = 1e-6  # below the gaps between these logits: the choices stay
                both = []
                for s in (h, -h):
                    x = logits.copy()
                    x[t, e] += s
                    again, w = R.route(x, 4, over)[:2]
                    assert np.array_equal(again, experts)
                    both.append((w * dw).sum())
                # truncation h^2, cancellation 2^-53 / h
                assert abs((both[0] - both[1]) / (2 * h) - want[t, e]) < 1e-8


@pytest.mark.gpu
def test_route_is_deterministic_and_follows_its_stream(S):
    logits = _logits(3000, 60, torch.float32, 1).cuda()
    first = S.route(logits, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = [S.route(logits, 4, stream=side) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for r in other:
        for f in ("experts", "weights", "offsets", "entries", "slots"):
            assert torch.equal(getattr(r, f), getattr(first, f)), f


@pytest.mark.gpu
def test_route_refusals(S):
    x = torch.zeros((4, 8), device="cuda")
    r = S.route(x, 2)
    for bad in (lambda: S.route(x.cpu(), 2), lambda: S.route(x.double(), 2),
                lambda: S.route(x[:, ::2], 2), lambda: S.route(x[0], 2), lambda: S.route(x, 0),
                lambda: S.route(x, 9), lambda: S.route(x, 2, over="none"),
                lambda: S.route(np.zeros((4, 8)), 2),
                lambda: S.route_backward(x, r, r.weights[:3]),
                lambda: S.route_backward(x, r, r.weights.half()),
                lambda: S.route_backward(x[:3], r, r.weights),
                lambda: S.group_entries(x, 3), lambda: S.group_entries(r.experts, 0),
                lambda: S.group_entries([1, 2], 3)):
        with pytest.raises(S.SpmmError) as e:
            bad()
        assert e.value.code == S.SPMM_INVALID
    for bad in (lambda: S.route(torch.zeros((2, 1025), device="cuda"), 2),
                lambda: S.route(torch.zeros((2, 100), device="cuda"), 65),
                lambda: S.group_entries(r.experts, 1025)):
        with pytest.raises(S.SpmmError) as e:
            bad()
        assert e.value.code == S.SPMM_UNSUPPORTED


def test_c_entry_refuses_bad_arguments(S):
    L = S.lib()
    assert L.spmm_c_route(None, 0, 4, 8, 2, 0, None, None, None, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_route(None, 9, 4, 8, 2, 0, None, None, None, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_route(None, 0, 4, 8, 2, 7, None, None, None, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_route(None, 0, -1, 8, 2, 0, None, None, None, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_group_entries(None, 5, 3, None, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_dispatch(None, 0, 4, 2, 8, None, None, 4, None, None) == S.SPMM_INVALID
    assert L.spmm_c_combine(None, 3, 4, 2, 8, None, None, None, None) == S.SPMM_INVALID
    assert L.spmm_c_combine_backward(None, None, 0, 4, 0, 8, None, None, None, 4, None, None,
                                     None) == S.SPMM_INVALID
    assert L.spmm_c_route_workspace(0, 8, 2) == 0 and L.spmm_c_route_workspace(100, 8, 2) > 0
