"""Grouped products, their gradients and adapters against 64-bit plain forms."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = np.random.default_rng(seed)
    return torch.from_numpy(g.standard_normal(shape) * scale).to(dtype)


def _np(t):
    return t.double().cpu().numpy()


def _offsets(counts, S):
    o = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    assert o[-1] <= S
    return o


# counts of the groups' rows, rows in all, N, K
SHAPES = [
    ([1], 1, 1, 1), ([1], 1, 64, 64), ([0, 1, 0], 1, 17, 33), ([3, 0, 5], 8, 128, 64),
    ([3, 0, 5], 11, 100, 72), ([130, 1, 0, 127], 258, 130, 200), ([129], 200, 257, 129),
    ([0, 0], 5, 40, 24), ([7] * 70, 490, 33, 65), ([64, 65, 63], 192, 256, 264),
    ([300, 20, 513], 833, 384, 512), ([16, 17, 32, 33, 48], 146, 1000, 1024),
    ([600], 600, 520, 1032),
]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,S_,N,K", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("w_in_rows", [False, True])
def test_grouped_mm_and_gradients(S, counts, S_, N, K, name, w_in_rows):
    dtype, G = R.TYPES[name], len(counts)
    o = _offsets(counts, S_)
    offsets = torch.from_numpy(o).cuda()
    x, dy = _values((S_, K), dtype, 1), _values((S_, N), dtype, 2)
    w = _values((G, K, N) if w_in_rows else (G, N, K), dtype, 3, K ** -0.5)
    y = S.grouped_mm(x.cuda(), w.cuda(), offsets, w_in_rows=w_in_rows)
    dx, dw = S.grouped_mm_backward(dy.cuda(), x.cuda(), w.cuda(), offsets, w_in_rows=w_in_rows)
    X, DY, W = _np(x), _np(dy), _np(w)
    if not w_in_rows:
        W = W.transpose(0, 2, 1)
    want = [np.zeros((S_, N)), np.zeros((S_, K)), np.zeros((G, K, N))]
    size = [np.zeros_like(v) for v in want]
    for g in range(G):
        s = slice(o[g], o[g + 1])
        want[0][s], size[0][s] = X[s] @ W[g], abs(X[s]) @ abs(W[g])
        want[1][s], size[1][s] = DY[s] @ W[g].T, abs(DY[s]) @ abs(W[g]).T
        want[2][g], size[2][g] = X[s].T @ DY[s], abs(X[s]).T @ abs(DY[s])
    if not w_in_rows:
        want[2], size[2] = want[2].transpose(0, 2, 1), size[2].transpose(0, 2, 1)
    # products of 16-bit values are exact in fp32; a sum of n terms has at most n roundings
    R.within(y, want[0], size[0], K)
    R.within(dx, want[1], size[1], N)
    R.within(dw, want[2], size[2], max(max(counts), 1))


@pytest.mark.gpu
def test_rows_of_other_groups_do_not_matter(S):
    """Infinities and NaN in a group's rows and weights stay in that group, and what lies
    behind the last group is not read."""
    counts = [5, 40, 3]
    offsets = torch.from_numpy(_offsets(counts, 60)).cuda()
    for K, N in ((64, 96), (65, 97)):
        for w_in_rows in (False, True):
            x = _values((60, K), torch.bfloat16, 1).cuda()
            w = _values((3, K, N) if w_in_rows else (3, N, K), torch.bfloat16, 2).cuda()
            dy = _values((60, N), torch.bfloat16, 3).cuda()
            y = S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows)
            dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
            for t in (x, dy):
                t[5:45] = float("nan")
                t[48:] = float("inf")
            w[1] = float("inf")
            y2 = S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows)
            dx2, dw2 = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
            for a, b in ((y, y2), (dx, dx2)):
                assert torch.equal(a[:5], b[:5]) and torch.equal(a[45:48], b[45:48])
                assert (b[48:] == 0).all()
            assert torch.equal(dw[0], dw2[0]) and torch.equal(dw[2], dw2[2])
            assert not torch.isfinite(y2[5:45]).any()


@pytest.mark.gpu
def test_offsets_out_of_order_stay_in_bounds(S):
    """Offsets that are no partition give some result, from the operands and nothing else."""
    x = _values((40, 64), torch.float16, 1).cuda()
    w = _values((4, 32, 64), torch.float16, 2).cuda()
    for bad in ([0, 50, 20, 90, 1000], [-5, 10, 5, -100, 40], [40, 30, 20, 10, 0]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        y = S.grouped_mm(x, w, offsets)
        dx, dw = S.grouped_mm_backward(y, x, w, offsets)
        torch.cuda.synchronize()
        assert y.shape == (40, 32) and dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.gpu
def test_grouped_gradient_against_differences(S):
    """The products are linear in x and in w: whole steps along small integers are exact."""
    g = np.random.default_rng(0)
    ints = lambda *s: torch.from_numpy(g.integers(-2, 3, s)).half().cuda()  # noqa: E731
    offsets = torch.tensor([0, 9, 9, 30], dtype=torch.int32, device="cuda")
    for w_in_rows in (False, True):
        x, w, dy = ints(30, 24), ints(3, 24, 20) if w_in_rows else ints(3, 20, 24), ints(30, 20)
        hx, hw = ints(30, 24), ints(*w.shape)
        dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
        loss = lambda a, b: (S.grouped_mm(a, b, offsets, w_in_rows=w_in_rows).double()  # noqa: E731
                             * dy.double()).sum().item()
        base = loss(x, w)
        assert loss(x + hx, w) - base == (dx.double() * hx.double()).sum().item()
        assert loss(x, w + hw) - base == (dw.double() * hw.double()).sum().item()


@pytest.mark.gpu
def test_grouped_no_rows_streams_and_unaligned(S):
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    x, w = torch.empty((0, 8), dtype=torch.half, device="cuda"), _values((2, 4, 8), torch.half, 1).cuda()
    assert S.grouped_mm(x, w, offsets).shape == (0, 4)
    dx, dw = S.grouped_mm_backward(torch.empty((0, 4), dtype=torch.half, device="cuda"), x, w, offsets)
    assert dx.shape == (0, 8) and (dw == 0).all()
    # operands that are only aligned for their elements, another stream, an output given
    K, N, S_ = 64, 128, 50
    offsets = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    x0, w0 = _values((S_, K), torch.half, 2).cuda(), _values((2, N, K), torch.half, 3).cuda()
    want = S.grouped_mm(x0, w0, offsets)
    x1 = torch.empty(S_ * K + 1, dtype=torch.half, device="cuda")[1:].view(S_, K).copy_(x0)
    w1 = torch.empty(2 * N * K + 3, dtype=torch.half, device="cuda")[3:].view(2, N, K).copy_(w0)
    out = torch.empty(S_ * N + 1, dtype=torch.half, device="cuda")[1:].view(S_, N)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert S.grouped_mm(x1, w1, offsets, out=out, stream=side) is out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


# ids outside [0, L) have no adapter
ADAPTERS = [(1, 1, 1, 1, 1), (1, 64, 64, 3, 16), (48, 256, 512, 48, 16), (33, 130, 129, 5, 12),
            (200, 96, 72, 2, 64), (17, 40, 1000, 4, 8), (700, 300, 264, 7, 40), (65, 128, 4096, 3, 4),
            (5, 33, 8, 0, 8), (20, 64, 64, 6, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,L,rank", ADAPTERS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["mixed", "packed", "none"])
def test_adapter_mm(S, T, N, K, L, rank, name, order):
    dtype = R.TYPES[name]
    g = np.random.default_rng(T + K)
    ids = g.integers(-1, L + 1, T).astype(np.int32)
    if order == "packed":
        ids = np.sort(ids)
    if order == "none":
        ids[:] = -7
    x, w = _values((T, K), dtype, 1), _values((N, K), dtype, 2, K ** -0.5)
    a, b = _values((L, rank, K), dtype, 3, K ** -0.5), _values((L, N, rank), dtype, 4, rank ** -0.5)
    scale = torch.from_numpy(g.uniform(0.5, 2.0, L)).float()
    dev = [t.cuda() for t in (x, w, a, b)] + [torch.from_numpy(ids).cuda()]
    y = S.adapter_mm(*dev, scale.cuda())
    one = S.adapter_mm(*dev)
    X, W, A, B = (_np(t) for t in (x, w, a, b))
    base, size = X @ W.T, abs(X) @ abs(W).T
    for got, f in ((y, scale.double().numpy()), (one, np.ones(L))):
        want, bound = base.copy(), size.copy()
        low = np.zeros_like(base)
        for i in range(L):
            t = ids == i
            h = f[i] * (X[t] @ A[i].T)
            want[t] += h @ B[i].T
            # h: K roundings of its sum and one to the operands' type
            low[t] = (R.ROUNDOFF[dtype] * abs(h) + (K + 1) * 2.0 ** -24 * f[i]
                      * (abs(X[t]) @ abs(A[i]).T)) @ abs(B[i]).T
            bound[t] += abs(h) @ abs(B[i]).T
        # the terms' own roundings beside those of h: K + rank sums, then the result's type
        off = np.abs(_np(got) - want)
        u = R.ROUNDOFF[dtype]
        allowed = u * np.abs(want) + (1 + u) * ((K + rank) * 2.0 ** -24 * bound + low * (1 + u)) \
            + R.TINY[dtype]
        assert (off <= allowed).all(), float((off / allowed).max())


@pytest.mark.gpu
def test_adapters_of_other_rows_do_not_matter(S):
    T, N, K, L, rank = 40, 64, 96, 4, 16
    x, w = _values((T, K), torch.bfloat16, 1).cuda(), _values((N, K), torch.bfloat16, 2).cuda()
    a, b = _values((L, rank, K), torch.bfloat16, 3).cuda(), _values((L, N, rank), torch.bfloat16, 4).cuda()
    ids = torch.arange(T, device="cuda", dtype=torch.int32) % 5 - 1
    y = S.adapter_mm(x, w, a, b, ids)
    a[2] = float("nan")
    b[2] = float("inf")
    x[1] = float("nan")  # id 0
    again = S.adapter_mm(x, w, a, b, ids)
    bad = (ids == 2)
    assert not torch.isfinite(again[bad]).any() and torch.isnan(again[1]).all()
    bad[1] = True
    assert torch.equal(again[~bad], y[~bad])


@pytest.mark.gpu
def test_refusals(S):
    h = lambda *s: torch.zeros(s, dtype=torch.half, device="cuda")  # noqa: E731
    x, w = h(6, 8), h(2, 4, 8)
    offsets = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    a, b = h(3, 2, 8), h(3, 4, 2)
    for bad in (lambda: S.grouped_mm(x, w, offsets[:2]), lambda: S.grouped_mm(x, w, offsets.long()),
                lambda: S.grouped_mm(x, w, offsets, w_in_rows=True),
                lambda: S.grouped_mm(x, w.bfloat16(), offsets), lambda: S.grouped_mm(x.t(), w, offsets),
                lambda: S.grouped_mm(x.cpu(), w, offsets), lambda: S.grouped_mm(x, w[0], offsets),
                lambda: S.grouped_mm(x, w, offsets, out=h(6, 5)),
                lambda: S.grouped_mm_backward(h(5, 4), x, w, offsets),
                lambda: S.grouped_mm(x.double(), w, offsets),
                lambda: S.adapter_mm(x, w[0], a, b, ids[:5]),
                lambda: S.adapter_mm(x, w[0], a, b[:2], ids),
                lambda: S.adapter_mm(x, w[0], a[:, :, :7], b, ids),
                lambda: S.adapter_mm(x, w[0], a, b, ids.long()),
                lambda: S.adapter_mm(x, w[0], a, b, ids, h(3)),
                lambda: S.adapter_mm(x, w[0], a[:, :0].contiguous(), b[:, :, :0].contiguous(), ids)):
        with pytest.raises(S.SpmmError) as e:
            bad()
        assert e.value.code == S.SPMM_INVALID
    with pytest.raises(S.SpmmError) as e:
        S.grouped_mm(x.float(), w.float(), offsets)
    assert e.value.code == S.SPMM_UNSUPPORTED


def test_c_entries_refuse_bad_arguments(S):
    L = S.lib()
    assert L.spmm_c_grouped_mm(None, None, 1, None, 2, 4, 8, 8, 0, None, None) == S.SPMM_INVALID
    assert L.spmm_c_grouped_mm(None, None, 1, None, 0, 4, 8, 8, 0, None, None) == S.SPMM_INVALID
    assert L.spmm_c_grouped_mm(None, None, 5, None, 2, 4, 8, 8, 0, None, None) == S.SPMM_INVALID
    assert L.spmm_c_grouped_mm(None, None, 1, None, 2, 4, 8, 1 << 23, 0, None,
                               None) == S.SPMM_UNSUPPORTED
    assert L.spmm_c_grouped_outer(None, None, 2, None, 2, 0, 8, 8, None, None) == S.SPMM_INVALID
    assert L.spmm_c_adapter_mm(None, None, None, None, None, None, 1, 4, 8, 8, 1, 0, None, None,
                               None) == S.SPMM_INVALID
    assert L.spmm_c_adapter_mm(None, None, None, None, None, None, 1, 4, 8, 8, 1, 2000, None, None,
                               None) == S.SPMM_UNSUPPORTED
    assert L.spmm_c_adapter_workspace(4, 12) == 4 * 32 * 2
