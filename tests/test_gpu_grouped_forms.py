"""Grouped products and adapters at sizes that take each of their kernels: tiles of 256
x 256, 128 x 128 and 64 x 64, few rows with sixteen and with 64 columns, operands that are no whole
pieces; and groups that do not begin at row zero.  Compared in 64 bits on the GPU."""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _check(got, want, size, roundings):
    R.within(got, want.cpu().numpy(), size.cpu().numpy(), roundings)


def _bounds(counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return o, torch.tensor(o, dtype=torch.int32, device="cuda")


# counts of the groups' rows, rows in all, N, K
FORMS = [
    ([2500, 4400], 7000, 2040, 1032),  # 256 x 256, edges part-filled, rows in no group
    ([4090], 4090, 4088, 520),         # 256 x 256 in all three products
    ([712], 712, 4088, 4088),          # 128 x 128; the weights' gradient 256 x 256
    ([900, 0, 1, 700], 1601, 1000, 776),
    ([32] * 64, 2048, 512, 4096),      # few rows, 64 columns a workgroup
    ([31, 1, 0, 64] * 16, 1540, 520, 4096),
    ([4] * 60, 256, 72, 520),          # few rows, several workgroups a CU
    ([20] * 12, 240, 264, 1032),
    ([70, 90], 160, 700, 2056),        # few rows, one workgroup a CU
    ([2500, 1400], 4000, 1001, 519),   # no whole pieces
    ([3] * 20, 64, 301, 1027),
    ([600], 600, 1024, 4096),      # 64 x 64 tiles whose waves share the contraction
    ([300, 1, 0, 20], 333, 200, 5121), ([3999], 4000, 130, 190), ([3000, 900], 3907, 129, 65),
    ([12], 12, 1500, 2057), ([20], 20, 1500, 2057), ([40], 40, 1500, 2057), ([60], 60, 1500, 2057),
]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", FORMS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("w_in_rows", [False, True])
def test_grouped_forms(S, counts, rows, N, K, name, w_in_rows):
    dtype, G = R.TYPES[name], len(counts)
    o, offsets = _bounds(counts)
    x, dy = _values((rows, K), dtype, 1), _values((rows, N), dtype, 2)
    w = _values((G, K, N) if w_in_rows else (G, N, K), dtype, 3, K ** -0.5)
    y = S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows)
    dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
    assert (y[o[-1]:] == 0).all() and (dx[o[-1]:] == 0).all()
    for g in range(G):
        s = slice(o[g], o[g + 1])
        X, DY, W = x[s].double(), dy[s].double(), w[g].double()
        if not w_in_rows:
            W = W.t().contiguous()
        # products of 16-bit values are exact in fp32; a sum of n terms has at most n roundings
        _check(y[s], X @ W, X.abs() @ W.abs(), K)
        _check(dx[s], DY @ W.t(), DY.abs() @ W.abs().t(), N)
        d, m = X.t() @ DY, X.abs().t() @ DY.abs()
        if not w_in_rows:
            d, m = d.t(), m.t()
        _check(dw[g], d, m, max(o[g + 1] - o[g], 1))


@pytest.mark.gpu
@pytest.mark.parametrize("first", [1, 7, 130, 300])
@pytest.mark.parametrize("groups", [1, 3, 62, 63, 64])
@pytest.mark.parametrize("K", [64, 65])
def test_groups_of_a_slice(S, first, groups, K):
    """The experts of one rank: rows before the first group and behind the last are zero,
    and their values do not matter."""
    N, counts = 72, [(5 * g) % 9 for g in range(groups)]
    o, offsets = _bounds(counts, first)
    rows = o[-1] + 40
    x, dy = _values((rows, K), torch.bfloat16, 1), _values((rows, N), torch.bfloat16, 2)
    x[:first] = float("nan")
    dy[o[-1]:] = float("inf")
    for w_in_rows in (False, True):
        w = _values((groups, K, N) if w_in_rows else (groups, N, K), torch.bfloat16, 3)
        out = torch.full((rows, N), 7.0, dtype=torch.bfloat16, device="cuda")
        y = S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows, out=out)
        dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
        for t in (y, dx):
            assert (t[:first] == 0).all() and (t[o[-1]:] == 0).all()
        inner = slice(first, o[-1])
        again = torch.tensor([v - first for v in o], dtype=torch.int32, device="cuda")
        want = [S.grouped_mm(x[inner], w, again, w_in_rows=w_in_rows)]
        want += S.grouped_mm_backward(dy[inner], x[inner], w, again, w_in_rows=w_in_rows)
        for a, b in zip((y[inner], dx[inner], dw), want):
            if b.numel() == 0:
                continue
            X = b.double()
            # the same terms in whichever order: each within its own rounding of the sum
            assert torch.allclose(a.double(), X, rtol=2.0 ** -7, atol=(max(K, N, rows) * 2.0 ** -22)
                                  * float(1 + X.abs().max()))


# rows, N, K, adapters, rank
ADAPTERS = [
    (4090, 4088, 1032, 3, 24),   # 256 x 256 tiles
    (1500, 1000, 520, 4, 16),    # 128 x 128 tiles
    (1500, 1000, 520, 4, 12),    # ranks that are no whole pieces
    (1500, 1000, 521, 4, 16),
    (128, 6144, 4096, 5, 16),    # few rows, 64 columns a workgroup
    (513, 264, 776, 20, 33),     # more adapters than workgroups share a row tile
    (512, 264, 776, 20, 33),
    (40, 520, 2056, 30, 8),
    (823, 200, 6787, 7, 12),     # 64 x 64 tiles
    (300, 256, 4096, 3, 48),
    (12, 1500, 2057, 3, 24), (20, 1500, 2057, 3, 9), (40, 1500, 2057, 3, 24), (60, 1500, 2057, 3, 24),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,L,rank", ADAPTERS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["mixed", "packed"])
def test_adapter_forms(S, T, N, K, L, rank, name, order):
    dtype, u = R.TYPES[name], R.ROUNDOFF[R.TYPES[name]]
    ids = torch.randint(-1, L + 1, (T,), dtype=torch.int32, device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(T))
    if order == "packed":
        ids = ids.sort().values
    x, w = _values((T, K), dtype, 1), _values((N, K), dtype, 2, K ** -0.5)
    a, b = _values((L, rank, K), dtype, 3, K ** -0.5), _values((L, N, rank), dtype, 4, rank ** -0.5)
    scale = torch.linspace(0.5, 2.0, L, device="cuda")
    y = S.adapter_mm(x, w, a, b, ids, scale)
    X, W = x.double(), w.double()
    want, size = X @ W.t(), X.abs() @ W.abs().t()
    low = torch.zeros_like(want)
    for i in range(L):
        t = (ids == i).nonzero()[:, 0]
        A, B, f = a[i].double(), b[i].double(), float(scale[i])
        h = f * (X[t] @ A.t())
        want[t] += h @ B.t()
        size[t] += h.abs() @ B.abs().t()
        # h: K roundings of its sum and one to the operands' type
        low[t] = (u * h.abs() + (K + 1) * 2.0 ** -24 * f * (X[t].abs() @ A.abs().t())) @ B.abs().t()
    off = (y.double() - want).abs()
    # the terms' own roundings beside those of h: K + rank sums, then the result's type
    allowed = u * want.abs() + (1 + u) * ((K + rank) * 2.0 ** -24 * size + low * (1 + u)) \
        + R.TINY[dtype]
    assert (off <= allowed).all(), float((off / allowed).max())


@pytest.mark.gpu
def test_more_than_32_bits_of_elements(S):
    """Weights and their gradient of more than 2^31 elements, each way round."""
    G, N, K, each = 64, 8192, 4224, 3
    o, offsets = _bounds([each] * G)
    x, dy = _values((o[-1], K), torch.bfloat16, 1), _values((o[-1], N), torch.bfloat16, 2)
    w = torch.zeros((G, N, K), dtype=torch.bfloat16, device="cuda")
    for g in (0, G - 2, G - 1):
        w[g] = _values((N, K), torch.bfloat16, 3 + g, K ** -0.5)
    y = S.grouped_mm(x, w, offsets)
    dx, dw = S.grouped_mm_backward(dy, x, w, offsets)
    z = S.grouped_mm(dy, w, offsets, w_in_rows=True)
    assert torch.equal(z, dx)
    for g in (0, 5, G - 2, G - 1):
        s = slice(o[g], o[g + 1])
        X, DY, W = x[s].double(), dy[s].double(), w[g].double()
        _check(y[s], X @ W.t(), X.abs() @ W.abs().t(), K)
        _check(dx[s], DY @ W, DY.abs() @ W.abs(), N)
        _check(dw[g], DY.t() @ X, DY.abs().t() @ X.abs(), each)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 200])
def test_adapters_of_many_columns(S, T):
    """An adapter's second matrix of more than 2^31 bytes."""
    N, K, rank = 2100000, 8, 520
    dtype, u = torch.bfloat16, R.ROUNDOFF[torch.bfloat16]
    x, w = _values((T, K), dtype, 1), _values((N, K), dtype, 2, K ** -0.5)
    a = _values((1, rank, K), dtype, 3, K ** -0.5)
    b = torch.zeros((1, N, rank), dtype=dtype, device="cuda")
    b[:, -300:] = _values((1, 300, rank), dtype, 4, rank ** -0.5)
    ids = torch.zeros(T, dtype=torch.int32, device="cuda")
    y = S.adapter_mm(x, w, a, b, ids)
    X, W, A, B = (v.double() for v in (x, w[-400:], a[0], b[0, -400:]))
    h = X @ A.t()
    want = X @ W.t() + h @ B.t()
    size = X.abs() @ W.abs().t() + h.abs() @ B.abs().t()
    low = (u * h.abs() + (K + 1) * 2.0 ** -24 * (X.abs() @ A.abs().t())) @ B.abs().t()
    off = (y[:, -400:].double() - want).abs()
    allowed = u * want.abs() + (1 + u) * ((K + rank) * 2.0 ** -24 * size + low * (1 + u)) \
        + R.TINY[dtype]
    assert (off <= allowed).all(), float((off / allowed).max())
