"""Gated products, their gradients and products in 8-bit integers at sizes that take each of
their kernels: few rows, the ring of 64 and of 128 rows, tiles of 128 x 128 and of 256 x 256
(also in two launches), for rows of whole pieces, of whole words, and between two words."""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _offsets(rows, groups):
    """Rows of groups that begin at row 1, the last but one empty."""
    cuts = [1 + (rows - 3) * i // (groups - 1) for i in range(groups)]
    cuts.insert(groups - 1, cuts[-2])
    cuts = sorted(cuts)
    return cuts, torch.tensor(cuts, dtype=torch.int32, device="cuda")


# rows, N, K, groups (0: one pair of weights)
GATED = [
    (1, 33, 521, 0), (1, 33, 64, 0), (1, 33, 66, 0), (20, 33, 521, 0), (20, 33, 64, 0), (20, 33, 66, 0),
    (50, 33, 521, 0), (50, 33, 64, 0), (50, 33, 66, 0), (40, 700, 1002, 0),
    (1, 33, 65, 0), (20, 2040, 64, 5), (20, 2040, 66, 5),             # ring, 64 rows
    (2000, 520, 521, 0), (2000, 520, 520, 0), (2000, 520, 522, 0),    # 128 rows
    (2000, 520, 575, 0), (2000, 520, 577, 0), (2000, 520, 574, 0), (2000, 520, 576, 0), (2000, 520, 63, 0),
    (20, 4090, 65, 5), (20, 4090, 64, 5), (20, 4090, 66, 5),          # 128 x 128
    (7000, 1000, 520, 0), (7000, 1000, 522, 0), (7000, 1000, 514, 0), (7000, 1000, 574, 0),  # 256 x 256
    (7000, 1000, 62, 0), (6400, 1500, 130, 5), (9000, 1024, 1030, 0), (9000, 1024, 1024, 0),
]


def _projections(x, w, cuts):
    rows, K = x.shape
    g = torch.zeros((2, rows, w.shape[2]), dtype=torch.float64, device="cuda")
    e = torch.zeros_like(g)
    for i in range(w.shape[0]):
        s = slice(cuts[i], cuts[i + 1])
        for j in range(2):
            g[j, s] = x[s].double() @ w[i, j].double().t()
            e[j, s] = K * 2.0 ** -24 * (x[s].double().abs() @ w[i, j].double().abs().t())
    return g, e


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,groups", GATED)
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_gated(S, rows, N, K, groups, name):
    dtype = R.TYPES[name]
    x, w = _values((rows, K), dtype, 1), _values((max(groups, 1), 2, N, K), dtype, 2, K ** -0.5)
    cuts, offsets = _offsets(rows, groups) if groups else ([0, rows], None)
    given = w if groups else w[0]
    (g, u), (eg, eu) = _projections(x, w, cuts)
    want, bound = G.value(g, "silu") * u, G.product_bound(g, u, eg, eu, "silu")
    h = S.gated_mm(x, given, offsets)
    G.close(h, want, bound)
    assert (h[:cuts[0]] == 0).all() and (h[cuts[-1]:] == 0).all()
    full, kept = S.gated_mm(x, given, offsets, keep="full")
    assert torch.equal(full, h)
    G.close(kept[:, 0], g, eg)
    G.close(kept[:, 1], u, eu)
    eight, packed = S.gated_mm(x, given, offsets, keep="8bit")
    G.close(eight, want, bound)
    # values and scales of the projections' own packing, but where a sum's rounding decides
    for j, (v, e) in enumerate(((g, eg), (u, eu))):
        ours = S.Packed8(packed.values[:, j].contiguous(), packed.scales[:, j].contiguous())
        q, scale = G.pack(v.float().cpu().numpy())
        there = torch.from_numpy(G.unpack(q, scale)).cuda()
        step = torch.exp2(torch.from_numpy(scale).cuda().double() - 133).repeat_interleave(32, 1)[:, :N]
        off = (S.unpack8(ours, torch.float32).double() - there).abs()
        # a step further where the sum is, two where its block's scale is another
        assert (off <= 2 * step + e).all() and (off > step / 4).double().mean() < 0.01


# rows, N, K, groups
INTS = [(1, 33, 64, 0), (1, 33, 64, 5), (20, 33, 64, 0), (50, 33, 64, 5), (50, 33, 64, 0), (100, 33, 64, 5),
        (200, 700, 4100, 0), (100, 9000, 200, 2), (4000, 520, 64, 0), (2000, 520, 520, 0), (4000, 520, 520, 0),
        (20, 4090, 64, 5), (20, 2040, 64, 5), (7000, 2040, 1030, 0), (7000, 1000, 1030, 0),
        (6400, 1500, 130, 5), (9000, 2048, 1030, 0), (9000, 1024, 1024, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,groups", INTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_integers(S, rows, N, K, groups, dtype):
    n = max(groups, 1)
    g = torch.Generator(device="cuda").manual_seed(rows)
    values = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int8, device="cuda")  # noqa: E731
    padded = (K + 15) // 16 * 16
    x, w = values(rows, padded), values(n, 2, N, padded)
    x[:, K:], w[..., K:] = 0, 0
    sx = torch.rand(rows, generator=g, device="cuda") * 2.0 ** -9
    sw = torch.rand((n, 2, N), generator=g, device="cuda") * 2.0 ** -5
    cuts, offsets = _offsets(rows, groups) if groups else ([0, rows], None)
    q = S.Rows8(x, sx, K)
    lay = lambda v: (v if groups else v[0]).contiguous()  # noqa: E731
    p, one = S.Rows8(lay(w), lay(sw), K), S.Rows8(lay(w[:, 0]), lay(sw[:, 0]), K)
    f = torch.zeros((2, rows, N), device="cuda")
    for i in range(n):
        s = slice(cuts[i], cuts[i + 1])
        for j in range(2):
            sums = x[s].double() @ w[i, j].double().t()  # exact
            f[j, s] = sums.float() * sw[i, j] * sx[s, None]
    assert torch.equal(S.int8_mm(q, one, offsets, dtype=dtype), f[0].to(dtype))
    h = S.gated_mm(q, p, offsets, act="gelu_tanh", dtype=dtype)
    zero = torch.zeros_like(f[0], dtype=torch.float64)
    G.close(h, G.value(f[0].double(), "gelu_tanh") * f[1].double(),
            G.product_bound(f[0].double(), f[1].double(), zero, zero, "gelu_tanh"))


# rows, N, K: the rows' gradient has K columns from 2 N, the weights' 2 N rows from `rows`
GRADIENTS = [(1000, 1500, 512), (1000, 1500, 514), (1000, 1500, 511), (1000, 1501, 514), (3000, 1024, 520),
             (3000, 1024, 522), (8200, 600, 2048), (8200, 600, 2050), (300, 3000, 130), (9000, 2300, 300),
             (70, 1000, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", GRADIENTS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_gradients(S, rows, N, K, name):
    dtype = R.TYPES[name]
    x, w = _values((rows, K), dtype, 1), _values((2, N, K), dtype, 2, K ** -0.5)
    kept, dh = _values((rows, 2, N), dtype, 3), _values((rows, N), dtype, 4)
    dx, dw = S.gated_mm_backward(dh, x, w, kept, act="gelu")
    g, u = kept.double().unbind(1)
    dg, du, eg, eu = G.gradients(dh.double(), g, u, "gelu")
    r = R.ROUNDOFF[dtype]
    d = torch.cat([dg, du], 1)
    e = torch.cat([eg, eu], 1) * (1 + r) + r * d.abs() + R.TINY[dtype]
    W, X = w.double().view(2 * N, K), x.double()
    G.close(dx, d @ W, (e + 2 * N * 2.0 ** -24 * (d.abs() + e)) @ W.abs())
    G.close(dw.view(2 * N, K), d.t() @ X, (e + rows * 2.0 ** -24 * (d.abs() + e)).t() @ X.abs())
    only, none = S.gated_mm_backward(dh, None, w, kept, act="gelu", weights=False)
    assert none is None and torch.equal(only, dx)
    none, only = S.gated_mm_backward(dh, x, w, kept, act="gelu", rows=False)
    assert none is None and torch.equal(only, dw)
