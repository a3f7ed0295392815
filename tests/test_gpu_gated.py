"""Gated products and their gradients against 64-bit plain forms on the GPU."""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _bounds(counts, first=0):
    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return o, torch.tensor(o, dtype=torch.int32, device="cuda")


# counts of the groups' rows (None: one pair of weights), rows in all, N, K
SHAPES = [
    (None, 1, 1, 1), (None, 1, 64, 64), (None, 3, 7, 33), (None, 16, 1000, 512), (None, 20, 264, 1032),
    (None, 47, 301, 1027), (None, 64, 4096, 512), (None, 70, 6400, 264), (None, 129, 257, 129),
    (None, 300, 520, 4096), (None, 333, 200, 5121), (None, 712, 2044, 1000), (None, 2100, 2040, 1032),
    (None, 3999, 65, 190), (None, 4099, 2052, 520),
    ([0, 1, 0], 1, 17, 33), ([3, 0, 5], 11, 100, 72), ([130, 1, 0, 127], 258, 130, 200),
    ([0, 0], 5, 40, 24), ([7] * 70, 490, 33, 65), ([300, 20, 513], 833, 384, 512),
    ([4] * 60, 256, 72, 520), ([32] * 64, 2048, 256, 2048), ([900, 0, 1, 700], 1601, 1000, 776),
    ([2500, 1400], 4000, 1001, 519), ([2500, 4400], 7000, 1020, 1032),
]


def _case(counts, rows, N, K, dtype):
    first = 0 if counts is None else min(2, rows - sum(counts))
    o, offsets = _bounds([rows] if counts is None else counts, first)
    n = len(o) - 1
    x, w = _values((rows, K), dtype, 1), _values((n, 2, N, K), dtype, 2, K ** -0.5)
    return o, None if counts is None else offsets, x, w


def _exact(o, x, w):
    """g and u in 64 bits [2, rows, N] and the errors of their fp32 sums."""
    rows, K = x.shape
    N = w.shape[2]
    g = torch.zeros((2, rows, N), dtype=torch.float64, device="cuda")
    e = torch.zeros_like(g)
    for i in range(w.shape[0]):
        s = slice(o[i], o[i + 1])
        for j in range(2):
            g[j, s] = x[s].double() @ w[i, j].double().t()
            e[j, s] = K * 2.0 ** -24 * (x[s].double().abs() @ w[i, j].double().abs().t())
    return g, e


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("act", G.ACTS)
def test_gated_mm(S, counts, rows, N, K, name, act):
    o, offsets, x, w = _case(counts, rows, N, K, R.TYPES[name])
    given = w[0] if offsets is None else w
    h = S.gated_mm(x, given, offsets, act=act)
    full, kept = S.gated_mm(x, given, offsets, act=act, keep="full")
    eight, packed = S.gated_mm(x, given, offsets, act=act, keep="8bit")
    (g, u), (eg, eu) = _exact(o, x, w)
    want, bound = G.value(g, act) * u, G.product_bound(g, u, eg, eu, act)
    for got in (h, full, eight):
        G.close(got, want, bound)
        assert (got[:o[0]] == 0).all() and (got[o[-1]:] == 0).all()
    assert kept.shape == (rows, 2, N)
    G.close(kept[:, 0], g, eg)
    G.close(kept[:, 1], u, eu)
    # packed from the fp32 sums: half a step off, a whole one next to a block's largest value
    for j, (v, e) in enumerate(((g, eg), (u, eu))):
        blocks = torch.nn.functional.pad(v.abs() + e, (0, -N % 32)).view(rows, -1, 32)
        largest = blocks.amax(2).clamp(min=2.0 ** -120)
        step = torch.exp2(torch.floor(torch.log2(largest)) - 6).repeat_interleave(32, 1)[:, :N]
        near = v.abs() + e >= 127.5 * step
        got = S.unpack8(S.Packed8(packed.values[:, j].contiguous(),
                                  packed.scales[:, j].contiguous()), torch.float32).double()
        assert ((got - v).abs() <= torch.where(near, step, 0.5 * step) + e).all()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("act", G.ACTS)
@pytest.mark.parametrize("held", ["full", "8bit"])
def test_gradients(S, counts, rows, N, K, name, act, held):
    dtype = R.TYPES[name]
    o, offsets, x, w = _case(counts, rows, N, K, dtype)
    given = w[0] if offsets is None else w
    kept, dh = _values((rows, 2, N), dtype, 3), _values((rows, N), dtype, 4)
    operands = (x, kept)
    if held == "8bit":
        operands = (S.pack8(x), S.pack8(kept))
        x, kept = (S.unpack8(t, dtype) for t in operands)
    dx, dw, h = S.gated_mm_backward(dh, operands[0], given, operands[1], offsets, act=act, hidden=True)
    g, u = kept.double().unbind(1)
    zero = torch.zeros_like(g)
    G.close(h, G.value(g, act) * u, G.product_bound(g, u, zero, zero, act))
    dg, du, eg, eu = G.gradients(dh.double(), g, u, act)
    r = R.ROUNDOFF[dtype]
    # the sums' terms: rounded to the operands' type, as many roundings as terms
    d = torch.cat([dg, du], 1)
    e = torch.cat([eg, eu], 1) * (1 + r) + r * d.abs() + R.TINY[dtype]
    want = [torch.zeros((rows, K), dtype=torch.float64, device="cuda"), torch.zeros_like(w, dtype=torch.float64)]
    bound = [torch.zeros_like(t) for t in want]
    for i in range(w.shape[0]):
        s = slice(o[i], o[i + 1])
        W, X = w[i].double().view(2 * N, K), x[s].double()
        want[0][s] = d[s] @ W
        bound[0][s] = (e[s] + 2 * N * 2.0 ** -24 * (d[s].abs() + e[s])) @ W.abs()
        n = max(o[i + 1] - o[i], 1)
        want[1][i] = (d[s].t() @ X).view(2, N, K)
        bound[1][i] = ((e[s] + n * 2.0 ** -24 * (d[s].abs() + e[s])).t() @ X.abs()).view(2, N, K)
    G.close(dx, want[0], bound[0])
    G.close(dw, want[1][0] if offsets is None else want[1], bound[1][0] if offsets is None else bound[1])
