"""Gradients of gated products in fp16 whose terms dh u act'(g) and dh act(g) lie past fp16's
range, at either end, while the gradients do not.

The kernels hold a row of the terms as fp16 times 2^e (for the weights' gradient, a group's rows
with the largest e among them), so a term is off by a rounding and by half of fp16's least number:
2^-11 of itself and 2^(e - 25); rows whose e is not their group's are rounded twice.
"""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402

HALF = torch.float16
# counts of the groups' rows (None: one pair of weights), rows in all, N, K: each kernel of the
# two products, rows of whole pieces, of words and between words, widths past what a row's
# workgroup holds
SIZES = [(None, 1, 1, 1), (None, 5, 9, 33), (None, 300, 264, 520), (None, 301, 267, 515),
         (None, 40, 2056, 64), (None, 17, 9001, 40), (None, 2, 8200, 24), (None, 300, 3000, 130),
         (None, 3000, 1024, 520), (None, 3000, 1024, 522), (None, 8200, 600, 2048), (None, 8200, 600, 2050),
         (None, 1000, 1501, 514), (None, 9000, 2300, 300), (None, 70, 1000, 1000), (None, 20000, 16, 16),
         (None, 3000, 4500, 2048), (None, 3000, 4500, 2050),
         ([3, 0, 5], 11, 100, 72), ([7] * 70, 493, 33, 65), ([900, 0, 1, 700], 1604, 1000, 776),
         ([2500, 1400], 4000, 1001, 519), ([2500, 4400], 7000, 1020, 1032), ([600, 300], 905, 1001, 1030)]


def _normal(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _exponent(largest):
    """e of rows whose largest magnitude is given."""
    a = torch.frexp(largest).exponent
    return torch.where(a > 15, a - 15, -((15 - a) // 16 * 16)).double().masked_fill(largest == 0, -112.0)


def _close(got, want, bound):
    """G.close, for sums that may pass fp16's largest number, 65504: from half a step above it on,
    65520, they round to an infinity."""
    may, must = want.abs() + bound >= 65520.0, want.abs() - bound >= 65520.0
    assert torch.equal(torch.isinf(got) & torch.isfinite(want) & ~may, torch.zeros_like(may))
    assert (got[torch.isfinite(want) & must].double() == want[torch.isfinite(want) & must].sign() * torch.inf).all()
    beyond = torch.isinf(got) & may & torch.isfinite(want)
    G.close(got.masked_fill(beyond, 0), want.masked_fill(beyond, 0), bound)


def _check(S, dh, x, w, kept, o, offsets, act="silu", operands=None):
    """w [groups, 2, N, K] and o, the groups' first rows."""
    rows, N = dh.shape
    K = x.shape[1]
    dx, dw = S.gated_mm_backward(dh, *(operands or (x, w if offsets is not None else w[0], kept)), offsets,
                                 act=act)
    g, u = kept.double().unbind(1)
    dg, du, eg, eu = G.gradients(dh.double(), g, u, act)
    d, e = torch.cat([dg, du], 1), torch.cat([eg, eu], 1)
    # fp32 errors may move a row's largest value over a power of two, not e by more than one
    top = _exponent((d.abs() + e).nan_to_num(0, 0, 0).amax(1))
    r = R.ROUNDOFF[HALF]
    e = torch.nan_to_num(e) * (1 + r) + r * torch.nan_to_num(d, 0, 0, 0).abs()
    want = [torch.zeros((rows, K), dtype=torch.float64, device="cuda"), torch.zeros_like(w, dtype=torch.float64)]
    bound = [torch.zeros_like(t) for t in want]
    for i in range(w.shape[0]):
        s = slice(o[i], o[i + 1])
        W, X = w[i].double().view(2 * N, K), x[s].double()
        one = e[s] + torch.exp2(top[s, None] - 25)
        want[0][s] = d[s] @ W
        bound[0][s] = (one + 2 * N * 2.0 ** -24 * (torch.nan_to_num(d[s], 0, 0, 0).abs() + one)) @ W.abs()
        n = max(o[i + 1] - o[i], 1)
        if o[i + 1] > o[i]:
            one = e[s] + 2 * torch.exp2(top[s].max() - 25)
        want[1][i] = (d[s].t() @ X).view(2, N, K)
        bound[1][i] = ((one + n * 2.0 ** -24 * (torch.nan_to_num(d[s], 0, 0, 0).abs() + one)).t()
                       @ X.abs()).view(2, N, K)
    _close(dx, want[0], bound[0])
    _close(dw if offsets is not None else dw[None], want[1], bound[1])
    return dx, dw, d


def _operands(counts, rows, N, K, big, w_scale, x_scale, seed=1):
    """dh and u of about `big`, in rows that differ by up to 2^6."""
    first = 0 if counts is None else min(2, rows - sum(counts))
    o = [first]
    for c in [rows] if counts is None else counts:
        o.append(o[-1] + c)
    offsets = None if counts is None else torch.tensor(o, dtype=torch.int32, device="cuda")
    row = 2.0 ** torch.randint(-3, 4, (rows, 1), device="cuda",
                               generator=torch.Generator(device="cuda").manual_seed(seed))
    dh = (_normal((rows, N), seed) * big * row).to(HALF)
    kept = _normal((rows, 2, N), seed + 1)
    kept[:, 1] *= big
    x = (_normal((rows, K), seed + 2) * x_scale).to(HALF)
    w = (_normal((len(o) - 1, 2, N, K), seed + 3) * w_scale).to(HALF)
    return dh, x, w, kept.to(HALF), o, offsets


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", SIZES)
def test_terms_past_the_largest_number(S, counts, rows, N, K):
    """dh u up to 2^25; the sums of 2 N or `rows` of them times 2^-13 and less are fp16 again."""
    dh, x, w, kept, o, offsets = _operands(counts, rows, N, K, 300.0, 2.0 ** -13 / N ** 0.5, 2.0 ** -13 / rows ** 0.5)
    *_, d = _check(S, dh, x, w, kept, o, offsets)
    assert N * rows < 1000 or (d.abs() > 65520).any()


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", SIZES)
def test_terms_below_the_least_number(S, counts, rows, N, K):
    """dh u of about 2^-26 and less, whose sums times 2^10 are fp16's normal numbers."""
    dh, x, w, kept, o, offsets = _operands(counts, rows, N, K, 2.0 ** -13, 2.0 ** 10, 2.0 ** 10)
    dx, dw, _ = _check(S, dh, x, w, kept, o, offsets, "gelu_tanh")
    assert (dx[o[0]:o[-1]] != 0).double().mean() > 0.9 and (rows < 20 or (dw != 0).double().mean() > 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", [(64, 96, 64), (65, 97, 65), (300, 1000, 520), (33, 4100, 72)])
def test_rows_and_groups_of_their_own_range(S, rows, N, K):
    """Rows from 2^-20 to 2^18, a group of the least, of the largest and of all; rows of zeros; rows in
    no group that hold infinities and NaN."""
    o = [1, 1 + rows // 4, 1 + rows // 2, rows - 1]
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    e = torch.randint(-9, 10, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
    e[:o[1]], e[o[1]:o[2]] = -9, 9
    scale = 2.0 ** e[:, None].double()
    dh = (_normal((rows, N), 1) * scale).to(HALF)
    kept = _normal((rows, 2, N), 2)
    kept[:, 1] *= scale
    kept = kept.to(HALF)
    dh[o[2] + 1] = 0
    x, w = (_normal((rows, K), 3) * 2.0 ** -9).to(HALF), (_normal((3, 2, N, K), 4) * 2.0 ** -9).to(HALF)
    dh[0], kept[-1] = float("inf"), float("nan")
    dx, _, _ = _check(S, dh, x, w, kept, o, offsets, "gelu")
    assert (dx[0] == 0).all() and (dx[-1] == 0).all()


@pytest.mark.gpu
def test_infinities_stay_in_their_row(S):
    """An infinity or a NaN among a row's terms: that row of dx and those rows of dW are no numbers,
    the others what they are without."""
    rows, N, K = 40, 72, 64
    dh, x, w, kept, o, offsets = _operands(None, rows, N, K, 300.0, 2.0 ** -13, 2.0 ** -13)
    dh[7, 5], dh[9, 11], dh[12] = float("inf"), float("nan"), float("-inf")
    dh[12, 1:], kept[12, 1, 0] = 0, 1.0
    dx, dw, _ = _check(S, dh, x, w, kept, o, offsets)
    assert not torch.isfinite(dx[[7, 9, 12]]).any() and torch.isfinite(dx[torch.arange(rows) % 20 > 12]).all()
    assert not torch.isfinite(dw[:, [0, 5, 11]]).any() and torch.isfinite(dw[:, 12:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [64, 97, 2100, 9001])
def test_packed_projections_past_the_range(S, N):
    """Projections that 8 bits hold and fp16 does not."""
    rows, K = 50, 40
    dh, x, w, _, o, offsets = _operands(None, rows, N, K, 2.0 ** -6, 2.0 ** -15, 2.0 ** -15)
    wide = _normal((rows, 2, N), 9)
    wide[:, 1] *= 2.0 ** 24
    packed, x8 = S.pack8(wide), S.pack8(x)
    kept, x = S.unpack8(packed, torch.float32), S.unpack8(x8, HALF)
    _check(S, dh, x, w, kept, o, offsets, operands=(x8, w[0], packed))


@pytest.mark.gpu
def test_captured(S):
    """A graph with rows of other scales each time, of two groups."""
    rows, N, K = 70, 200, 136
    o = [0, 30, 70]
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    dh, x, w, kept = (_normal(s, i).to(HALF) for i, s in enumerate([(rows, N), (rows, K), (2, 2, N, K),
                                                                    (rows, 2, N)]))
    w.mul_(2.0 ** -10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.gated_mm_backward(dh, x, w, kept, offsets, hidden=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = S.gated_mm_backward(dh, x, w, kept, offsets, hidden=True)
    for seed in range(4):
        dh.copy_(_normal((rows, N), 10 + seed) * 2.0 ** (5 * seed - 12) * (torch.arange(rows, device="cuda")[:, None] % 3 * 60 + 1))
        graph.replay()
        want = S.gated_mm_backward(dh, x, w, kept, offsets, hidden=True)
        torch.cuda.synchronize()
        for a, b in zip(want, held):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_one_gradient_alone(S):
    dh, x, w, kept, o, offsets = _operands([40, 0, 83], 130, 201, 72, 300.0, 2.0 ** -16, 2.0 ** -16)
    dx, dw = S.gated_mm_backward(dh, x, w, kept, offsets)
    only, none = S.gated_mm_backward(dh, None, w, kept, offsets, weights=False)
    assert none is None and torch.equal(only, dx)
    none, only = S.gated_mm_backward(dh, x, w, kept, offsets, rows=False)
    assert none is None and torch.equal(only, dw)


def test_c_entries_refuse_bad_arguments(S):
    import ctypes
    L, some, top = S.lib(), ctypes.c_void_p(4096), 0x7fffffff  # never read: the calls end before
    bad, not_here = S.SPMM_INVALID, S.SPMM_UNSUPPORTED
    grad = lambda **k: L.spmm_c_gated_grad_scaled(*{**dict(  # noqa: E731
        dh=some, kept=some, scales=None, rows=4, width=8, act=0, dkept=some, row_scales=some, h=None,
        stream=None), **k}.values())
    assert grad(dh=None) == grad(kept=None) == grad(dkept=None) == grad(row_scales=None) == bad
    assert grad(act=3) == grad(act=-1) == grad(rows=-1) == grad(width=0) == bad
    assert grad(width=1 << 23) == not_here
    assert grad(rows=0, dh=None, row_scales=None) == S.SPMM_OK
    back = lambda **k: L.spmm_c_gated_mm_backward_scaled(*{**dict(  # noqa: E731
        dkept=some, row_scales=some, x=some, w=some, offsets=some, groups=2, rows=4, width=8, depth=8,
        dx=some, dw=some, workspace=some, stream=None), **k}.values())
    only = lambda **k: back(dx=None, **k)  # noqa: E731
    assert back(row_scales=None) == back(dkept=None) == back(w=None) == back(offsets=None) == bad
    assert only(workspace=None) == only(dkept=None) == only(x=None) == only(offsets=None) == bad
    for f in (back, only):
        assert f(rows=-1) == f(width=0) == f(groups=0) == f(depth=0) == bad
        assert f(depth=1 << 23) == f(width=top) == f(width=1 << 22) == not_here
        assert f(groups=1 << 24, rows=1 << 24) == not_here
    assert back(dx=None, dw=None, workspace=None) == S.SPMM_OK


@pytest.mark.gpu
def test_more_rows_than_one_launch_takes(S):
    """Rows past 2^22, whose workgroups of a row each are another launch's."""
    rows, N, K, tail = (1 << 22) + 1000, 8, 8, 2000
    o = [0, rows - tail, rows]
    offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
    dh = torch.zeros((rows, N), dtype=HALF, device="cuda")
    kept = torch.zeros((rows, 2, N), dtype=HALF, device="cuda")
    x = torch.zeros((rows, K), dtype=HALF, device="cuda")
    d, x1, w, k1, *_ = _operands(None, tail, N, K, 300.0, 2.0 ** -13, 2.0 ** -15)
    w = torch.cat([w, w])
    dh[-tail:], kept[-tail:], x[-tail:] = d, k1, x1
    dx, dw = S.gated_mm_backward(dh, x, w, kept, offsets)
    only = torch.tensor([0, tail], dtype=torch.int32, device="cuda")
    dx1, dw1, terms = _check(S, d, x1, w[1:].contiguous(), k1, [0, tail], only)
    assert torch.equal(dx[-tail:], dx1) and (dx[:-tail] == 0).all()
    assert (dw[0] == 0).all()
    # the same rounded terms in another order: fp32 sums apart, then a rounding each
    sums = tail * 2.0 ** -24 * (terms.abs().t() @ x1.double().abs()).view(2, N, K) * (1 + 2.0 ** -10)
    assert ((dw[1].double() - dw1[0].double()).abs()
            <= 2 * sums + 2 * R.ROUNDOFF[HALF] * (dw1[0].double().abs() + 2 * sums)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rows,N,K", [(300, 264, 520), (65, 97, 65), (9, 9001, 40)])
def test_the_entries_without_scales(S, rows, N, K, packed):
    """In fp16 too.  dg and du within their bounds (not the same bits as with scales: without, the
    last product is rounded to fp16 at once, with them to fp32 first), and from the same dg and du
    the same bits as with scales of 1."""
    dh, kept = _normal((rows, N), 1).to(HALF), _normal((rows, 2, N), 2).to(HALF)
    dh[:, 0], kept[:, :, 0] = 4.0, 4.0
    x, w = _normal((rows, K), 3).to(HALF), (_normal((2, N, K), 4) * K ** -0.5).to(HALF)
    p = S.pack8(kept)
    held = (p.values.data_ptr(), p.scales.data_ptr()) if packed else (kept.data_ptr(), None)
    dkept, h, dx, dw = (torch.empty_like(t) for t in (kept, dh, x, w))
    L, stream = S.lib(), torch.cuda.current_stream().cuda_stream
    assert L.spmm_c_gated_grad(dh.data_ptr(), 1, *held, rows, N, 0, dkept.data_ptr(), h.data_ptr(),
                               stream) == S.SPMM_OK
    assert L.spmm_c_gated_mm_backward(dkept.data_ptr(), x.data_ptr(), w.data_ptr(), 1, None, 1, rows, N, K,
                                      dx.data_ptr(), dw.data_ptr(), stream) == S.SPMM_OK
    g, u = (S.unpack8(p, HALF) if packed else kept).double().unbind(1)
    dg, du, eg, eu = G.gradients(dh.double(), g, u, "silu")
    G.close(dkept[:, 0], dg, eg)
    G.close(dkept[:, 1], du, eu)
    *_, again = S.gated_mm_backward(dh, x, w, p if packed else kept, hidden=True)
    assert torch.equal(h, again)
    one, dx1, dw1, before = torch.ones(rows + 1, device="cuda"), torch.empty_like(x), torch.empty_like(w), dkept.clone()
    assert L.spmm_c_gated_mm_backward_scaled(
        dkept.data_ptr(), one.data_ptr(), x.data_ptr(), w.data_ptr(), None, 1, rows, N, K, dx1.data_ptr(),
        dw1.data_ptr(), one.data_ptr() + 4 * rows, stream) == S.SPMM_OK
    assert torch.equal(dx1, dx) and torch.equal(dw1, dw) and torch.equal(dkept, before)
