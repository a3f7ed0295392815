"""Gated products, packed activations and 8-bit integers as they may be called: operands at
any address, other streams, captured graphs, groups that hold nothing or infinities, and
what is refused."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _at(t, by):
    """A copy that lies `by` elements into an allocation."""
    return torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)[by:].view(t.shape).copy_(t)


def _int(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", [(9, 40, 64), (200, 72, 128), (300, 1000, 1032), (1400, 2048, 256)])
def test_operands_at_any_address(S, rows, N, K):
    x, w = _values((rows, K), torch.half, 1), _values((2, N, K), torch.half, 2, K ** -0.5)
    dh = _values((rows, N), torch.half, 3)
    h, kept = S.gated_mm(x, w, keep="full")
    _, packed = S.gated_mm(x, w, keep="8bit")
    dx, dw, again = S.gated_mm_backward(dh, x, w, kept, hidden=True)
    x8 = S.pack8(x)
    dx8, dw8, again8 = S.gated_mm_backward(dh, x8, w, packed, hidden=True)
    # every alignment sums the same terms, in an order that tiles or few rows may choose
    (g, u), e = _exact(x, w)
    bound = G.product_bound(g, u, e[0], e[1], "silu")
    for i, j in ((1, 0), (0, 3), (2, 2), (1, 1), (2, 5)):
        out = torch.empty(rows * N + 3, dtype=torch.half, device="cuda")
        x1, w1, dh1 = _at(x, i), _at(w, j), _at(dh, j)
        out = out[j % 3:][:rows * N].view(rows, N)
        got, k1 = S.gated_mm(x1, w1, keep="full", out=out)
        assert got is out
        G.close(got, G.value(g, "silu") * u, bound)
        G.close(k1[:, 0], g, e[0])
        a, b, c = S.gated_mm_backward(dh1, x1, w1, _at(kept, i), hidden=True)
        assert torch.equal(c, again)
        # the sums of the same terms: fp32 roundings apart, then one rounding each
        for p, q in ((a, dx), (b, dw)):
            assert ((p.double() - q.double()).abs() <= 2.0 ** -9 * q.double().abs() + 2.0 ** -9).all()
        p8 = S.Packed8(_at(packed.values, i), _at(packed.scales, j))
        a, b, c = S.gated_mm_backward(dh1, S.Packed8(_at(x8.values, j), _at(x8.scales, i)), w1, p8,
                                      hidden=True)
        assert torch.equal(c, again8)
        for p, q in ((a, dx8), (b, dw8)):
            assert ((p.double() - q.double()).abs() <= 2.0 ** -9 * q.double().abs() + 2.0 ** -9).all()
        t8, r8 = S.pack8(x1), S.quantize_rows(x1)
        assert torch.equal(t8.values, x8.values) and torch.equal(t8.scales, x8.scales)
        r = S.quantize_rows(x)
        assert torch.equal(r8.values, r.values) and torch.equal(r8.scales, r.scales)
        assert torch.equal(S.unpack8(S.Packed8(_at(x8.values, 1), _at(x8.scales, 1)), torch.half,
                                     out=_at(x, 1)), S.unpack8(x8, torch.half))


def _exact(x, w):
    K = x.shape[1]
    g = torch.stack([x.double() @ m.double().t() for m in w])
    return g, torch.stack([K * 2.0 ** -24 * (x.double().abs() @ m.double().abs().t()) for m in w])


@pytest.mark.gpu
@pytest.mark.parametrize("K,N,rows", [(64, 96, 60), (65, 97, 60), (66, 98, 60), (64, 96, 600),
                                      (65, 97, 600), (66, 98, 600), (128, 1024, 3000)])
def test_rows_of_other_groups_do_not_matter(S, K, N, rows):
    """Infinities and NaN in a group's rows and weights stay in that group, and what lies
    behind the last group is not read."""
    cut = [0, rows // 12, rows * 3 // 4, rows * 4 // 5]
    offsets = _int(*cut)
    x, w = _values((rows, K), torch.bfloat16, 1), _values((3, 2, N, K), torch.bfloat16, 2)
    dh = _values((rows, N), torch.bfloat16, 3)
    kept = _values((rows, 2, N), torch.bfloat16, 4)
    first = (S.gated_mm(x, w, offsets), *S.gated_mm_backward(dh, x, w, kept, offsets))
    q, p = S.quantize_rows(x), S.quantize_rows(w)
    ints = S.gated_mm(q, p, offsets), S.int8_mm(q, S.Rows8(p.values[:, 0].contiguous(),
                                                          p.scales[:, 0].contiguous(), K), offsets)
    a, b, c = cut[1], cut[2], cut[3]
    for t in (x, dh, kept, q.scales):
        t[a:b] = float("nan")
        t[c:] = float("inf")
    w[1] = float("inf")
    p.scales[1] = float("nan")
    then = (S.gated_mm(x, w, offsets), *S.gated_mm_backward(dh, x, w, kept, offsets))
    ints2 = S.gated_mm(q, p, offsets), S.int8_mm(q, S.Rows8(p.values[:, 0].contiguous(),
                                                           p.scales[:, 0].contiguous(), K), offsets)
    for one, two in zip((first[0], first[1]) + ints, (then[0], then[1]) + ints2):
        assert torch.equal(one[:a], two[:a]) and torch.equal(one[b:c], two[b:c])
        assert (two[c:] == 0).all() and not torch.isfinite(two[a:b]).any()
    assert torch.equal(first[2][0], then[2][0]) and torch.equal(first[2][2], then[2][2])
    assert not torch.isfinite(then[2][1]).any()


@pytest.mark.gpu
def test_offsets_out_of_order_stay_in_bounds(S):
    """Offsets that are no partition give some result, from the operands and nothing else."""
    x, w = _values((400, 66), torch.half, 1), _values((4, 2, 32, 66), torch.half, 2)
    q, p = S.quantize_rows(x), S.quantize_rows(w)
    for bad in ([0, 500, 200, 900, 1000], [-5, 100, 50, -100, 400], [400, 300, 200, 100, 0]):
        for keep in ("full", "8bit"):
            h, kept = S.gated_mm(x, w, _int(*bad), keep=keep)
            dx, dw = S.gated_mm_backward(h, x, w, kept, _int(*bad))
        y = S.gated_mm(q, p, _int(*bad))
        torch.cuda.synchronize()
        assert h.shape == y.shape == (400, 32) and dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["full", "8bit"])
def test_no_rows(S, keep):
    w = _values((2, 8, 24), torch.half, 1)
    x, h = torch.empty((0, 24), dtype=torch.half, device="cuda"), torch.empty((0, 8), dtype=torch.half,
                                                                              device="cuda")
    for offsets, weights in ((None, w), (_int(0, 0, 0), torch.stack([w, w]))):
        got, kept = S.gated_mm(x, weights, offsets, keep=keep)
        assert got.shape == (0, 8)
        dx, dw, again = S.gated_mm_backward(h, x, weights, kept, offsets, hidden=True)
        assert dx.shape == (0, 24) and (dw == 0).all() and again.shape == (0, 8)
        assert S.gated_mm(x, S.quantize_rows(weights), offsets).shape == (0, 8)
    assert S.unpack8(S.pack8(x)).shape == (0, 24)
    assert S.int8_mm(x, S.quantize_rows(w[0].contiguous())).shape == (0, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("act", G.ACTS)
def test_far_gates(S, act):
    """Gates far out on either side, infinities and NaN: the limits of act(g) and act'(g)."""
    far = [-float("inf"), -3e38, -1e30, -500.0, -90.0, -20.0, -6.0, -0.0, 0.0, 6.0, 20.0, 90.0, 500.0, 1e30,
           float("inf"), float("nan")]
    g = torch.tensor(far, device="cuda").bfloat16()
    n = len(far)
    kept = torch.stack([g, torch.ones_like(g)])[None].contiguous()
    dh = torch.ones((1, n), device="cuda").bfloat16()
    dkept, h = torch.empty_like(kept), torch.empty_like(dh)
    code = S.lib().spmm_c_gated_grad(dh.data_ptr(), 2, kept.data_ptr(), None, 1, n, G.ACTS.index(act),
                                     dkept.data_ptr(), h.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream)
    assert code == S.SPMM_OK
    wide = g.double()
    p, gp, _ = G.share(wide, act)
    value = torch.where(wide == -float("inf"), 0.0, wide * p)
    slope = torch.where(wide.abs() > 200, (wide > 0).double(), p + gp)
    slope = torch.where(torch.isnan(wide), wide, slope)
    # u and dh are 1: dg is act'(g), du and h are act(g)
    for got, want in ((dkept[0, 0], slope), (dkept[0, 1], value), (h[0], value)):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        near = torch.isfinite(want)
        far_off = ~near & ~torch.isnan(want)
        assert torch.equal(got[far_off].double(), want[far_off])
        off = (got[near].double() - want[near]).abs()
        # bf16's rounding and a share off by 2^-12 at the most
        assert (off <= (2.0 ** -8 + 2.0 ** -12) * want[near].abs() + 2.0 ** -100).all()


@pytest.mark.gpu
def test_another_stream(S):
    x, w = _values((300, 264), torch.half, 1), _values((2, 1000, 264), torch.half, 2, 264 ** -0.5)
    dh, p = _values((300, 1000), torch.half, 3), S.quantize_rows(w)
    want = _all(S, x, w, dh, p, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = _all(S, x, w, dh, p, side)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def _all(S, x, w, dh, p, stream):
    h, kept = S.gated_mm(x, w, keep="full", stream=stream)
    _, packed = S.gated_mm(x, w, keep="8bit", stream=stream)
    dx, dw = S.gated_mm_backward(dh, x, w, kept, stream=stream)
    x8 = S.pack8(x, stream=stream)
    dx8, dw8, again = S.gated_mm_backward(dh, x8, w, packed, hidden=True, stream=stream)
    back = S.unpack8(x8, torch.half, stream=stream)
    q = S.quantize_rows(x, stream=stream)
    one = S.Rows8(p.values[0], p.scales[0], p.width)
    return (h, kept, packed.values, packed.scales, dx, dw, dx8, dw8, again, back, q.values, q.scales,
            S.gated_mm(q, p, stream=stream), S.int8_mm(x, one, stream=stream))


@pytest.mark.gpu
def test_captured(S):
    """A graph of all the calls, replayed with other values in between, gives each time what
    the calls give."""
    x, w = _values((70, 130), torch.bfloat16, 1), _values((2, 200, 130), torch.bfloat16, 2, 130 ** -0.5)
    dh = _values((70, 200), torch.bfloat16, 3)
    p = S.quantize_rows(w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _all(S, x, w, dh, p, None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _all(S, x, w, dh, p, None)
    for seed in range(4):
        x.copy_(_values((70, 130), torch.bfloat16, 10 + seed))
        dh.copy_(_values((70, 200), torch.bfloat16, 20 + seed))
        graph.replay()
        want = _all(S, x, w, dh, p, None)
        torch.cuda.synchronize()
        for a, b in zip(want, held):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_same_bits_every_time(S):
    x, w = _values((900, 1032), torch.half, 1), _values((2, 1000, 1032), torch.half, 2, 1032 ** -0.5)
    dh, p = _values((900, 1000), torch.half, 3), S.quantize_rows(w)
    want = _all(S, x, w, dh, p, None)
    for _ in range(5):
        for a, b in zip(want, _all(S, x, w, dh, p, None)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [32, 1000, 4096])
def test_a_cast_of_packed_values(S, width):
    """Packing what was unpacked gives the same back."""
    x = _values((50, width), torch.bfloat16, 1)
    once = S.pack8(x)
    back = S.unpack8(once)
    twice = S.pack8(back)
    assert torch.equal(S.unpack8(twice), back)
    # half a step of 2^-6 of the largest value's power of two, a whole one next to it
    blocks = torch.nn.functional.pad(x.double(), (0, -width % 32)).view(50, -1, 32)
    step = torch.exp2(torch.floor(torch.log2(blocks.abs().amax(2).clamp(min=1e-30))) - 6)
    step = step.repeat_interleave(32, 1)[:, :width]
    near = x.double().abs() >= 127.5 * step
    assert ((back.double() - x.double()).abs() <= torch.where(near, step, step / 2)).all()


@pytest.mark.gpu
def test_refusals(S):
    h = lambda *s: torch.zeros(s, dtype=torch.half, device="cuda")  # noqa: E731
    x, w, pair = h(6, 8), h(2, 4, 8), h(3, 2, 4, 8)
    offsets = _int(0, 3, 4, 6)
    kept, dh = h(6, 2, 4), h(6, 4)
    p8 = S.pack8(kept)
    q, qw, qp = S.quantize_rows(x), S.quantize_rows(w[0]), S.quantize_rows(pair)
    byte = torch.empty(6 * 16 + 1, dtype=torch.int8, device="cuda")[1:].view(6, 16)
    bad = [lambda: S.gated_mm(x, w, act="relu"), lambda: S.gated_mm(x, w, act=["silu"]),
           lambda: S.gated_mm(x, w, keep="4bit"),
           lambda: S.gated_mm(x, w[0]), lambda: S.gated_mm(x, pair), lambda: S.gated_mm(x, w, offsets),
           lambda: S.gated_mm(x, pair, offsets[:2]), lambda: S.gated_mm(x, pair, offsets.long()),
           lambda: S.gated_mm(x, h(3, 4, 8)), lambda: S.gated_mm(x, h(2, 4, 9)),
           lambda: S.gated_mm(x.bfloat16(), w), lambda: S.gated_mm(x.t(), w),
           lambda: S.gated_mm(x.cpu(), w), lambda: S.gated_mm(x.double(), w),
           lambda: S.gated_mm(x, w, out=h(6, 5)), lambda: S.gated_mm(x, h(2, 0, 8)),
           lambda: S.gated_mm(x, w, dtype=torch.float32), lambda: S.gated_mm(x, "w"),
           lambda: S.gated_mm_backward(h(5, 4), x, w, kept), lambda: S.gated_mm_backward(h(6, 5), x, w, kept),
           lambda: S.gated_mm_backward(dh, h(5, 8), w, kept), lambda: S.gated_mm_backward(dh, x, w, h(6, 4)),
           lambda: S.gated_mm_backward(dh, x, w, kept.bfloat16()),
           lambda: S.gated_mm_backward(dh, x, w, S.Packed8(p8.values[:5], p8.scales[:5])),
           lambda: S.gated_mm_backward(dh, x, w, S.Packed8(p8.values, p8.scales.int())),
           lambda: S.gated_mm_backward(dh, S.pack8(h(6, 9)), w, kept),
           lambda: S.gated_mm_backward(dh, x, w, kept, act=None),
           lambda: S.gated_mm_backward(dh, x, w, kept, offsets),
           lambda: S.pack8(x.int()), lambda: S.pack8(x.t()), lambda: S.pack8(h(3, 0)),
           lambda: S.pack8(x.cpu()), lambda: S.pack8([1.0]), lambda: S.pack8(x[0, 0]),
           lambda: S.unpack8(p8, torch.int8), lambda: S.unpack8(p8.values),
           lambda: S.unpack8(S.Packed8(p8.values, None)), lambda: S.unpack8(S.Packed8(None, p8.scales)),
           lambda: S.unpack8(S.Packed8(p8.values.float(), p8.scales)),
           lambda: S.unpack8(p8, torch.half, out=h(6, 8)),
           lambda: S.quantize_rows(x.long()), lambda: S.quantize_rows(h(0, 0)),
           lambda: S.int8_mm(x, w[0]), lambda: S.int8_mm(q, qp), lambda: S.int8_mm(q, qw, offsets),
           lambda: S.int8_mm(q, S.quantize_rows(h(4, 9))), lambda: S.int8_mm(h(6, 9), qw),
           lambda: S.int8_mm(q, qw, dtype=torch.int32), lambda: S.int8_mm(q, qw, out=h(6, 4)),
           lambda: S.int8_mm(S.Rows8(q.values, q.scales, 20), qw),
           lambda: S.int8_mm(S.Rows8(q.values, q.scales, "8"), qw),
           lambda: S.int8_mm(S.Rows8(q.values, q.scales[:5], 8), qw),
           lambda: S.int8_mm(S.Rows8(q.values.cpu(), q.scales, 8), qw),
           lambda: S.int8_mm(S.Rows8(byte, q.scales, 8), qw),
           lambda: S.gated_mm(q, w), lambda: S.gated_mm(q, qw), lambda: S.gated_mm(q, qp),
           lambda: S.gated_mm(q, qp, offsets[:3])]
    for i, call in enumerate(bad):
        with pytest.raises(S.SpmmError) as e:
            call()
        assert e.value.code == S.SPMM_INVALID, (i, str(e.value))
    for call in (lambda: S.gated_mm(x.float(), w.float()),
                 lambda: S.gated_mm_backward(dh.float(), x.float(), w.float(), kept.float()),
                 lambda: S.gated_mm(q, qp, offsets, keep="full")):
        with pytest.raises(S.SpmmError) as e:
            call()
        assert e.value.code == S.SPMM_UNSUPPORTED
    for call in (lambda s: S.gated_mm(x, w, stream=s), lambda s: S.pack8(x, stream=s),
                 lambda s: S.gated_mm_backward(dh, x, w, kept, stream=s),
                 lambda s: S.unpack8(p8, stream=s), lambda s: S.quantize_rows(x, stream=s),
                 lambda s: S.int8_mm(x, qw, stream=s)):
        with pytest.raises(S.SpmmError) as e:
            call(0)
        assert e.value.code == S.SPMM_INVALID and "stream" in str(e.value)


def test_c_entries_refuse_bad_arguments(S):
    import ctypes
    L, some, top = S.lib(), ctypes.c_void_p(4096), 0x7fffffff  # never read: the calls end before
    bad, not_here = S.SPMM_INVALID, S.SPMM_UNSUPPORTED
    gated = lambda **k: L.spmm_c_gated_mm(*{**dict(  # noqa: E731
        x=some, w=some, type=1, offsets=some, groups=2, rows=4, width=8, depth=8, act=0, out=some,
        kept=None, scales=None, stream=None), **k}.values())
    assert gated(x=None) == gated(w=None) == gated(offsets=None) == gated(out=None) == bad
    assert gated(scales=some) == gated(act=3) == gated(act=-1) == gated(type=7) == bad
    assert gated(groups=0) == gated(rows=-1) == gated(width=0) == gated(depth=0) == bad
    assert gated(type=0) == gated(depth=1 << 23) == gated(width=1 << 23) == gated(rows=top) == not_here
    many = 1 << 24
    assert gated(groups=many, rows=many) == not_here and b"2^32" in L.spmm_c_last_error()
    assert gated(groups=many, rows=many, kept=some, scales=some) == not_here
    assert gated(groups=many, rows=many, depth=7) == not_here
    assert gated(rows=0, x=None, out=None) == S.SPMM_OK
    grad = lambda **k: L.spmm_c_gated_grad(*{**dict(  # noqa: E731
        dh=some, type=1, kept=some, scales=None, rows=4, width=8, act=0, dkept=some, h=None,
        stream=None), **k}.values())
    assert grad(dh=None) == grad(kept=None) == grad(dkept=None) == grad(act=9) == grad(type=3) == bad
    assert grad(rows=-1) == grad(width=0) == bad
    assert grad(type=0) == grad(width=1 << 23) == not_here
    back = lambda **k: L.spmm_c_gated_mm_backward(*{**dict(  # noqa: E731
        dkept=some, x=some, w=some, type=1, offsets=some, groups=2, rows=4, width=8, depth=8, dx=some,
        dw=some, stream=None), **k}.values())
    assert back(dkept=None) == back(w=None) == back(offsets=None) == back(type=9) == bad
    assert back(dx=None, x=None) == back(rows=-1) == back(width=0) == back(groups=0) == bad
    assert back(type=0) == back(depth=1 << 23) == back(width=top) == back(width=1 << 22) == not_here
    assert back(groups=many, rows=many) == back(groups=many, rows=many, dx=None) == not_here
    assert back(dx=None, dw=None) == S.SPMM_OK
    for f in (lambda **k: L.spmm_c_pack8(*{**dict(x=some, type=0, rows=4, width=8, values=some,
                                                 scales=some, stream=None), **k}.values()),
              lambda **k: L.spmm_c_unpack8(*{**dict(values=some, scales=some, type=0, rows=4, width=8,
                                                   x=some, stream=None), **k}.values()),
              lambda **k: L.spmm_c_quantize_rows(*{**dict(x=some, type=0, rows=4, width=8, values=some,
                                                         scales=some, stream=None), **k}.values())):
        assert f(x=None) == f(values=None) == f(scales=None) == f(type=4) == bad
        assert f(rows=-1) == f(width=0) == bad
        assert f(width=top) == f(rows=1 << 40) == not_here
        assert f(rows=0, x=None, values=None, scales=None) == S.SPMM_OK
    ints = lambda **k: L.spmm_c_int8_mm(*{**dict(  # noqa: E731
        x=some, xs=some, w=some, ws=some, offsets=some, groups=2, rows=4, width=8, depth=16, type=1,
        out=some, stream=None), **k}.values())
    pair = lambda **k: L.spmm_c_gated_int8_mm(*{**dict(  # noqa: E731
        x=some, xs=some, w=some, ws=some, offsets=some, groups=2, rows=4, width=8, depth=16, act=0,
        type=1, out=some, stream=None), **k}.values())
    for f in (ints, pair):
        for name in ("x", "xs", "w", "ws", "offsets", "out"):
            assert f(**{name: None}) == bad
        assert f(depth=8) == f(depth=0) == f(depth=-16) == f(groups=0) == f(rows=-1) == f(width=0) == bad
        assert f(type=-1) == f(x=ctypes.c_void_p(4100)) == f(w=ctypes.c_void_p(4098)) == bad
        assert f(depth=131072) == f(width=1 << 23) == f(rows=top) == not_here
        assert f(groups=many, rows=many) == not_here
    assert pair(act=3) == bad
