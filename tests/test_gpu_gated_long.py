"""Gated products and packed activations past 2^31 elements, and calls at the same time from
several threads."""
import threading

import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402

ROWS, N, K = 135000, 8192, 72  # both projections hold 2.2e9 elements
TAIL = 300


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _exact(x, w):
    x, w = x.double(), w.double()
    return ([x @ w[j].t() for j in range(2)],
            [K * 2.0 ** -24 * (x.abs() @ w[j].abs().t()) for j in range(2)])


@pytest.mark.gpu
@pytest.mark.parametrize("keep", ["full", "8bit"])
def test_rows_past_31_bits(S, keep):
    """The last rows, which lie past 2^31 elements, are what the formulas give, forth and back."""
    dtype = torch.bfloat16
    x, w = _values((ROWS, K), dtype, 1), _values((2, N, K), dtype, 2, K ** -0.5)
    h, kept = S.gated_mm(x, w, keep=keep)
    (g, u), (eg, eu) = _exact(x[-TAIL:], w)
    G.close(h[-TAIL:], G.value(g, "silu") * u, G.product_bound(g, u, eg, eu, "silu"))
    if keep == "full":
        G.close(kept[-TAIL:, 0], g, eg)
        G.close(kept[-TAIL:, 1], u, eu)
        held = kept[-TAIL:]
    else:
        held = S.unpack8(S.Packed8(kept.values[-TAIL:].contiguous(), kept.scales[-TAIL:].contiguous()), dtype)
        assert torch.equal(S.unpack8(kept, dtype)[-TAIL:], held)
    del h
    # only the last rows' gradients, so that the weights' are theirs alone
    dh = torch.zeros((ROWS, N), dtype=dtype, device="cuda")
    dh[-TAIL:] = _values((TAIL, N), dtype, 3)
    dx, dw, again = S.gated_mm_backward(dh, x, w, kept, hidden=True)
    g, u = held.double().unbind(1)
    zero = torch.zeros_like(g)
    G.close(again[-TAIL:], G.value(g, "silu") * u, G.product_bound(g, u, zero, zero, "silu"))
    dg, du, eg, eu = G.gradients(dh[-TAIL:].double(), g, u, "silu")
    r = R.ROUNDOFF[dtype]
    d = torch.cat([dg, du], 1)
    e = torch.cat([eg, eu], 1) * (1 + r) + r * d.abs() + R.TINY[dtype]
    W, X = w.double().view(2 * N, K), x[-TAIL:].double()
    G.close(dx[-TAIL:], d @ W, (e + 2 * N * 2.0 ** -24 * (d.abs() + e)) @ W.abs())
    assert (dx[:-TAIL] == 0).all()
    # sums of as many terms other than zero as there are rows at the end
    G.close(dw.view(2 * N, K), d.t() @ X, (e + TAIL * 2.0 ** -24 * (d.abs() + e)).t() @ X.abs())


@pytest.mark.gpu
def test_bytes_past_31_bits(S):
    """Packed and quantised values past 2^31, and products of integers past 2^31 results."""
    width = 2 * N
    x = torch.zeros((ROWS, width), dtype=torch.float16, device="cuda")
    x[-TAIL:] = _values((TAIL, width), torch.float16, 1)
    alone = x[-TAIL:].contiguous()
    packed, part = S.pack8(x), S.pack8(alone)
    assert torch.equal(packed.values[-TAIL:], part.values) and torch.equal(packed.scales[-TAIL:], part.scales)
    assert torch.equal(S.unpack8(packed, torch.float16)[-TAIL:], S.unpack8(part, torch.float16))
    rows, part = S.quantize_rows(x), S.quantize_rows(alone)
    assert torch.equal(rows.values[-TAIL:], part.values) and torch.equal(rows.scales[-TAIL:], part.scales)
    w = S.quantize_rows(_values((40, width), torch.float16, 2))
    full = S.int8_mm(rows, w, dtype=torch.float32)
    sums = part.values.double() @ w.values.double().t()  # whole numbers below 2^53
    want = sums * part.scales.double()[:, None] * w.scales.double()
    # the sum as fp32 and two products
    assert ((full[-TAIL:].double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all()
    del packed, rows, full, x
    t, w = _values((ROWS, 32), torch.float16, 3), S.quantize_rows(_values((width, 32), torch.float16, 4))
    y = S.int8_mm(t, w, dtype=torch.float16)
    q = S.quantize_rows(t[-TAIL:].contiguous())
    want = (q.values.double() @ w.values.double().t()) * q.scales.double()[:, None] * w.scales.double()
    G.close(y[-TAIL:], want, 3.01 * 2.0 ** -24 * want.abs())


@pytest.mark.gpu
def test_calls_at_the_same_time(S):
    """Threads with a stream each get what one call after the other gets."""
    x, w = _values((333, 520), torch.float16, 1), _values((2, 264, 520), torch.float16, 2, 520 ** -0.5)
    dh, w8 = _values((333, 264), torch.float16, 3), S.quantize_rows(w)

    def calls():
        h, kept = S.gated_mm(x, w, keep="8bit")
        return [h, *S.gated_mm_backward(dh, S.pack8(x), w, kept), S.gated_mm(x, w8),
                S.int8_mm(x, S.quantize_rows(w[0].contiguous()))]

    want = calls()
    torch.cuda.synchronize()
    got, wrong = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = calls()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - a thread's own is lost
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for each in got:
        for a, b in zip(each, want):
            assert torch.equal(a, b)
