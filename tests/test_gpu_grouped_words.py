"""Grouped products whose rows are whole words but no whole 16-byte pieces: the tiles that
take them straight into LDS add up in the order of those that take them through registers,
as operands do that begin between two words."""
import pytest

torch = pytest.importorskip("torch")


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _between_words(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


# counts of the groups' rows, rows in all, N, K
SHAPES = [([1000, 0, 700, 1300], 3003, 2002, 1030), ([4096], 4100, 2052, 998), ([2000], 2000, 1002, 2050),
          ([130, 1, 900], 1040, 390, 4102), ([3000], 3000, 4094, 514), ([600, 600, 600], 1800, 770, 258)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("w_in_rows", [False, True])
def test_words_and_registers(S, counts, rows, N, K, dtype, w_in_rows):
    G = len(counts)
    x, dy = _values((rows, K), dtype, 1), _values((rows, N), dtype, 2)
    w = _values((G, K, N) if w_in_rows else (G, N, K), dtype, 3, K ** -0.5)
    first = rows - sum(counts)
    offsets = torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(G)], dtype=torch.int32,
                           device="cuda")
    y = S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows)
    dx, dw = S.grouped_mm_backward(dy, x, w, offsets, w_in_rows=w_in_rows)
    x1, w1, dy1 = (_between_words(t) for t in (x, w, dy))
    assert torch.equal(S.grouped_mm(x1, w1, offsets, w_in_rows=w_in_rows), y)
    dx1, dw1 = S.grouped_mm_backward(dy1, x1, w1, offsets, w_in_rows=w_in_rows)
    assert torch.equal(dx1, dx) and torch.equal(dw1, dw)
    assert (y[:first] == 0).all() and (dx[:first] == 0).all()
    # and they are the products: fp32 sums of up to as many terms, and one rounding
    for g in range(G):
        s = slice(first + sum(counts[:g]), first + sum(counts[:g + 1]))
        W = w[g].double() if w_in_rows else w[g].double().t()
        for got, a, b, n in ((y[s], x[s].double(), W, K), (dx[s], dy[s].double(), W.t(), N),
                             (dw[g] if w_in_rows else dw[g].t(), x[s].double().t(), dy[s].double(),
                              max(counts[g], 1))):
            u = torch.finfo(dtype).eps / 2
            off = n * 2.0 ** -24 * (a.abs() @ b.abs())
            want = a @ b
            assert ((got.double() - want).abs() <= u * want.abs() + (1 + u) * off + 2.0 ** -25).all()
