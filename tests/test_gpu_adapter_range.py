"""The adapters' inner product scale x a^T keeps fp32's range and precision on its way
into the second product: values past fp16's largest and far below its smallest, and
results that are nothing but adapter."""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402

# of h, by what the 16-bit parts that stand for it leave out
SPLIT = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}

# rows, N, K, adapters, rank
SHAPES = [
    (5, 64, 64, 3, 16), (48, 256, 512, 20, 16),  # few rows
    (300, 256, 4096, 3, 48),                     # 64 x 64 tiles
    (1500, 1000, 520, 4, 8),                     # few rows, 64 columns a workgroup
    (4000, 1024, 1024, 4, 16), (4000, 1024, 1024, 3, 76),  # 128 x 128 tiles
    (4090, 4088, 1032, 3, 24), (4090, 4088, 1032, 3, 100),  # 256 x 256 tiles
    # rows that begin between two words, in few rows and tiles
    (33, 130, 129, 5, 12), (823, 200, 6787, 7, 12), (1500, 1000, 521, 4, 9),
]


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _check(S, x, w, a, b, ids, scale):
    dtype, u = x.dtype, R.ROUNDOFF[x.dtype]
    K, (L, rank) = x.shape[1], a.shape[:2]
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
        # h's own sum: K roundings in fp32; its parts, the low one of which has no bits below
        # 2^-38 of the row's largest in fp16
        own = (K + 1) * 2.0 ** -24 * abs(f) * (X[t].abs() @ A.abs().t()) + SPLIT[dtype] * h.abs()
        if dtype == torch.float16 and len(t):
            own += 2.0 ** -38 * h.abs().amax(1, keepdim=True)
        low[t] = own @ B.abs().t()
    assert want.abs().max() < torch.finfo(dtype).max / 2
    off = (y.double() - want).abs()
    # K + rank + 2 sums in fp32 beside that, then the one rounding to the result's type
    allowed = u * want.abs() + (1 + u) * ((K + rank + 2) * 2.0 ** -24 * size + low) + R.TINY[dtype]
    assert (off <= allowed).all(), float((off / allowed).max())
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,L,rank", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["mixed", "packed"])
def test_precision(S, T, N, K, L, rank, name, order):
    """A projection of zeros: the result is the adapter's part alone."""
    dtype = R.TYPES[name]
    ids = torch.arange(T, dtype=torch.int32, device="cuda") * 7 % (L + 1) - 1
    if order == "packed":
        ids = ids.sort().values
    x, w = _values((T, K), dtype, 1), torch.zeros((N, K), dtype=dtype, device="cuda")
    a, b = _values((L, rank, K), dtype, 2, K ** -0.5), _values((L, N, rank), dtype, 3)
    _check(S, x, w, a, b, ids, torch.linspace(0.5, 2.0, L, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,L,rank", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("f", [2.0 ** 22, 2.0 ** -40])
def test_range(S, T, N, K, L, rank, name, f):
    """scale x a^T of some 2^22 and 2^-40, against b (and x) the other way round; row 0 has
    large and small ones together."""
    dtype = R.TYPES[name]
    ids = torch.arange(T, dtype=torch.int32, device="cuda") % (L + 1) - 1
    ids[0] = 0
    big = f > 1
    x = _values((T, K), dtype, 1, 1.0 if big else 64.0)
    w = _values((N, K), dtype, 4, K ** -0.5 / 64)
    a = _values((L, rank, K), dtype, 2, K ** -0.5 if big else 256 * K ** -0.5)
    a[0, : rank // 2] *= 2.0 ** -6
    b = _values((L, N, rank), dtype, 3, 2.0 ** -14 if big else 1024.0)
    scale = torch.full((L,), f, device="cuda")
    want = _check(S, x, w, a, b, ids, scale)
    with_one = (ids >= 0).nonzero()[:, 0]
    h = f * (x[with_one].double() @ a[ids[with_one[-1]]].double().t()).abs()
    assert (h.max() > 65504) == big
    if big:
        part = want[with_one] - x[with_one].double() @ w.double().t()
        assert part.abs().max() > 8  # the adapters are what the result is made of


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,L,rank", SHAPES)
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_infinite_second_matrix(S, T, N, K, L, rank, name):
    """An infinity in b gives its column the infinity of the sum's sign, as the formula does."""
    dtype = R.TYPES[name]
    ids = torch.arange(T, dtype=torch.int32, device="cuda") % L
    x, w = _values((T, K), dtype, 1), _values((N, K), dtype, 4, K ** -0.5)
    a, b = _values((L, rank, K), dtype, 2, K ** -0.5), _values((L, N, rank), dtype, 3, rank ** -0.5)
    b[0, N // 2, rank - 1] = float("inf")
    y = S.adapter_mm(x, w, a, b, ids)
    rows = ids == 0
    h = x[rows].double() @ a[0, rank - 1].double()
    assert torch.equal(y[rows, N // 2].double(), torch.sign(h) * float("inf"))
    y[:, N // 2] = 0
    assert torch.isfinite(y).all()
