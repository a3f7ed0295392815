"""Packed activations and quantised rows, bit for bit against numpy, and products in 8-bit
integers, whose sums are exact and whose scaling is three roundings in a known order."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402
import gated_reference as G  # noqa: E402

SHAPES = [(1, 1), (1, 8), (3, 7), (2, 31), (5, 32), (4, 33), (7, 64), (3, 100), (2, 5, 48), (61, 1000),
          (9, 2047), (6, 2050), (4, 8192), (2, 8200), (1, 40000), (1000, 17), (64,), (600, 2056)]


def _values(shape, dtype, seed, scale=1.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal(shape) * scale * 2.0 ** g.integers(-12, 4, shape[:-1] + (1,))
    x[g.random(shape) < 0.05] = 0
    return torch.from_numpy(x).to(dtype)


def _f32(t):
    return t.float().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", sorted(R.TYPES))
def test_pack_and_unpack(S, shape, name):
    x = _values(shape, R.TYPES[name], 1)
    packed = S.pack8(x.cuda())
    q, scale = G.pack(_f32(x))
    assert packed.values.shape == x.shape and packed.scales.shape == scale.shape
    assert np.array_equal(packed.values.cpu().numpy(), q)
    assert np.array_equal(packed.scales.cpu().numpy(), scale)
    want = torch.from_numpy(G.unpack(q, scale))
    for dtype in R.TYPES.values():
        assert torch.equal(S.unpack8(packed, dtype).cpu(), want.to(dtype))


def _special(dtype):
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [[0.0], [top], [-top, top], [float("inf")], [1.0, float("nan")], [-float("inf"), 2.0],
            [low], [low / 2], [-low / 8, low], [1.0, 127.5 / 128, 127 / 128, -255 / 256],
            [64.5, 65.5, -64.5, 0.5, 1.5, 127.0, 127.5, -127.75], [2.0 ** -14], [top / 3, 1.0]]
    x = torch.zeros((len(rows), 40), dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, 3:3 + len(r)] = torch.tensor(r, dtype=torch.float64)
        x[i, 35] = r[-1]
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(R.TYPES))
def test_special_values(S, name):
    x = _special(R.TYPES[name])
    packed = S.pack8(x.cuda())
    q, scale = G.pack(_f32(x))
    assert np.array_equal(packed.values.cpu().numpy(), q)
    assert np.array_equal(packed.scales.cpu().numpy(), scale)
    want = torch.from_numpy(G.unpack(q, scale))
    for dtype in R.TYPES.values():
        got = S.unpack8(packed, dtype).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0, 9, -9), want.to(dtype).nan_to_num(0, 9, -9))
    rows = S.quantize_rows(x.cuda())
    q, scale = G.quantise(_f32(x))
    assert np.array_equal(rows.values.cpu().numpy(), q)
    assert np.array_equal(rows.scales.cpu().numpy(), scale, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", sorted(R.TYPES))
def test_quantize_rows(S, shape, name):
    x = _values(shape, R.TYPES[name], 2)
    rows = S.quantize_rows(x.cuda())
    q, scale = G.quantise(_f32(x))
    assert rows.width == shape[-1]
    assert np.array_equal(rows.values.cpu().numpy(), q)
    assert np.array_equal(rows.scales.cpu().numpy(), scale)


def _rows8(S, shape, seed):
    """Quantised rows of all values an int8 has, and their scales."""
    g = np.random.default_rng(seed)
    K = shape[-1]
    q = np.zeros(shape[:-1] + (-(-K // 16) * 16,), np.int8)
    q[..., :K] = g.integers(-128, 128, shape)
    scale = (2.0 ** g.uniform(-9, 1, shape[:-1])).astype(np.float32)
    return q, scale, S.Rows8(torch.from_numpy(q).cuda(), torch.from_numpy(scale).cuda(), K)


def _sums(q, w):
    return torch.from_numpy(q).cuda().double() @ torch.from_numpy(w).cuda().double().t()


def _scaled(sums, sx, sw, dtype):
    f = sums.float() * torch.from_numpy(sw).cuda() * torch.from_numpy(sx).cuda()[:, None]
    return f.to(dtype)


# rows, N, K
PRODUCTS = [(1, 1, 1), (1, 64, 16), (2, 33, 100), (16, 512, 4096), (20, 264, 1040), (40, 1000, 2050),
            (64, 4096, 512), (70, 12800, 272), (130, 200, 777), (300, 520, 4096), (600, 1024, 8200),
            (2100, 2040, 1030), (4099, 4088, 520), (33, 8, 131056)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", PRODUCTS)
@pytest.mark.parametrize("name", sorted(R.TYPES))
def test_int8_mm(S, rows, N, K, name):
    q, sx, x = _rows8(S, (rows, K), 1)
    p, sw, w = _rows8(S, (N, K), 2)
    dtype = R.TYPES[name]
    y = S.int8_mm(x, w, dtype=dtype)
    assert y.dtype == dtype and torch.equal(y, _scaled(_sums(q, p), sx, sw, dtype))


GROUPS = [([0, 1, 0], 1, 17, 33), ([3, 0, 5], 11, 100, 72), ([130, 1, 0, 127], 258, 130, 200),
          ([7] * 70, 490, 33, 65), ([4] * 60, 256, 72, 520), ([900, 0, 1, 700], 1601, 1000, 776),
          ([2500, 4400], 7000, 2040, 1032), ([32] * 64, 2048, 512, 4096), ([0, 0], 5, 40, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", GROUPS)
def test_int8_groups(S, counts, rows, N, K):
    n = len(counts)
    q, sx, x = _rows8(S, (rows, K), 3)
    p, sw, w = _rows8(S, (n, N, K), 4)
    first = min(2, rows - sum(counts))
    o = first + np.concatenate([[0], np.cumsum(counts)])
    # scales of rows in no group are not looked at
    x.scales[:first] = float("nan")
    x.scales[o[-1]:] = float("nan")
    y = S.int8_mm(x, w, torch.from_numpy(o.astype(np.int32)).cuda())
    want = torch.zeros((rows, N), dtype=torch.bfloat16, device="cuda")
    for g in range(n):
        s = slice(o[g], o[g + 1])
        want[s] = _scaled(_sums(q[s], p[g]), sx[s], sw[g], torch.bfloat16)
    assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(R.TYPES))
def test_int8_of_a_tensor(S, name):
    """A tensor is quantised a row at a time; a row with an infinity becomes NaN, no other."""
    x = _values((37, 500), R.TYPES[name], 5)
    x[4, 7] = float("inf")
    w = _values((90, 500), R.TYPES[name], 6)
    w[11, 3] = float("nan")
    y = S.int8_mm(x.cuda(), S.quantize_rows(w.cuda()))
    assert y.dtype == x.dtype
    (q, sx), (p, sw) = G.quantise(_f32(x)), G.quantise(_f32(w))
    want = _scaled(_sums(q, p), sx, sw, x.dtype)
    assert torch.isnan(y[4]).all() and torch.isnan(y[:, 11]).all()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y.nan_to_num(0), want.nan_to_num(0))
