"""Quantised rows against max / 127 and x 127 / max in 64 bits, whatever way the kernel forms them.

The scale is a product of max with 1 / 127 in fp32, so two roundings from max / 127; the factor is
1 / max times 127, so two roundings from 127 / max, and an integer is the one next to x times that
factor: within half of x 127 / max, but for 127 times those two roundings.  Rows whose largest value
is below 2^-100 take that as their largest.
"""
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402

TWO = 2.01 * 2.0 ** -24  # two roundings to fp32


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(R.TYPES))
@pytest.mark.parametrize("rows,K", [(3000, 64), (2000, 1000), (700, 2050), (40, 8200)])
def test_quotients(S, name, rows, K):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, K), generator=g, device="cuda", dtype=torch.float64)
    low, high = {"f16": (-10, 12), "bf16": (-119, 120), "f32": (-119, 120)}[name]
    x *= torch.exp2(torch.randint(low, high, (rows, 1), generator=g, device="cuda").double())
    x = x.to(R.TYPES[name])
    q = S.quantize_rows(x)
    wide = x.double()
    largest = wide.abs().amax(1).clamp(min=2.0 ** -100)
    scale = q.scales.double()
    assert ((scale - largest / 127).abs() <= TWO * largest / 127).all()
    off = (q.values[:, :K].double() - wide * (127 / largest)[:, None]).abs()
    assert (off <= 0.5 + 127 * TWO).all()
    # so a value is off by half a step, and rows below the least one by as much
    assert ((q.values[:, :K].double() * scale[:, None] - wide).abs()
            <= (0.5 + 127 * 2 * TWO) * largest[:, None] / 127).all()
    if low < -108:
        tiny = wide.abs().amax(1) < 2.0 ** -108
        assert tiny.any() and (q.values[tiny] == 0).all()
