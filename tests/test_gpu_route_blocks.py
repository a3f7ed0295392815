"""Routing where the tokens go from one block to several, by choices, experts and type, and
the share of them that a block takes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import expert_reference as R  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("T", [48, 49, 64, 65, 128, 129, 8191, 8193, 16385])
@pytest.mark.parametrize("E,k", [(8, 1), (64, 4), (65, 5), (300, 1), (20, 17)])
@pytest.mark.parametrize("name", ["f32", "f16"])
def test_order(S, T, E, k, name):
    g = np.random.default_rng(T + E)
    v = g.uniform(-4.0, 4.0, (T, E))
    v[g.random((T, E)) < 0.3] = -np.inf
    logits = torch.from_numpy(v).to(R.TYPES[name])
    r = S.route(logits.cuda(), k)
    experts, weights, offsets, entries, slots = R.route(logits.double().numpy(), k, "chosen")
    for got, want in ((r.experts, experts), (r.offsets, offsets), (r.entries, entries),
                      (r.slots, slots)):
        assert np.array_equal(got.cpu().numpy(), want)
    # as in test_gpu_route.py: 64 roundings in fp32
    assert np.abs(r.weights.cpu().numpy() - weights).max() <= 64 * 2.0 ** -24


def _blocks(S, tokens, experts, k):
    """Blocks that the workspace has room for: an int an expert each."""
    return S.lib().spmm_c_route_workspace(tokens, experts, k) // (4 * experts)


@pytest.mark.parametrize("k", [1, 2, 4, 8, 64])
def test_tokens_are_shared(S, k):
    """Choices do not keep the tokens on few compute units, and blocks stay within 256."""
    for tokens, at_least in ((128, 4), (512, 16), (1024, 32), (8192, 256), (100000, 200)):
        assert at_least <= _blocks(S, tokens, 64, k) <= 256
    assert _blocks(S, 1, 64, k if k < 64 else 1) == 1
