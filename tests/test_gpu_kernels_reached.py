"""Which kernel each size of the gated, integer and grouped products' tests takes: where the choice
of forms changes, these say which sizes no longer reach the kernel that they are there for.  And
sizes for kernels that the other tests' do not reach: integers' gated products in two launches, the
256 x 256 tiles of gated groups, a weights' gradient in two launches, contractions of one part-filled
stage in 256 x 256 tiles of words."""
import pytest

torch = pytest.importorskip("torch")

import kernel_names  # noqa: E402
import test_gpu_gated_forms as F  # noqa: E402
import test_gpu_gated_range as range_tests  # noqa: E402
import test_gpu_grouped_words as W  # noqa: E402


def _some(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


# rows, N, K, groups, kernels without and with projections packed (None: the same)
GATED = [
    (20, 33, 521, 0, ["few"], ["ring64 odd"]), (50, 33, 64, 0, ["few"], ["ring64 pieces"]),
    (40, 700, 1002, 0, ["few"], ["ring64 words"]), (1, 33, 65, 0, ["ring64 odd"], None),
    (20, 2040, 64, 5, ["ring64 pieces"], None), (20, 2040, 66, 5, ["ring64 words"], None),
    (2000, 520, 521, 0, ["ring128 odd"], None), (2000, 520, 520, 0, ["ring128 pieces"], None),
    (2000, 520, 522, 0, ["ring128 words"], None), (2000, 520, 63, 0, ["tile odd"], None),
    (20, 4090, 64, 5, ["tile pieces"], None), (20, 4090, 66, 5, ["tile words"], None),
    (7000, 1000, 520, 0, ["wide pieces"], None), (7000, 1000, 574, 0, ["wide words"], None),
    (9000, 1024, 1030, 0, ["wide words", "ring64 words"], None),
    (9000, 1024, 1024, 0, ["wide pieces", "ring64 pieces"], None),
    (20000, 1024, 1024, 5, ["wide pieces"], None), (20000, 1024, 1026, 5, ["wide words"], None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,groups,plain,packed", GATED)
def test_gated(S, rows, N, K, groups, plain, packed):
    x, w = _some(rows, K), _some(*((groups, 2) if groups else (2,)), N, K)
    offsets = F._offsets(rows, groups)[1] if groups else None
    assert kernel_names.kernels(lambda: S.gated_mm(x, w, offsets)) == plain
    assert kernel_names.kernels(lambda: S.gated_mm(x, w, offsets, keep="full")) == plain
    assert kernel_names.kernels(lambda: S.gated_mm(x, w, offsets, keep="8bit")) == (packed or plain)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,groups", [(20000, 1024, 1024, 5), (20000, 1024, 1026, 5)])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_gated_values(S, rows, N, K, groups, name):
    F.test_gated(S, rows, N, K, groups, name)


# rows, N, K, groups, kernels of a product and of a gated one
INTS = [
    (200, 700, 4100, 0, ["few"], ["few"]), (100, 9000, 200, 2, ["ring64 pieces"], ["tile pieces"]),
    (2000, 520, 520, 0, ["ring64 pieces"], ["ring128 pieces"]),
    (4000, 520, 520, 0, ["ring128 pieces"], ["tile pieces"]),
    (20, 2040, 64, 5, ["few"], ["ring64 pieces"]), (7000, 2040, 1030, 0, ["wide pieces"], ["wide pieces"]),
    (9000, 2048, 1030, 0, ["wide pieces", "ring64 pieces"], ["tile pieces"]),
    (9000, 2048, 2050, 0, ["wide pieces", "ring64 pieces"], ["wide pieces", "ring128 pieces"]),
    (9000, 1024, 4096, 0, ["wide pieces"], ["wide pieces", "ring64 pieces"]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,groups,plain,gated", INTS)
def test_integers(S, rows, N, K, groups, plain, gated):
    lead = (groups,) if groups else ()
    x, one, pair = (S.quantize_rows(_some(*s, K)) for s in ((rows,), lead + (N,), lead + (2, N)))
    offsets = F._offsets(rows, groups)[1] if groups else None
    assert kernel_names.kernels(lambda: S.int8_mm(x, one, offsets)) == plain
    assert kernel_names.kernels(lambda: S.gated_mm(x, pair, offsets)) == gated


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", [(9000, 2048, 2050), (9000, 1024, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_integers_values(S, rows, N, K, dtype):
    F.test_integers(S, rows, N, K, 0, dtype)


# rows, N, K, kernels of the rows' and of the weights' gradient
GRADIENTS = [
    (1000, 1500, 511, ["shared"], ["shared"]), (1000, 1500, 514, ["shared"], ["ring128 words"]),
    (3000, 1024, 520, ["ring64 pieces"], ["tile pieces"]), (3000, 1024, 522, ["ring64 words"], ["ring128 words"]),
    (8200, 600, 2050, ["wide words", "ring128 words"], ["ring128 words"]),
    (8200, 600, 2048, ["wide pieces", "shared"], ["tile pieces"]),
    (3000, 4500, 2048, None, ["wide pieces", "tile pieces"]),
    (3000, 4500, 2050, None, ["wide words", "ring128 words"]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K,of_rows,of_weights", GRADIENTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients(S, rows, N, K, of_rows, of_weights, dtype):
    """(None: whatever it is)"""
    x, w, dh, kept = (_some(*s, dtype=dtype) for s in ((rows, K), (2, N, K), (rows, N), (rows, 2, N)))
    got = kernel_names.kernels(lambda: S.gated_mm_backward(dh, None, w, kept, weights=False))
    assert of_rows is None or got == of_rows
    assert kernel_names.kernels(lambda: S.gated_mm_backward(dh, x, w, kept, rows=False)) == of_weights


@pytest.mark.gpu
@pytest.mark.parametrize("rows,N,K", [(3000, 4500, 2048), (3000, 4500, 2050)])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_gradients_values(S, rows, N, K, name):
    F.test_gradients(S, rows, N, K, name)


@pytest.mark.gpu
def test_rows_times_powers_of_two_go_through_every_kernel(S):
    """The sizes of the tests of fp16's range."""
    rows_kernels, weights_kernels = set(), set()
    for counts, rows, N, K in range_tests.SIZES:
        x, dh, kept = (_some(*s, dtype=torch.half) for s in ((rows, K), (rows, N), (rows, 2, N)))
        w = _some(*(() if counts is None else (len(counts),)), 2, N, K, dtype=torch.half)
        offsets = None if counts is None else torch.tensor([0] + counts, device="cuda").cumsum(0).int()
        rows_kernels.update(kernel_names.kernels(
            lambda: S.gated_mm_backward(dh, None, w, kept, offsets, weights=False)))
        weights_kernels.update(kernel_names.kernels(
            lambda: S.gated_mm_backward(dh, x, w, kept, offsets, rows=False)))
    tiles = {"shared", "wide pieces", "wide words", "tile pieces", "tile odd", "ring128 words"}
    assert rows_kernels >= tiles | {"ring64 pieces", "ring64 words"}, rows_kernels
    assert weights_kernels >= tiles | {"tile words"}, weights_kernels


# counts of the groups' rows, rows in all, N, K: one stage, whose last 16 bytes a row are part-filled
ONE_STAGE = [([16384], 16384, 1024, 62), ([20000], 20003, 2050, 34), ([16384], 16384, 1024, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("counts,rows,N,K", ONE_STAGE)
@pytest.mark.parametrize("w_in_rows", [False, True])
def test_one_stage_of_words(S, counts, rows, N, K, w_in_rows):
    x, w = _some(rows, K), _some(*((1, K, N) if w_in_rows else (1, N, K)))
    offsets = torch.tensor([rows - counts[0], rows], dtype=torch.int32, device="cuda")
    assert kernel_names.kernels(lambda: S.grouped_mm(x, w, offsets, w_in_rows=w_in_rows)) == ["wide words"]
    for dtype in (torch.float16, torch.bfloat16):
        W.test_words_and_registers(S, counts, rows, N, K, dtype, w_in_rows)
