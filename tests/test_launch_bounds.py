"""Launches of 2^32 threads and more, which HIP takes without an error and does not run,
are refused by the C entries before anything reaches a GPU, and so are sizes whose last
tile or step would not be a 32-bit integer."""
import ctypes

import spmm_amd as S

F16, BF16 = 1, 2
SOME = ctypes.c_void_p(4096)  # never read: the call ends before


def _refused(code):
    assert code == S.SPMM_UNSUPPORTED
    assert "2^32 threads" in S.lib().spmm_c_last_error().decode()


def test_products_of_too_many_tiles():
    L = S.lib()
    many = 1 << 24  # groups, each with a tile of its own
    _refused(L.spmm_c_grouped_mm(SOME, SOME, F16, SOME, many, many, 8, 8, 0, SOME, None))
    _refused(L.spmm_c_grouped_mm(SOME, SOME, F16, SOME, many, many, 8, 8, 1, SOME, None))
    _refused(L.spmm_c_grouped_mm(SOME, SOME, BF16, SOME, many, many, 7, 9, 1, SOME, None))
    _refused(L.spmm_c_grouped_outer(SOME, SOME, F16, SOME, many, many, 8, 8, SOME, None))


def test_adapters_of_too_many_rows():
    _refused(S.lib().spmm_c_adapter_mm(SOME, SOME, SOME, SOME, SOME, None, BF16, 3 << 28, 8, 8, 4,
                                       8, SOME, SOME, None))


def test_sizes_next_to_the_largest_integer():
    L, top = S.lib(), 0x7fffffff
    for code in (L.spmm_c_dispatch(SOME, F16, 1, 1, top, SOME, SOME, 1, SOME, None),
                 L.spmm_c_combine(SOME, F16, 1, 1, top, SOME, None, SOME, None),
                 L.spmm_c_combine_backward(SOME, SOME, F16, 1, 1, top, SOME, SOME, SOME, 1, SOME, SOME,
                                           None),
                 L.spmm_c_grouped_mm(SOME, SOME, F16, SOME, 1, top, 8, 8, 1, SOME, None),
                 L.spmm_c_grouped_outer(SOME, SOME, F16, SOME, 1, top, 8, 8, SOME, None),
                 L.spmm_c_adapter_mm(SOME, SOME, SOME, SOME, SOME, None, BF16, top, 8, 8, 4, 8, SOME,
                                     SOME, None)):
        assert code == S.SPMM_UNSUPPORTED
