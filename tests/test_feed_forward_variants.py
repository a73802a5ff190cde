"""Which variant of the dense layers' kernels a call of given sizes takes: the rules, on the host (no GPU needed), and on
the GPU the results of each of them against float64."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from xnn_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("dtype", [0, 2, 3])
@pytest.mark.parametrize("grouped", [0, 1])
def test_long_reductions_of_one_or_two_rows_are_cut_into_parts(lib, dtype, grouped):
    """A stream of the weight, which needs no workspace, up to 1,500 inputs; then tiles, whose parts have sums there."""
    size = ctypes.c_size_t()
    for rows in (1, 2):
        for n_in, parts in ((64, False), (1500, False), (4096, True), (8192, True)):
            assert lib.xnn_linear_work_size(dtype, rows, n_in, 1024, 1 + 2 * grouped, grouped, ctypes.byref(size)) == 0
            assert (size.value > 0) is parts, (rows, n_in)
