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


# --------------------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 70])
@pytest.mark.parametrize("n_in", [10, 1500, 1501])
def test_an_infinite_float32_input(rows, n_in):
    """NaN, for infinity has no planes; in one or two rows of up to 1,500 inputs the product's own infinity."""
    import torch
    import xnn_amd as xa
    x = torch.ones(rows, n_in, device="cuda")
    x[:, n_in // 2] = float("inf")
    w = torch.randn(n_in, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    w = torch.where(w == 0, torch.ones_like(w), w)
    got = xa.linear(x, w)
    if rows <= 2 and n_in <= 1500:
        assert torch.equal(got, (w[n_in // 2].sign() * float("inf")).expand(rows, 40))
    else:
        assert got.isnan().all()
